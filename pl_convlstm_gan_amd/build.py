"""In-tree build of libplconvlstm.so with hipcc for gfx950 (cross-compiles without a GPU) and of its PyTorch binding."""
from __future__ import annotations

import glob
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
# (the rollout engine, the layer operators, and the group norm's kernels by element type: compiled side by side)
SRCS = [os.path.join(HERE, "csrc", name + ".hip") for name in ("plc_api", "plc_layers", "plc_norm_f32", "plc_norm_bf16", "plc_norm_f16")]
OUT = os.path.join(HERE, "libplconvlstm.so")
# (the PyTorch binding of the layer operators: host code against torch's headers, no device code)
BINDING_SRC = os.path.join(HERE, "csrc", "plc_torch.cpp")
BINDING = os.path.join(HERE, "_plc_torch.so")
DEPS = sorted(glob.glob(os.path.join(HERE, "csrc", "*.h")) + glob.glob(os.path.join(HERE, "csrc", "*.hip")) + [BINDING_SRC]) + \
       [os.path.join(os.path.dirname(HERE), "include", "plconvlstm.h"), os.path.abspath(__file__)]


def is_stale() -> bool:
    if not (os.path.exists(OUT) and os.path.exists(BINDING)):
        return True
    t = min(os.path.getmtime(OUT), os.path.getmtime(BINDING))
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in DEPS)


def _binding_command():
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    libs = library_paths()
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_plc_torch",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            *(f"-I{p}" for p in include_paths()), "-I/opt/rocm/include", f"-I{sysconfig.get_paths()['include']}", BINDING_SRC, "-o", BINDING,
            *(f"-L{p}" for p in libs), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python", *(f"-Wl,-rpath,{p}" for p in libs)]


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and not is_stale():
        return OUT
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    # No packed fp32 arithmetic: on the MI355X a packed fp32 instruction whose SECOND source takes its low half from the
    # high dword (v_pk_fma_f32 ... op_sel:[0,1,0], v_pk_add_f32 ... op_sel:[0,1]) gives wrong results now and then while
    # an MFMA kernel runs on the chip at the same time (devtools/pk_opsel_probe.hip: 1.5e-4 of the instructions; never
    # alone), and the compiler forms such encodings from ordinary scalar code and from vector types.
    # -fno-slp-vectorize keeps it from pairing scalar arithmetic, the target feature takes the instructions away
    # (tests/test_host_logic.py checks the built code object).  Measured cost of both: none (default train step 21.73 ms
    # without the instructions, 21.76 with the hand-paired ones; forward 5.11 and 5.12).
    flags = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-fno-slp-vectorize", "-fPIC",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    objs = [os.path.splitext(src)[0] + ".o" for src in SRCS]
    cmds = [[hipcc, *flags, "-c", "-o", obj, src] for src, obj in zip(SRCS, objs)]
    link = [hipcc, "--offload-arch=gfx950", "-shared", "-o", OUT, *objs]
    if verbose:
        for cmd in cmds + [_binding_command(), link]:
            print(" ".join(cmd), flush=True)
    cmds.append(_binding_command())
    running = [subprocess.Popen(cmd) for cmd in cmds]
    failed = [cmd for cmd, proc in zip(cmds, running) if proc.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    subprocess.run(link, check=True)
    return OUT


if __name__ == "__main__":
    build(force=True)
