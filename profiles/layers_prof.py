"""Records of the layer operators (layers_kernel_stats.txt, layers_kernel_traffic.csv, layers_head_step.txt), made by layers_prof.sh.

    layers_prof.py run NAME-PART[,NAME-PART] PASSES    passes of the cases of perf/operators.py whose names hold a part
    layers_prof.py stats FOLDER                        kernels of a `rocprofv3 --kernel-trace` run of one case
    layers_prof.py traffic FETCH-FOLDER WRITE-FOLDER   bytes by kernel from two `rocprofv3 --pmc` runs
    layers_prof.py head                                train step and forward pass with and without the feature head (256 x 256, T = 10, batch 32)
"""
import collections
import csv
import glob
import os
import re
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def median(v):
    return sorted(v)[len(v) // 2]


def run(parts, passes):
    import importlib.util
    import torch
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    for c in cases.listed():
        if any(p in c["name"] for p in parts.split(",")):
            states = [cases.prepare(c, k) for k in range(3)]
            for i in range(int(passes)):
                cases.run(states[i % 3])
            torch.cuda.synchronize()
            print(c["name"], flush=True)


def stats(folder):
    d = collections.OrderedDict()
    for path in glob.glob(folder + "/**/*kernel_trace.csv", recursive=True):
        for r in csv.DictReader(open(path)):
            m = re.search(r"plc_\w+?_kernel", r["Kernel_Name"])
            if m:
                key = (m.group(0), r["Kernel_Name"], r["Grid_Size_X"], r["VGPR_Count"], r["LDS_Block_Size"])
                d.setdefault(key, []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    for (name, _, grid, vgpr, lds), v in d.items():
        print("  %-32s work items %9s  VGPRs %3s  LDS %5s  launches %3d  median %8.2f us  min %8.2f" % (name, grid, vgpr, lds, len(v), median(v), min(v)))


def traffic(fetch, write):
    # (FETCH_SIZE counts half of what is read on this card, WRITE_SIZE all that is written; both in KiB)
    d = collections.OrderedDict()
    for counter, folder in (("FETCH_SIZE", fetch), ("WRITE_SIZE", write)):
        for path in glob.glob(folder + "/**/*counter_collection.csv", recursive=True):
            for r in csv.DictReader(open(path)):
                m = re.search(r"plc_\w+?_kernel", r["Kernel_Name"])
                if m:
                    d.setdefault((m.group(0), r["Grid_Size"], r["Kernel_Name"]), {}).setdefault(counter, []).append(float(r["Counter_Value"]))
    print("kernel,work items,launches,fetched MB (2 x FETCH_SIZE),written MB (WRITE_SIZE)")
    for (name, grid, _), v in d.items():
        print("%s,%s,%d,%.1f,%.1f" % (name, grid, len(v["FETCH_SIZE"]), 2 * median(v["FETCH_SIZE"]) * 1024 / 1e6, median(v.get("WRITE_SIZE", [0])) * 1024 / 1e6))


def head():
    import torch
    from bench import synthetic
    from pl_convlstm_gan_amd import Generator
    from pl_convlstm_gan_amd.losses import CombinedLoss
    from pl_convlstm_gan_amd.optim import FusedAdam
    from pl_convlstm_gan_amd.training import train_step
    dev = torch.device("cuda:0")
    data = synthetic(32, 10, 256, 256, 1, 1234, dev)
    heads = (("no head", None), ("8 groups, silu", (8, "silu", 0.0)), ("8 groups, silu, dropout 0.1", (8, "silu", 0.1)))
    times = collections.defaultdict(list)
    for _ in range(3):                               # (in turn: the card's clock moves)
        for name, args in heads:
            torch.manual_seed(0)
            model = Generator(hidden_dims=[16, 32], lu_channels=5, scale_factor=1)
            if args:
                model.set_feature_head(*args)
            model = model.to(dev)
            with torch.no_grad():
                model(*(t[:1, :1].contiguous() if t.dim() == 5 else t[:1].contiguous() for t in data[:3]))
            loss, opt = CombinedLoss(), FusedAdam(model.parameters(), lr=5e-4)

            def forward():
                with torch.no_grad():
                    return model(*data[:3])
            for kind, call in (("train step", lambda: train_step(model, loss, opt, *data, max_norm=0.5, nan_check="device")), ("forward", forward)):
                for _ in range(4):
                    call()
                torch.cuda.synchronize()
                t0 = time.perf_counter()
                for _ in range(15):
                    call()
                torch.cuda.synchronize()
                times[kind, name].append((time.perf_counter() - t0) / 15 * 1e3)
            del model, loss, opt
            torch.cuda.empty_cache()
    print("256 x 256, T = 10, batch 32, hidden [16, 32], bf16: ms, median of three runs in turn")
    for (kind, name), v in times.items():
        print("%-12s %-30s %7.2f   (%s)" % (kind, name, median(v), ", ".join("%.2f" % t for t in v)), flush=True)


if __name__ == "__main__":
    {"run": run, "stats": stats, "traffic": traffic, "head": head}[sys.argv[1]](*sys.argv[2:])
