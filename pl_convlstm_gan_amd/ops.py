"""Thin Python wrappers over the C ABI: pointer/stream plumbing only, no arithmetic.

Every function requires CUDA(HIP) fp32 contiguous tensors and raises otherwise; there is no
CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _require_dev(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(
            f"{name} is on {t.device}: the ConvLSTM engine runs on MI355X (HIP) only; there is no CPU fallback")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32 (got {t.dtype}); the engine converts to bf16 internally")
    return t.contiguous()


def staging_device() -> torch.device:
    """Where CPU-resident operands are staged for the HIP kernels.  There is no CPU arithmetic path:
    without a GPU this raises."""
    if not torch.cuda.is_available():
        raise RuntimeError("the ConvLSTM engine runs on MI355X (HIP) only and no GPU is visible; "
                           "there is no CPU fallback")
    return torch.device("cuda", torch.cuda.current_device())


def workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def convlstm_cell_forward(x, h, c, weight, bias):
    """ConvLSTMCell.forward on the HIP kernel.  NCHW fp32 in, (h', c') NCHW fp32 out."""
    L = _lib.lib()
    x = _require_dev(x, "x")
    h = _require_dev(h, "h_cur")
    c = _require_dev(c, "c_cur")
    weight = _require_dev(weight, "weight")
    B, Cin, H, W = x.shape
    Ch = h.shape[1]
    if weight.shape != (4 * Ch, Cin + Ch, 3, 3):
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match (4*{Ch}, {Cin}+{Ch}, 3, 3)")
    if h.shape != (B, Ch, H, W) or c.shape != (B, Ch, H, W):
        raise ValueError("h_cur / c_cur shape mismatch")
    bias_p = _require_dev(bias, "bias").data_ptr() if bias is not None else None
    h2 = torch.empty_like(h)
    c2 = torch.empty_like(c)
    nbytes = L.plc_convlstm_cell_workspace_bytes(B, Cin, Ch, H, W)
    ws = workspace(nbytes, x.device)
    rc = L.plc_convlstm_cell_fwd(x.data_ptr(), h.data_ptr(), c.data_ptr(), weight.data_ptr(), bias_p,
                                 h2.data_ptr(), c2.data_ptr(), ws.data_ptr(), nbytes, B, Cin, Ch, H, W, _stream())
    _lib.check(rc, "plc_convlstm_cell_fwd")
    return h2, c2


def convlstm_cell_backward(x, h, c, weight, bias, dh_next, dc_next):
    """Gradients of ConvLSTMCell.forward: returns (dx, dh, dc, dweight, dbias)."""
    L = _lib.lib()
    x, h, c, weight = (_require_dev(t, n) for t, n in ((x, "x"), (h, "h_cur"), (c, "c_cur"), (weight, "weight")))
    dh_next = _require_dev(dh_next, "dh_next")
    dc_next = _require_dev(dc_next, "dc_next")
    B, Cin, H, W = x.shape
    Ch = h.shape[1]
    dx, dh, dc = torch.empty_like(x), torch.empty_like(h), torch.empty_like(c)
    dw = torch.empty_like(weight)
    db = torch.empty(4 * Ch, dtype=torch.float32, device=x.device)
    nbytes = L.plc_convlstm_cell_bwd_workspace_bytes(B, Cin, Ch, H, W)
    ws = workspace(nbytes, x.device)
    bias_p = _require_dev(bias, "bias").data_ptr() if bias is not None else None
    rc = L.plc_convlstm_cell_bwd(x.data_ptr(), h.data_ptr(), c.data_ptr(), weight.data_ptr(), bias_p,
                                 dh_next.data_ptr(), dc_next.data_ptr(), dx.data_ptr(), dh.data_ptr(), dc.data_ptr(),
                                 dw.data_ptr(), db.data_ptr(), ws.data_ptr(), nbytes, B, Cin, Ch, H, W, _stream())
    _lib.check(rc, "plc_convlstm_cell_bwd")
    return dx, dh, dc, dw, (db if bias is not None else None)


def to_cb8_bf16(x: torch.Tensor) -> torch.Tensor:
    """NCHW fp32 -> CB8 bf16 [N][ceil(C/8)][H][W][8] (returned as an int16 tensor)."""
    L = _lib.lib()
    x = _require_dev(x, "x")
    N, Cc, H, W = x.shape
    out = torch.empty((N, (Cc + 7) // 8, H, W, 8), dtype=torch.int16, device=x.device)
    _lib.check(L.plc_nchw_f32_to_cb8_bf16(x.data_ptr(), out.data_ptr(), N, Cc, H, W, _stream()), "to_cb8_bf16")
    return out


def from_cb8_bf16(x: torch.Tensor, channels: int) -> torch.Tensor:
    L = _lib.lib()
    N, ncb, H, W, _ = x.shape
    out = torch.empty((N, channels, H, W), dtype=torch.float32, device=x.device)
    _lib.check(L.plc_cb8_bf16_to_nchw_f32(x.data_ptr(), out.data_ptr(), N, channels, H, W, _stream()),
               "from_cb8_bf16")
    return out


# ------------------------------------------------------------------------------------------------ layer operators
# The explicit forward and backward passes behind layers.py (plc_gated_scan_*, plc_group_norm_*, plc_dropout).  fp32, bf16
# and fp16 tensors, on any device and on its current stream; checks, allocation and calls are native (csrc/plc_torch.cpp).
_ACTS = {"none": 0, "relu": 1, "silu": 2}
_U64 = 1 << 64


def _act(act) -> int:
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)} (got {act!r})")
    return _ACTS[act]


def _draw(seed, offset):
    """-> (seed, offset, device offset or None); ``offset``: an integer, or an int64 tensor of one element that the
    kernel reads when it runs."""
    if not 0 <= seed < _U64:
        raise ValueError(f"seed must be in 0 .. 2^64 - 1 (got {seed})")
    if isinstance(offset, torch.Tensor):
        return seed, 0, offset
    if not 0 <= offset < _U64:
        raise ValueError(f"offset must be in 0 .. 2^64 - 1 (got {offset})")
    return seed, offset, None


def _inside_backward() -> bool:
    """Whether this thread is running a backward pass, as where activations are recomputed."""
    return torch._C._current_graph_task_id() != -1


def gated_scan_forward(x, f, h0=None, lengths=None, coupled=True, save_states=False, h_last=None):
    """plc_gated_scan_fwd on [B, T, ...]: returns (y, h_last, states); states (what the backward pass needs beside the
    inputs) is None unless ``save_states`` and T > 8.  ``h_last``: where the last state goes (may be h0 itself)."""
    return _lib.binding().scan_forward(x, f, h0, lengths, coupled, save_states, h_last)


def gated_scan_backward(x, f, h0, lengths, coupled, states, dy, dh_last, need_dh0=True):
    """plc_gated_scan_bwd: returns (dx, df, dh0); dy [B, T, ...] in x's type or None, dh_last fp32 [B, ...] or None."""
    return _lib.binding().scan_backward(x, f, h0, lengths, coupled, states, dy, dh_last, need_dh0)


def dropout_forward(x, p, seed, offset=0, residual=None, used_offset=None):
    """plc_dropout on the elements of x in their logical order: returns y.  ``used_offset``: int64 tensor of one
    element that receives the offset a device ``offset`` held."""
    seed, offset, offset_t = _draw(seed, offset)
    return _lib.binding().dropout_forward(x, p, seed, offset, offset_t, residual, used_offset)


def group_norm_forward(x, groups, weight=None, bias=None, eps=1e-5, act="none", p=0.0, seed=0, offset=0, used_offset=None):
    """plc_group_norm_fwd on [N, C, H, W], channels last in memory (other layouts are copied into it): returns
    (y, stats), y channels last, stats fp32 [N, groups, 2]."""
    seed, offset, offset_t = _draw(seed, offset)
    return _lib.binding().norm_forward(x, groups, weight, bias, eps, _act(act), p, seed, offset, offset_t, used_offset)


def group_norm_backward(x, groups, weight, bias, eps, act, p, seed, offset, stats, dy):
    """plc_group_norm_bwd: returns (dx, dweight, dbias); dx channels last, dweight / dbias None without weight / bias."""
    seed, offset, offset_t = _draw(seed, offset)
    return _lib.binding().norm_backward(x, groups, weight, bias, eps, _act(act), p, seed, offset, offset_t, stats, dy)
