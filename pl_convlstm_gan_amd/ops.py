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
# (plc_gated_scan_*, plc_group_norm_*, plc_dropout: fp32, bf16 and fp16 tensors, on any device and on its current stream)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"none": 0, "relu": 1, "silu": 2}
_U64 = 1 << 64


class _Launch:
    """Context of a library call: makes ``device`` the current one where it is not (a launch goes to the current
    device) and gives the address of its current stream."""

    def __init__(self, device: torch.device):
        self.index = device.index
        self.guard = None

    def __enter__(self) -> int:
        if self.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _require_layer(t, name: str, like: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(
            f"{name} is on {t.device}: the layer operators run on MI355X (HIP) only; there is no CPU fallback")
    if dtype is not None:
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    elif t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the input on {like.device}")
    return t


def _steps(t: torch.Tensor):
    """[B, T, ...] -> (tensor, stride of a sample, stride of a step) with the rest contiguous; copies only if it is not."""
    inner = t.numel() // max(t.shape[0] * t.shape[1], 1)
    if t.is_contiguous():
        return t, t.shape[1] * inner, inner
    if t.numel() and t[0, 0].is_contiguous():
        return t, t.stride(0), t.stride(1)
    t = t.contiguous()
    return t, t.shape[1] * inner, inner


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _scan_desc(x, f, h0, lengths, coupled):
    d = _lib.ScanDesc()
    d.B, d.T = x.shape[0], x.shape[1]
    D = 1
    for n in x.shape[2:]:
        D *= n
    d.D = D
    d.dtype = _DTYPES[x.dtype]
    d.coupled = 1 if coupled else 0
    x, d.x_batch, d.x_step = _steps(x)
    f, d.f_batch, d.f_step = _steps(f)
    d.x, d.f, d.h0, d.lengths = x.data_ptr(), f.data_ptr(), _ptr(h0), _ptr(lengths)
    return d, (x, f)


def gated_scan_check(x, f, h0, lengths):
    """The checks of gated_scan_forward; returns (x, f, h0, lengths) as the kernels take them."""
    x = _require_layer(x, "x")
    f = _require_layer(f, "f", x, x.dtype)
    if x.dim() < 2 or x.shape != f.shape:
        raise ValueError(f"x and f must both be [B, T, ...] (got {tuple(x.shape)} and {tuple(f.shape)})")
    if h0 is not None:
        h0 = _require_layer(h0, "h0", x, torch.float32)
        if h0.shape != x.shape[:1] + x.shape[2:]:
            raise ValueError(f"h0 must be {tuple(x.shape[:1] + x.shape[2:])} (got {tuple(h0.shape)})")
        h0 = h0.contiguous()
    if lengths is not None:
        lengths = _require_layer(lengths, "lengths", x, torch.int32)
        if lengths.shape != x.shape[:1]:
            raise ValueError(f"lengths must be [{x.shape[0]}] (got {tuple(lengths.shape)})")
        lengths = lengths.contiguous()
    return x, f, h0, lengths


def gated_scan_forward(x, f, h0=None, lengths=None, coupled=True, save_states=False, h_last=None):
    """plc_gated_scan_fwd: returns (y, h_last, states); states (what the backward pass needs beside the inputs) is
    None unless ``save_states``.  ``h_last``: where the last state goes (may be h0 itself)."""
    L = _lib.lib()
    x, f, h0, lengths = gated_scan_check(x, f, h0, lengths)
    d, keep = _scan_desc(x, f, h0, lengths, coupled)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if h_last is None:
        h_last = torch.empty(x.shape[:1] + x.shape[2:], dtype=torch.float32, device=x.device)
    states = None
    if save_states:
        n = L.plc_gated_scan_states_bytes(d.B, d.T, d.D)
        states = torch.empty(n // 4, dtype=torch.float32, device=x.device) if n else None
    d.y, d.h_last, d.states = y.data_ptr(), h_last.data_ptr(), _ptr(states)
    n = L.plc_gated_scan_workspace_bytes(C.byref(d), 0)
    ws = workspace(n, x.device) if n else None
    d.workspace, d.workspace_bytes = _ptr(ws), n
    with _Launch(x.device) as stream:
        rc = L.plc_gated_scan_fwd(C.byref(d), stream)
    _lib.check(rc, "plc_gated_scan_fwd")
    return y, h_last, states


def gated_scan_backward(x, f, h0, lengths, coupled, states, dy, dh_last, need_dh0=True):
    """plc_gated_scan_bwd: returns (dx, df, dh0); dy [B, T, ...] in x's type or None, dh_last fp32 [B, ...] or None."""
    L = _lib.lib()
    x, f, h0, lengths = gated_scan_check(x, f, h0, lengths)
    d, keep = _scan_desc(x, f, h0, lengths, coupled)
    dy = torch.zeros_like(x) if dy is None else _require_layer(dy, "dy", x, x.dtype)
    if dy.shape != x.shape:
        raise ValueError(f"dy must be {tuple(x.shape)} (got {tuple(dy.shape)})")
    dy, d.dy_batch, d.dy_step = _steps(dy)
    if dh_last is not None:
        dh_last = _require_layer(dh_last, "dh_last", x, torch.float32).contiguous()
        if dh_last.shape != x.shape[:1] + x.shape[2:]:
            raise ValueError(f"dh_last must be {tuple(x.shape[:1] + x.shape[2:])} (got {tuple(dh_last.shape)})")
    n = L.plc_gated_scan_states_bytes(d.B, d.T, d.D)
    if n:
        states = _require_layer(states, "states", x, torch.float32)
        if states.numel() * 4 < n:
            raise ValueError("states do not belong to these inputs")
    dx, df = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dh0 = torch.empty(x.shape[:1] + x.shape[2:], dtype=torch.float32, device=x.device) if need_dh0 else None
    d.states, d.dy, d.dh_last, d.dx, d.df, d.dh0 = _ptr(states), dy.data_ptr(), _ptr(dh_last), dx.data_ptr(), df.data_ptr(), _ptr(dh0)
    n = L.plc_gated_scan_workspace_bytes(C.byref(d), 1)
    ws = workspace(n, x.device) if n else None
    d.workspace, d.workspace_bytes = _ptr(ws), n
    with _Launch(x.device) as stream:
        rc = L.plc_gated_scan_bwd(C.byref(d), stream)
    _lib.check(rc, "plc_gated_scan_bwd")
    return dx, df, dh0


def _drop_args(p, seed, offset, like):
    """-> (p, seed, offset, device offset or None); ``offset``: an integer, or an int64 tensor of one element that
    the kernel reads when it runs."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be a probability (got {p})")
    if not 0 <= seed < _U64:
        raise ValueError(f"seed must be in 0 .. 2^64 - 1 (got {seed})")
    if isinstance(offset, torch.Tensor):
        _require_layer(offset, "offset", like, torch.int64)
        if offset.numel() != 1:
            raise ValueError(f"offset must have one element (got {offset.numel()})")
        return p, int(seed), 0, offset
    if not 0 <= offset < _U64:
        raise ValueError(f"offset must be in 0 .. 2^64 - 1 (got {offset})")
    return p, int(seed), int(offset), None


def dropout_forward(x, p, seed, offset=0, residual=None, used_offset=None):
    """plc_dropout on the elements of x in their logical order: returns y.  ``used_offset``: int64 tensor of one
    element that receives the offset a device ``offset`` held."""
    L = _lib.lib()
    x = _require_layer(x, "x").contiguous()
    if residual is not None:
        residual = _require_layer(residual, "residual", x, x.dtype)
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)} (got {tuple(residual.shape)})")
        residual = residual.contiguous()
    p, seed, off, off_t = _drop_args(p, seed, offset, x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _Launch(x.device) as stream:
        rc = L.plc_dropout(x.data_ptr(), _ptr(residual), y.data_ptr(), x.numel(), _DTYPES[x.dtype], p, seed, off,
                           _ptr(off_t), _ptr(used_offset), stream)
    _lib.check(rc, "plc_dropout")
    return y


def _nhwc(t: torch.Tensor) -> torch.Tensor:
    return t.contiguous(memory_format=torch.channels_last)


def _norm_desc(x, groups, weight, bias, eps, act, p, seed, off, off_t, stats):
    d = _lib.NormDesc()
    d.N, d.C, d.G, d.HW = x.shape[0], x.shape[1], groups, x.shape[2] * x.shape[3]
    d.dtype, d.layout, d.act, d.eps = _DTYPES[x.dtype], 0, _ACTS[act], eps
    d.x, d.weight, d.bias, d.stats = x.data_ptr(), _ptr(weight), _ptr(bias), stats.data_ptr()
    d.p, d.seed, d.offset, d.offset_ptr = p, seed, off, _ptr(off_t)
    return d


def group_norm_check(x, groups, weight, bias, eps, act):
    x = _require_layer(x, "x")
    if x.dim() != 4:
        raise ValueError(f"x must be [N, C, H, W] (got {tuple(x.shape)})")
    ch = x.shape[1]
    if groups < 1 or ch < 1 or ch % groups:
        raise ValueError(f"{ch} channels do not divide into {groups} groups")
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)} (got {act!r})")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    out = []
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            t = _require_layer(t, name, x, torch.float32)
            if t.shape != (ch,):
                raise ValueError(f"{name} must be [{ch}] (got {tuple(t.shape)})")
            t = t.contiguous()
        out.append(t)
    return _nhwc(x), out[0], out[1]


def group_norm_forward(x, groups, weight=None, bias=None, eps=1e-5, act="none", p=0.0, seed=0, offset=0, used_offset=None):
    """plc_group_norm_fwd on [N, C, H, W], channels last in memory (other layouts are copied into it): returns
    (y, stats), y channels last, stats fp32 [N, groups, 2]."""
    L = _lib.lib()
    x, weight, bias = group_norm_check(x, groups, weight, bias, eps, act)
    p, seed, off, off_t = _drop_args(p, seed, offset, x)
    y = torch.empty_like(x, memory_format=torch.channels_last)
    stats = torch.empty((x.shape[0], groups, 2), dtype=torch.float32, device=x.device)
    d = _norm_desc(x, groups, weight, bias, eps, act, p, seed, off, off_t, stats)
    d.y, d.used_offset = y.data_ptr(), _ptr(used_offset)
    n = L.plc_group_norm_workspace_bytes(C.byref(d), 0)
    ws = workspace(n, x.device)
    d.workspace, d.workspace_bytes = ws.data_ptr(), n
    with _Launch(x.device) as stream:
        rc = L.plc_group_norm_fwd(C.byref(d), stream)
    _lib.check(rc, "plc_group_norm_fwd")
    return y, stats


def group_norm_backward(x, groups, weight, bias, eps, act, p, seed, offset, stats, dy):
    """plc_group_norm_bwd: returns (dx, dweight, dbias); dx channels last, dweight / dbias None without weight / bias."""
    L = _lib.lib()
    x, weight, bias = group_norm_check(x, groups, weight, bias, eps, act)
    p, seed, off, off_t = _drop_args(p, seed, offset, x)
    dy = _nhwc(_require_layer(dy, "dy", x, x.dtype))
    if dy.shape != x.shape:
        raise ValueError(f"dy must be {tuple(x.shape)} (got {tuple(dy.shape)})")
    stats = _require_layer(stats, "stats", x, torch.float32)
    if stats.shape != (x.shape[0], groups, 2) or not stats.is_contiguous():
        raise ValueError("stats do not belong to these inputs")
    dx = torch.empty_like(x, memory_format=torch.channels_last)
    dw = torch.empty_like(weight) if weight is not None else None
    db = torch.empty_like(bias) if bias is not None else None
    d = _norm_desc(x, groups, weight, bias, eps, act, p, seed, off, off_t, stats)
    d.dy, d.dx, d.dweight, d.dbias = dy.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(db)
    n = L.plc_group_norm_workspace_bytes(C.byref(d), 1)
    ws = workspace(n, x.device)
    d.workspace, d.workspace_bytes = ws.data_ptr(), n
    with _Launch(x.device) as stream:
        rc = L.plc_group_norm_bwd(C.byref(d), stream)
    _lib.check(rc, "plc_group_norm_bwd")
    return dx, dw, db
