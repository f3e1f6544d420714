"""Forms of the layer operators that only certain sizes take: the recurrence in more than 1024 segments, the norm's split form
with means far from 0, with NaN and infinities, with narrow units and with many groups.  Bounds as in layer_refs.py."""
import pytest
import torch

import layer_refs as R
from test_gpu_layers import DTYPES, norm_case, rand


@pytest.fixture(scope="module")
def layers():
    from pl_convlstm_gan_amd import layers as m
    return m


@pytest.mark.parametrize("coupled", [True, False])
def test_reference_of_long_sequences(coupled):
    """The doubling form of the reference against its loop (64 bits: 1e-12 of values of order 1 to 10)."""
    dev = torch.device("cpu")
    x, f, dy = rand((3, 130, 4), 1, torch.float32, dev), rand((3, 130, 4), 2, torch.float32, dev, 1.5, 2.0), rand((3, 130, 4), 3, torch.float32, dev)
    h0, dh = rand((3, 4), 4, torch.float32, dev), rand((3, 4), 5, torch.float32, dev)
    for n in (None, torch.tensor([130, 0, 77], dtype=torch.int32)):
        for p, q in zip(R.scan(x, f, h0, n, coupled, dy, dh), R.scan_long(x, f, h0, n, coupled, dy, dh)):
            for k in p:
                assert float((p[k] - q[k]).abs().max()) <= 1e-12 * max(1.0, float(p[k].abs().max())), k


@pytest.mark.gpu
@pytest.mark.parametrize("B,D,lengths", [(1, 3, None), (2, 2, [(1 << 18) + 5, 100003]), (1, 8, [(1 << 18) - 1]), (3, 1, [0, 1, (1 << 18) + 5])])
@pytest.mark.parametrize("dtype,coupled", [(torch.float32, True), (torch.float32, False), (torch.bfloat16, True)])
def test_scan_in_thousands_of_segments(layers, gpu, B, D, lengths, dtype, coupled):
    """From 2^18 steps on a sequence is cut into up to 4096 segments, and the carry reads its runs in several pieces."""
    T = (1 << 18) + 5
    x, f, dy = rand((B, T, D), 1, dtype, gpu), rand((B, T, D), 2, dtype, gpu, 1.5, 2.0), rand((B, T, D), 3, dtype, gpu)
    h0, dh = rand((B, D), 4, torch.float32, gpu), rand((B, D), 5, torch.float32, gpu)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=gpu)
    leaves = [t.requires_grad_() for t in (x, f, h0)]
    y, h = layers.gated_linear_scan(x, f, h0, lengths=n, coupled=coupled)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    val, err = R.scan_long(x, f, h0, n, coupled, dy, dh)
    for k, v in zip(("y", "h_last", "dx", "df", "dh0"), (y, h) + tuple(grads)):
        R.check(v, val[k], err[k], f"{k} {B} {D} {dtype} coupled={coupled} lengths={lengths}")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 16, 128, 130), 4), ((1, 7, 150, 151), 1), ((1, 2056, 20, 21), 1), ((1, 64, 96, 100), 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_split_form_with_a_far_mean(layers, gpu, shape, groups, dtype):
    """The mean 300 deviations from 0 in frames that no workgroup holds: block means, pivots and partial sums are merged without
    the loss that sums of squares around 0 would have.  (A 16-bit x has lost digits before the operator sees it.)"""
    norm_case(layers, gpu, shape, groups, dtype, shift=200.0)
    norm_case(layers, gpu, shape, groups, dtype, "relu", shift=-200.0, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("groups,act,p", [(4, "silu", 0.0), (1, "relu", 0.3)])
def test_norm_engine_layout_with_a_far_mean(gpu, groups, act, p):
    import ctypes as C
    from pl_convlstm_gan_amd import _lib, ops
    L, st = _lib.lib(), ops._stream()
    N, ch, H, W = 2, 32, 130, 131
    x, dy = rand((N, ch, H, W), 1, torch.bfloat16, gpu, 4.0, 200.0), rand((N, ch, H, W), 2, torch.bfloat16, gpu)
    w, b = rand((ch,), 3, torch.float32, gpu, 0.3, 1.0), rand((ch,), 4, torch.float32, gpu, 0.3)
    cb8 = lambda t: t.view(N, ch // 8, 8, H, W).permute(0, 1, 3, 4, 2).contiguous()  # noqa: E731
    nchw = lambda t: t.permute(0, 1, 4, 2, 3).reshape(N, ch, H, W)  # noqa: E731
    X, G = cb8(x), cb8(dy)
    Y, DX = torch.empty_like(X), torch.empty_like(X)
    stats, dw, db = torch.empty(N, groups, 2, device=gpu), torch.empty(ch, device=gpu), torch.empty(ch, device=gpu)
    d = _lib.NormDesc()
    d.N, d.C, d.G, d.HW, d.dtype, d.layout, d.act, d.eps, d.p, d.seed, d.offset = N, ch, groups, H * W, 1, 1, ops._act(act), 1e-5, p, 9, 4
    d.x, d.weight, d.bias, d.y, d.stats = X.data_ptr(), w.data_ptr(), b.data_ptr(), Y.data_ptr(), stats.data_ptr()
    d.dy, d.dx, d.dweight, d.dbias = G.data_ptr(), DX.data_ptr(), dw.data_ptr(), db.data_ptr()
    for backward, call in ((0, L.plc_group_norm_fwd), (1, L.plc_group_norm_bwd)):
        n = L.plc_group_norm_workspace_bytes(C.byref(d), backward)
        ws = torch.empty(n, dtype=torch.uint8, device=gpu)
        d.workspace, d.workspace_bytes = ws.data_ptr(), n
        _lib.check(call(C.byref(d), st), "group norm")
    val, err = R.norm(x, groups, w, b, 1e-5, act, p, 9, 4, dy)
    for k, v in (("y", nchw(Y)), ("dx", nchw(DX)), ("dw", dw), ("db", db)):
        R.check(v, val[k], err[k], f"{k} {groups} {act} {p}")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1, 7, 150, 151), 1), ((2, 7, 150, 151), 7), ((1, 6, 150, 151), 2), ((1, 12, 130, 121), 4), ((1, 30, 128, 131), 3), ((1, 3, 257, 511), 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_split_form_with_narrow_units(layers, gpu, shape, groups, dtype):
    """Units of one, two or four elements, for which activation and dropout are not compiled in, in whole rounds of pixels and the rest."""
    norm_case(layers, gpu, shape, groups, dtype, "silu")
    norm_case(layers, gpu, shape, groups, dtype, "relu", 0.25, seed=9)
    norm_case(layers, gpu, shape, groups, dtype, "none", 0.5, affine=False, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 8, 9, 9), 4), ((2, 8, 150, 151), 4), ((1, 6, 150, 151), 3), ((1, 2056, 20, 21), 2), ((2, 64, 96, 100), 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_keeps_what_is_not_finite_in_its_group(layers, gpu, shape, groups, value, dtype):
    """One NaN or infinity: every output of its group is NaN (its variance is), every other value, gradients included, has
    the bits it has without.  Both forms."""
    N, C, H, W = shape
    x = rand((N, H, W, C), 1, dtype, gpu).permute(0, 3, 1, 2)
    bad = x.clone(memory_format=torch.preserve_format)
    bad[0, 1, H // 2, W // 2] = value
    dy = rand((N, H, W, C), 2, dtype, gpu).permute(0, 3, 1, 2)
    inside = torch.zeros(shape, dtype=torch.bool, device=gpu)
    channels = torch.arange(C, device=gpu) // (C // groups) == 1 // (C // groups)       # (of channel 1's group)
    inside[0, channels] = True
    for act in ("none", "relu", "silu"):
        out = []
        for v in (x, bad):
            leaves = [v.detach().requires_grad_(), torch.ones(C, device=gpu, requires_grad=True), torch.zeros(C, device=gpu, requires_grad=True)]
            y = layers.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act)
            out.append((y.detach(),) + torch.autograd.grad(y, leaves, dy))
        (y0, dx0, dw0, db0), (y1, dx1, dw1, db1) = out
        assert torch.equal(torch.isnan(y1), inside), act
        assert torch.equal(y1[~inside], y0[~inside]) and torch.equal(dx1[~inside], dx0[~inside]), act
        assert torch.equal(dw1[~channels], dw0[~channels]) and torch.equal(db1[~channels], db0[~channels]), act
        assert torch.isnan(dx1[inside]).all(), act
