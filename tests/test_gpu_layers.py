"""The layer operators (gated linear recurrence, group norm with an activation, counter-based dropout) on the GPU against
64-bit references, element by element, within bounds that follow the operations (tests/layer_refs.py)."""
import pytest
import torch

import layer_refs as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def layers():
    from pl_convlstm_gan_amd import layers as m
    return m


def rand(shape, seed, dtype, dev, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(dev)


# ------------------------------------------------------------------------------------ gated linear recurrence
def scan_case(layers, gpu, shape, dtype, coupled=True, lengths=None, h0=True, last=True, seed=0):
    B = shape[0]
    state = shape[:1] + shape[2:]
    x, f = rand(shape, seed, dtype, gpu), rand(shape, seed + 1, dtype, gpu, 1.5, 2.0)
    s0 = rand(state, seed + 2, torch.float32, gpu) if h0 else None
    dy, dh = rand(shape, seed + 3, dtype, gpu), rand(state, seed + 4, torch.float32, gpu) if last else None
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=gpu)
    leaves = [t.requires_grad_() for t in (x, f, s0) if t is not None]
    y, h = layers.gated_linear_scan(x, f, s0, lengths=n, coupled=coupled)
    outs, up = ((y, h), (dy, dh)) if last else ((y,), (dy,))
    grads = torch.autograd.grad(outs, leaves, up)
    val, err = R.scan(x, f, s0, n, coupled, dy, dh)
    got = dict(zip(("y", "h_last", "dx", "df", "dh0"), (y, h) + tuple(grads)))
    for k, v in got.items():
        R.check(v, val[k], err[k], f"{k} {shape} {dtype} coupled={coupled} lengths={lengths}")
    assert y.dtype == x.dtype and h.dtype == torch.float32 and grads[0].dtype == x.dtype
    # without gradients: the same bits
    with torch.no_grad():
        y2, h2 = layers.gated_linear_scan(x, f, s0, lengths=n, coupled=coupled)
    assert torch.equal(y2, y) and torch.equal(h2, h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("coupled", [True, False])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 100])
def test_scan_lengths_in_time(layers, gpu, T, coupled, dtype):
    scan_case(layers, gpu, (3, T, 24), dtype, coupled)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 4, 7, 8, 12, 48, 129, 520])
def test_scan_widths(layers, gpu, D, dtype):
    scan_case(layers, gpu, (2, 19, D), dtype)


@pytest.mark.parametrize("shape", [(2, 1000, 5), (1, 4099, 16), (1, 8192, 3), (5, 700, 6, 4), (2, 18, 9, 7, 8), (70, 20, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_long_and_shaped(layers, gpu, shape, dtype):
    scan_case(layers, gpu, shape, dtype)


@pytest.mark.parametrize("T,lengths", [(20, [20, 0, 7, 16, 1]), (500, [500, 0, 33, 480, 16]), (3000, [1, 2999, 0, 1024, 3000]), (9, [-4, 1 << 30, 0, 3, 9])])
@pytest.mark.parametrize("coupled", [True, False])
def test_scan_lengths_of_samples(layers, gpu, T, lengths, coupled):
    for dtype in (torch.float32, torch.bfloat16):
        scan_case(layers, gpu, (5, T, 24), dtype, coupled, lengths)


@pytest.mark.parametrize("h0,last", [(False, True), (True, False), (False, False)])
def test_scan_without_states(layers, gpu, h0, last):
    scan_case(layers, gpu, (2, 37, 10), torch.float32, True, None, h0, last)
    scan_case(layers, gpu, (2, 1500, 10), torch.float32, False, [1500, 3], h0, last)


@pytest.mark.parametrize("T", [40, 2000])
def test_scan_padding_never_reaches_a_result(layers, gpu, T):
    """NaN and infinities behind a sample's length: outputs and gradients there are 0, everything else as without them."""
    shape, n = (3, T, 20), torch.tensor([T, 5, 0], dtype=torch.int32, device=gpu)
    x, f, dy = (rand(shape, k, torch.float32, gpu) for k in range(3))
    h0, dh = rand((3, 20), 4, torch.float32, gpu), rand((3, 20), 5, torch.float32, gpu)

    def run(x, f, dy):
        x, f, s = (t.clone().requires_grad_() for t in (x, f, h0))
        y, h = layers.gated_linear_scan(x, f, s, lengths=n)
        return (y, h) + torch.autograd.grad((y, h), (x, f, s), (dy, dh))

    clean = run(x, f, dy)
    for t, v in ((x, float("nan")), (f, float("inf")), (dy, float("-inf"))):
        t[1, 5:], t[2] = v, v
    dirty = run(x, f, dy)
    for k, (a, b) in enumerate(zip(clean, dirty)):
        assert torch.equal(a, b), k
    assert torch.equal(dirty[1][2], h0[2]) and torch.equal(dirty[4][2], dh[2])       # a sample without a step
    assert float(dirty[0].detach()[1, 5:].abs().max()) == 0 and float(dirty[2][1, 5:].abs().max()) == 0


def test_scan_strides_views_and_broadcasts(layers, gpu):
    base = rand((3, 2, 40, 26), 1, torch.bfloat16, gpu)
    tmajor = base[0].transpose(0, 1).contiguous().transpose(0, 1)         # [T][B][D] in memory
    views = {
        "time major": (tmajor, base[1].transpose(0, 1).contiguous().transpose(0, 1)),
        "slice of channels": (base[0][:, :, 1:24], base[1][:, :, 2:25]),
        "every second step": (base[0][:, ::2], base[1][:, 1::2]),
        "flipped copy": (base[0].flip(1), base[1]),
        "inner not contiguous": (base[0][:, :, ::2], base[1][:, :, 1::2]),
        "one gate for all samples": (base[0], base[1][:1].expand(2, 40, 26)),
        "one gate for all steps": (base[0], base[1][:, :1].expand(2, 40, 26)),
    }
    for name, (x, f) in views.items():
        a = layers.gated_linear_scan(x, f)
        b = layers.gated_linear_scan(x.clone(memory_format=torch.contiguous_format), f.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), name
    # gradient of a broadcast gate: the sum over what it was broadcast to; of a strided dy: as of its copy
    x, f, dy = base[0].float(), base[1][:1].float().requires_grad_(), base[2].float()
    y, _ = layers.gated_linear_scan(x, f.expand(2, 40, 26))
    (df,) = torch.autograd.grad(y, f, dy.transpose(1, 2).contiguous().transpose(1, 2))
    val, err = R.scan(x, f.detach().expand(2, 40, 26), None, None, True, dy)
    R.check(df, val["df"].sum(0, keepdim=True), err["df"].sum(0, keepdim=True) + 4 * R.U * val["df"].abs().sum(0, keepdim=True), "df")
    x = base[0].float().requires_grad_()
    layers.gated_linear_scan(x, base[1].float())[0].sum().backward()       # dy: one value, expanded
    val, err = R.scan(x, base[1].float(), None, None, True, torch.ones_like(x))
    R.check(x.grad, val["dx"], err["dx"], "dx of a sum")


def test_scan_extreme_gates(layers, gpu):
    """Gates of the types' largest values and infinities: s is exactly 0 or 1, no NaN appears."""
    for dtype in DTYPES:
        big = torch.finfo(dtype).max
        f = torch.tensor([float("inf"), big, 100.0, -100.0, -big, float("-inf"), 0.0], device=gpu).repeat(6, 1).to(dtype)[None]
        x = rand((1, 6, 7), 3, dtype, gpu)
        h0 = rand((1, 7), 4, torch.float32, gpu)
        x.requires_grad_(), f.requires_grad_()
        y, h = layers.gated_linear_scan(x, f, h0)
        dx, df = torch.autograd.grad(y, (x, f), torch.ones_like(y))
        assert torch.isfinite(y).all() and torch.isfinite(dx).all() and torch.isfinite(df).all()
        assert torch.equal(h[0, :3], h0[0, :3]) and torch.equal(y[0, :, 5], x[0, :, 5])
    # a NaN stays in its own sample and channel
    x = rand((2, 30, 8), 5, torch.float32, gpu)
    x[0, 3, 2] = float("nan")
    y, h = layers.gated_linear_scan(x, rand((2, 30, 8), 6, torch.float32, gpu))
    bad = torch.isnan(y)
    assert bad[0, 3:, 2].all() and int(bad.sum()) == 27 and int(torch.isnan(h).sum()) == 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_step_by_step_is_the_scan(layers, gpu, dtype):
    """The single-step form carried through time gives the scan's states; the state in place and in a new tensor."""
    for coupled in (True, False):
        x, f = rand((3, 12, 5, 7), 1, dtype, gpu), rand((3, 12, 5, 7), 2, dtype, gpu)
        state = rand((3, 5, 7), 3, torch.float32, gpu)
        y, h = layers.gated_linear_scan(x, f, state, coupled=coupled)
        inplace = state.clone()
        for t in range(12):
            got, state = layers.gated_linear_step(x[:, t], f[:, t], state, coupled=coupled)
            got2, same = layers.gated_linear_step(x[:, t], f[:, t], inplace, coupled=coupled, inplace=True)
            assert same.data_ptr() == inplace.data_ptr() and torch.equal(got, got2) and torch.equal(state, inplace)
            assert torch.equal(got, y[:, t])
        assert torch.equal(state, h)


@pytest.mark.parametrize("T", [1, 30, 700])
def test_scan_state_in_place(layers, gpu, T):
    """The last state may overwrite the first, also where the sequence is worked on in segments."""
    from pl_convlstm_gan_amd import ops
    x, f, h0 = rand((2, T, 6), 1, torch.float32, gpu), rand((2, T, 6), 2, torch.float32, gpu), rand((2, 6), 3, torch.float32, gpu)
    y, h, _ = ops.gated_scan_forward(x, f, h0)
    state = h0.clone()
    y2, h2, _ = ops.gated_scan_forward(x, f, state, h_last=state)
    assert h2.data_ptr() == state.data_ptr() and torch.equal(y, y2) and torch.equal(h, state)


def test_explicit_passes_are_autograds(layers, gpu):
    """ops.*_forward / *_backward, the passes without autograd, give what autograd gives, bit for bit."""
    from pl_convlstm_gan_amd import ops
    x, f, h0 = rand((2, 50, 6), 1, torch.bfloat16, gpu), rand((2, 50, 6), 2, torch.bfloat16, gpu), rand((2, 6), 3, torch.float32, gpu)
    dy, dh = rand((2, 50, 6), 4, torch.bfloat16, gpu), rand((2, 6), 5, torch.float32, gpu)
    n = torch.tensor([50, 11], dtype=torch.int32, device=gpu)
    _, _, states = ops.gated_scan_forward(x, f, h0, n, True, save_states=True)
    a = ops.gated_scan_backward(x, f, h0, n, True, states, dy, dh)
    leaves = [t.clone().requires_grad_() for t in (x, f, h0)]
    b = torch.autograd.grad(layers.gated_linear_scan(*leaves, lengths=n), leaves, (dy, dh))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    x, w = rand((2, 12, 9, 7), 6, torch.float32, gpu), rand((12,), 7, torch.float32, gpu)
    dy = rand((2, 12, 9, 7), 8, torch.float32, gpu)
    y, stats = ops.group_norm_forward(x, 3, w, None, 1e-5, "silu", 0.2, 5, 6)
    a = ops.group_norm_backward(x, 3, w, None, 1e-5, "silu", 0.2, 5, 6, stats, dy)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    z = layers.group_norm_act(leaves[0], 3, leaves[1], None, act="silu", p=0.2, seed=5, offset=6)
    b = torch.autograd.grad(z, leaves, dy)
    assert torch.equal(y, z) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[2] is None
    with pytest.raises(ValueError, match="states"):
        ops.gated_scan_backward(rand((2, 50, 6), 1, torch.bfloat16, gpu), f[:, :50], h0, n, True, None, rand((2, 50, 6), 4, torch.bfloat16, gpu), dh)


def test_changed_inputs_are_refused_in_the_backward_pass(layers, gpu):
    x, f = (rand((1, 20, 8), k, torch.float32, gpu).requires_grad_() for k in (1, 2))
    a = x * 1
    y, _ = layers.gated_linear_scan(a, f)
    a.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_two_threads_at_once(layers, gpu):
    """Calls from two host threads, each on its own stream: the results of the calls alone."""
    import threading
    leaves, _ = block_inputs(gpu, torch.bfloat16)
    leaves = [t.detach() for t in leaves]
    want = [block(layers, *leaves, o)[0] for o in (1, 2)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(block(layers, *leaves, i + 1)[0])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert all(len(g) == 20 and all(torch.equal(o, w) for o in g) for g, w in zip(got, want))


def test_scan_pieces_carry_the_state(layers, gpu):
    """A sequence in two pieces, the state carried in fp32: as in one, values and gradients.  The bits need not agree: the
    sequence in one call may be computed as segments whose maps h -> A h + S are joined, the pieces step by step.  Either
    is within e + r of the 64-bit value v (e the recurrence's bound over all 90 steps, r half a step of the type), so by the
    triangle inequality they are within 2 (e + r) of one another; both bounds are checked as |one - v|, |two - v| <= e + r."""
    x, f = rand((2, 90, 12), 1, torch.bfloat16, gpu).requires_grad_(), rand((2, 90, 12), 2, torch.bfloat16, gpu).requires_grad_()
    y, h = layers.gated_linear_scan(x, f)
    a, ha = layers.gated_linear_scan(x[:, :48], f[:, :48])
    b, hb = layers.gated_linear_scan(x[:, 48:], f[:, 48:], ha)
    dy = rand((2, 90, 12), 3, torch.bfloat16, gpu)
    one = torch.autograd.grad(y, (x, f), dy)
    two = torch.autograd.grad((a, b), (x, f), (dy[:, :48], dy[:, 48:]))
    val, err = R.scan(x, f, None, None, True, dy)
    for k, p, q in zip(("y", "h_last", "dx", "df"), (y, h) + one, (torch.cat([a, b], 1), hb) + two):
        R.check(p, val[k], err[k], k + " in one")
        R.check(q, val[k], err[k], k + " in two pieces")


def test_scan_step_in_place_is_seen_by_autograd(layers, gpu):
    """A state that a backward pass still needs and a step in place overwrites: an error, not a wrong gradient."""
    x, f = rand((2, 5, 12), 1, torch.float32, gpu).requires_grad_(), rand((2, 5, 12), 2, torch.float32, gpu)
    h0 = rand((2, 12), 3, torch.float32, gpu)
    y, _ = layers.gated_linear_scan(x, f, h0)
    layers.gated_linear_step(f[:, 0], f[:, 1], h0)
    y.sum().backward(retain_graph=True)
    layers.gated_linear_step(f[:, 0], f[:, 1], h0, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        state = torch.zeros(2, 12, device=gpu)
        layers.gated_linear_step(f[:, 0], f[:, 1], state, inplace=True)
        assert torch.equal(state, layers.gated_linear_step(f[:, 0], f[:, 1], torch.zeros(2, 12, device=gpu))[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", [(1, 79, 6), (1, 80, 6), (2, 96, 1024), (3, 127, 2048), (3, 250, 2048), (2, 129, 1030), (1, 2100, 40), (1, 9000, 16), (2, 300, 20482)])
def test_scan_around_the_split(layers, gpu, dtype, B, T, D):
    """Lengths and widths on both sides of every choice between one pass and segments, and of the carry's run lengths."""
    scan_case(layers, gpu, (B, T, D), dtype, True, [T - 3, T // 2, T][:B])


def test_scan_gradient_against_differences(layers, gpu):
    """Directional derivatives of the 64-bit recurrence by central differences (step 1e-6: truncation 1e-12, rounding
    1e-10 of the value) against the kernel's gradients."""
    shape = (2, 300, 4)
    x, f, h0 = rand(shape, 1, torch.float32, gpu), rand(shape, 2, torch.float32, gpu), rand((2, 4), 3, torch.float32, gpu)
    dy, dh = rand(shape, 4, torch.float32, gpu), rand((2, 4), 5, torch.float32, gpu)
    v = [rand(t.shape, 6 + k, torch.float32, gpu).double() for k, t in enumerate((x, f, h0))]
    for coupled in (True, False):
        xs = [t.clone().requires_grad_() for t in (x, f, h0)]
        grads = torch.autograd.grad(layers.gated_linear_scan(*xs, coupled=coupled), xs, (dy, dh))
        _, err = R.scan(x, f, h0, None, coupled, dy, dh)
        for k, name in enumerate(("dx", "df", "dh0")):
            def value(e):
                args = [t.double() + (e * v[k] if i == k else 0) for i, t in enumerate((x, f, h0))]
                val, _ = R.scan(*args, None, coupled)
                return float((val["y"] * dy.double()).sum() + (val["h_last"] * dh.double()).sum())
            diff = (value(1e-6) - value(-1e-6)) / 2e-6
            got = float((grads[k].double() * v[k]).sum())
            allowed = float(((err[name] + R.rounding(grads[k].double(), torch.float32)) * v[k].abs()).sum()) + 1e-6 * (1 + abs(diff))
            assert abs(got - diff) <= allowed, (name, got, diff, allowed)


# ------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2049, 100003])
def test_dropout_values(layers, gpu, n, dtype):
    for p, seed, offset in ((0.1, 0, 0), (0.5, (1 << 63) + 12345, (1 << 40) + 7), (0.9, 99, 1 << 63)):
        x = rand((n,), n, dtype, gpu).requires_grad_()
        y = layers.counter_dropout(x, p, seed, offset)
        keep = R.keep_mask(n, p, seed, offset).to(gpu)
        scale = torch.tensor(R.keep_scale(p), dtype=torch.float32, device=gpu)
        assert torch.equal(y, torch.where(keep, x.float() * scale, 0.0).to(dtype))
        dy = rand((n,), n + 1, dtype, gpu)
        (dx,) = torch.autograd.grad(y, x, dy)
        assert torch.equal(dx, torch.where(keep, dy.float() * scale, 0.0).to(dtype))


def test_dropout_generator_known_answers():
    """The reference generator against the published test vectors of Philox4x32-10."""
    ones = 0xFFFFFFFF
    for ctr, key, want in (((0,) * 4, (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                           ((ones,) * 4, (ones, ones), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                            (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w[0]) for w in R.philox([[c] for c in ctr], key)) == want


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_residual_ends_and_views(layers, gpu, dtype):
    x, r = rand((41, 13), 1, dtype, gpu).requires_grad_(), rand((41, 13), 2, dtype, gpu).requires_grad_()
    y = layers.counter_dropout(x, 0.3, 5, 6, residual=r)
    keep = R.keep_mask(x.numel(), 0.3, 5, 6).view(x.shape).to(gpu)
    val = torch.where(keep, x.double() * R.keep_scale(0.3), 0.0) + r.double()
    R.check(y, val, 4 * R.U * (x.double().abs() * R.keep_scale(0.3) + r.double().abs()), "residual")
    dy = rand((41, 13), 3, dtype, gpu)
    dx, dr = torch.autograd.grad(y, (x, r), dy)
    assert torch.equal(dr, dy) and torch.equal(dx != 0, keep & (dy != 0))
    x = x.detach()
    assert torch.equal(layers.counter_dropout(x, 0.0, 1), x)
    assert float(layers.counter_dropout(x, 1.0, 1).abs().max()) == 0
    # a view with an odd base address, and one that is not contiguous: as their copies
    for v in (x.reshape(-1)[3:], x.t(), x[:, 1:6]):
        assert torch.equal(layers.counter_dropout(v, 0.3, 5, 6), layers.counter_dropout(v.clone(memory_format=torch.contiguous_format), 0.3, 5, 6))
    # what is dropped is 0, finite or not; what stays, stays
    bad = torch.full((1000,), float("nan"), dtype=dtype, device=gpu)
    y = layers.counter_dropout(bad, 0.5, 8)
    keep = R.keep_mask(1000, 0.5, 8, 0).to(gpu)
    assert torch.equal(torch.isnan(y), keep) and float(y[~keep].abs().max()) == 0


def test_dropout_mask_statistics(layers, gpu):
    """The share that stays over 2^22 elements is within 5 standard deviations, and so is the overlap of two offsets."""
    n, p = 1 << 22, 0.25
    x = torch.ones(n, device=gpu)
    a, b = (layers.counter_dropout(x, p, 3, o) != 0 for o in (0, 1))
    for share, want in ((a.double().mean(), 1 - p), ((a & b).double().mean(), (1 - p) ** 2)):
        assert abs(float(share) - want) < 5 * (want * (1 - want) / n) ** 0.5


# ------------------------------------------------------------------------------------ group norm
def norm_case(layers, gpu, shape, groups, dtype, act="silu", p=0.0, affine=True, shift=0.3, seed=0, eps=1e-5):
    N, C, H, W = shape
    x = rand((N, H, W, C), seed, dtype, gpu, 0.7, shift).permute(0, 3, 1, 2).requires_grad_()
    w = rand((C,), seed + 1, torch.float32, gpu, 0.3, 1.0).requires_grad_() if affine else None
    b = rand((C,), seed + 2, torch.float32, gpu, 0.3).requires_grad_() if affine else None
    dy = rand((N, H, W, C), seed + 3, dtype, gpu).permute(0, 3, 1, 2)
    y = layers.group_norm_act(x, groups, w, b, eps, act, p, seed=77, offset=seed)
    assert y.dtype == dtype and y.is_contiguous(memory_format=torch.channels_last)
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy)
    val, err = R.norm(x, groups, w, b, eps, act, p, 77, seed, dy)
    for k, v in zip(("y", "dx", "dw", "db"), (y,) + tuple(grads)):
        R.check(v, val[k], err[k], f"{k} {shape} G={groups} {dtype} {act} p={p}")
    with torch.no_grad():
        assert torch.equal(layers.group_norm_act(x, groups, w, b, eps, act, p, seed=77, offset=seed), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_types_and_activations(layers, gpu, p, act, dtype):
    norm_case(layers, gpu, (3, 32, 15, 12), 8, dtype, act, p)


@pytest.mark.parametrize("shape,groups", [((2, 1, 5, 3), 1), ((2, 3, 7, 5), 3), ((1, 6, 9, 11), 2), ((2, 20, 13, 17), 5), ((1, 24, 8, 8), 2),
                                          ((1, 10, 31, 3), 1), ((2, 512, 6, 5), 32), ((1, 300, 4, 4), 3), ((1, 2056, 3, 2), 8), ((1, 259, 5, 5), 7),
                                          ((1, 32, 1, 1), 4), ((1, 16, 1, 1), 16), ((4, 16, 64, 80), 4), ((1, 32, 128, 160), 8), ((300, 8, 3, 3), 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_shapes(layers, gpu, shape, groups, dtype):
    norm_case(layers, gpu, shape, groups, dtype)
    norm_case(layers, gpu, shape, groups, dtype, "relu", 0.2, seed=9)


@pytest.mark.parametrize("shape,groups,dtype", [((256, 32, 30, 24), 8, torch.float32), ((256, 32, 41, 40), 1, torch.bfloat16), ((640, 32, 23, 23), 8, torch.float16),
                                                ((530, 24, 30, 31), 3, torch.bfloat16), ((40, 512, 23, 24), 32, torch.float16), ((16, 32, 256, 257), 8, torch.bfloat16)])
def test_norm_beyond_the_caches(layers, gpu, shape, groups, dtype):
    """More than 20 MB in many small samples, where the choice between the forms is another one."""
    norm_case(layers, gpu, shape, groups, dtype, "silu")


def test_norm_without_affine_and_far_mean(layers, gpu):
    norm_case(layers, gpu, (2, 16, 20, 20), 4, torch.float32, affine=False)
    # the mean 300 deviations from 0: sums of squares around 0 would lose the variance
    norm_case(layers, gpu, (2, 16, 40, 40), 4, torch.float32, shift=200.0)
    # a constant group: variance 0, everything is the bias
    x = torch.full((1, 8, 6, 6), 3.0, device=gpu).contiguous(memory_format=torch.channels_last)
    b = torch.arange(8.0, device=gpu)
    y = layers.group_norm_act(x, 2, None, b)
    assert torch.equal(y, b.view(1, 8, 1, 1).expand(1, 8, 6, 6))


def test_norm_other_memory_orders(layers, gpu):
    x = rand((2, 12, 10, 14), 1, torch.float32, gpu)          # NCHW
    w = rand((12,), 2, torch.float32, gpu)
    y = layers.group_norm_act(x, 3, w, None, act="silu")
    z = layers.group_norm_act(x.contiguous(memory_format=torch.channels_last), 3, w, None, act="silu")
    assert torch.equal(y, z) and y.is_contiguous(memory_format=torch.channels_last)
    part = rand((2, 20, 14, 16), 3, torch.bfloat16, gpu).permute(0, 3, 1, 2)[:, 3:15]        # channels inside a wider row
    assert torch.equal(layers.group_norm_act(part, 3), layers.group_norm_act(part.contiguous(), 3))


def test_norm_nan_stays_in_its_group(layers, gpu):
    x = rand((2, 8, 9, 9), 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last)
    x[0, 1, 4, 4] = float("nan")
    for act in ("none", "relu", "silu"):
        bad = torch.isnan(layers.group_norm_act(x, 4, act=act))
        assert bad[0, :2].all() and int(bad.sum()) == 2 * 81


def test_norm_gradient_against_differences(layers, gpu):
    shape, G = (2, 6, 5, 4), 3
    x = rand(shape, 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last)
    w, b, dy = rand((6,), 2, torch.float32, gpu, 0.3, 1.0), rand((6,), 3, torch.float32, gpu), rand(shape, 4, torch.float32, gpu)
    v = [rand(t.shape, 5 + k, torch.float32, gpu).double() for k, t in enumerate((x, w, b))]
    leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layers.group_norm_act(leaves[0], G, leaves[1], leaves[2], act="silu", p=0.2, seed=4), leaves, dy)
    _, err = R.norm(x, G, w, b, 1e-5, "silu", 0.2, 4, 0, dy)
    for k, name in enumerate(("dx", "dw", "db")):
        def value(e):
            args = [t.double() + (e * v[k] if i == k else 0) for i, t in enumerate((x, w, b))]
            return float((R.norm(args[0], G, args[1], args[2], 1e-5, "silu", 0.2, 4, 0)[0]["y"] * dy.double()).sum())
        diff = (value(1e-6) - value(-1e-6)) / 2e-6
        got = float((grads[k].double() * v[k]).sum())
        allowed = float(((err[name] + R.rounding(grads[k].double(), torch.float32)) * v[k].abs()).sum()) + 1e-6 * (1 + abs(diff))
        assert abs(got - diff) <= allowed, (name, got, diff, allowed)


# ------------------------------------------------------------------------------------ together, streams, graphs
def block(layers, x, f, h0, w, b, offset):
    """recurrence -> norm + activation + dropout -> dropout onto the input: a recurrent block on [B, T, H, W, C]."""
    B, T, H, W, C = x.shape
    y, h = layers.gated_linear_scan(x, f, h0)
    z = layers.group_norm_act(y.flatten(0, 1).permute(0, 3, 1, 2), 4, w, b, act="silu", p=0.1, seed=3, offset=offset)
    z = z.permute(0, 2, 3, 1).reshape(x.shape)
    return layers.counter_dropout(z, 0.2, 4, offset, residual=x), h


def block_inputs(gpu, dtype, seed=0):
    shape = (2, 18, 6, 5, 16)
    t = [rand(shape, seed, dtype, gpu), rand(shape, seed + 1, dtype, gpu, 1.5, 2.0), rand((2, 6, 5, 16), seed + 2, torch.float32, gpu),
         rand((16,), seed + 3, torch.float32, gpu, 0.3, 1.0), rand((16,), seed + 4, torch.float32, gpu, 0.3)]
    return [v.requires_grad_() for v in t], rand(shape, seed + 5, dtype, gpu)


def test_block_against_the_references(layers, gpu):
    leaves, dy = block_inputs(gpu, torch.float32)
    x, f, h0, w, b = leaves
    out, _ = block(layers, *leaves, 11)
    grads = torch.autograd.grad(out, leaves, dy)
    # the same in float64 with autograd, masks from the reference generator
    xs = [t.detach().cpu().double().requires_grad_() for t in leaves]
    X, F, h, Wt, Bt = xs
    ys = []
    for t in range(18):
        s = torch.sigmoid(F[:, t])
        h = s * h + (1 - s) * X[:, t]
        ys.append(h)
    y = torch.stack(ys, 1).flatten(0, 1).permute(0, 3, 1, 2)
    z = torch.nn.functional.silu(torch.nn.functional.group_norm(y, 4, Wt, Bt)).permute(0, 2, 3, 1).reshape(X.shape)
    for p, seed in ((0.1, 3), (0.2, 4)):
        z = z * R.keep_mask(z.numel(), p, seed, 11).view(z.shape).double() * R.keep_scale(p)
    want = z + X
    ref = torch.autograd.grad(want, xs, dy.cpu().double())
    # (rel. 2-norm: a few hundred roundings of 2^-24 behind each value, most of which cancel)
    assert float((out.cpu().double() - want).norm() / want.norm()) < 2e-6
    for k, (g, r) in enumerate(zip(grads, ref)):
        assert float((g.cpu().double() - r).norm() / r.norm()) < 4e-6, k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_on_another_stream(layers, gpu, dtype):
    leaves, dy = block_inputs(gpu, dtype)
    want = block(layers, *leaves, 5)
    gw = torch.autograd.grad(want, leaves, (dy, torch.ones_like(want[1])))
    want = tuple(t.detach() for t in want)          # (no graph of the leaves from this stream stays alive)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [block(layers, *leaves, 5) for _ in range(3)]
        gs = [torch.autograd.grad(o, leaves, (dy, torch.ones_like(o[1]))) for o in outs]
    side.synchronize()
    for o, g in zip(outs, gs):
        assert all(torch.equal(p, q) for p, q in zip(o + tuple(g), want + tuple(gw)))


def test_block_captured_and_replayed(layers, gpu):
    """Forward and backward of the block in a graph whose dropout offset lives on the device and advances with every
    replay: each replay equals the eager pass of that offset, with eager work and synchronisations in between."""
    leaves, dy = block_inputs(gpu, torch.bfloat16)
    offset = torch.zeros(1, dtype=torch.int64, device=gpu)

    def step():
        out, h = block(layers, *leaves, offset)
        offset.add_(1)                                  # (before the backward pass: it keeps the offset the forward used)
        return (out, h) + torch.autograd.grad((out, h), leaves, (dy, torch.ones_like(h)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    offset.fill_(100)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    assert int(offset) == 100
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert int(offset) == 101 + k
        out, h = block(layers, *leaves, 100 + k)
        want = (out, h) + torch.autograd.grad((out, h), leaves, (dy, torch.ones_like(h)))
        for i, (p, q) in enumerate(zip(got, want)):
            assert torch.equal(p, q), (k, i)
        torch.randn(1000, device=gpu).sum().item()


def test_capture_beside_a_live_eager_graph_is_refused(layers, gpu):
    """Outputs of an eager pass over the same leaves are alive when a training pass is captured: an error at the first
    operator; once they are dropped the capture works."""
    def calls(m):
        x = rand((2, 16, 8, 8), 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last)
        return {"norm": lambda: layers.group_norm_act(x, 4, m["w"], m["b"]),
                "scan": lambda: layers.gated_linear_scan(m["s"], m["s"])[0],
                "dropout": lambda: layers.counter_dropout(m["s"], 0.5, 1)}
    leaves = {"w": torch.ones(16, device=gpu, requires_grad=True), "b": torch.zeros(16, device=gpu, requires_grad=True),
              "s": rand((2, 20, 12), 3, torch.float32, gpu).requires_grad_()}
    for name, call in calls(leaves).items():
        call()                                            # (its graph is dropped with it)
        want = torch.autograd.grad(call().sum(), [t for t in leaves.values()], allow_unused=True)
        alive = call()
        with pytest.raises(RuntimeError, match="earlier pass over the same leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()                                        # (no gradients, no difficulty)
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call().sum(), [t for t in leaves.values()], allow_unused=True)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            for p, q in zip(got, want):
                assert (p is None and q is None) or torch.equal(p, q), name


def test_modules(layers, gpu):
    m = layers.GroupNormAct(4, 16, act="relu", p=0.3, seed=9).to(gpu)
    x = rand((2, 16, 8, 8), 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last)
    a, b = m(x), m(x)
    assert not torch.equal(a, b) and int(m.offset) == 2
    assert torch.equal(a, layers.group_norm_act(x, 4, m.weight, m.bias, act="relu", p=0.3, seed=9, offset=0))
    m.eval()
    assert torch.equal(m(x), layers.group_norm_act(x, 4, m.weight, m.bias, act="relu")) and int(m.offset) == 2
    d = layers.CounterDropout(0.5, seed=2).to(gpu)
    assert torch.equal(d(x), layers.counter_dropout(x, 0.5, 2, 0)) and torch.equal(d(x, x), layers.counter_dropout(x, 0.5, 2, 1, residual=x))
    d.eval()
    assert d(x) is x


def test_empty_sizes(layers, gpu):
    for shape in ((0, 5, 4), (3, 0, 4), (2, 5, 0)):
        x = torch.zeros(shape, device=gpu, requires_grad=True)
        f = torch.zeros(shape, device=gpu, requires_grad=True)
        h0 = torch.randn(shape[0], shape[2], device=gpu).requires_grad_()
        y, h = layers.gated_linear_scan(x, f, h0)
        assert y.shape == x.shape and torch.equal(h, h0)
        dx, df, dh = torch.autograd.grad((y, h), (x, f, h0), (torch.zeros_like(y), torch.ones_like(h)))
        assert dx.shape == x.shape and torch.equal(dh, torch.ones_like(h))
    assert layers.counter_dropout(torch.zeros(0, 3, device=gpu), 0.5, 1).shape == (0, 3)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device=gpu, requires_grad=True)
        w = torch.ones(8, device=gpu, requires_grad=True)
        y = layers.group_norm_act(x, 2, w, None)
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert y.shape == x.shape and dx.shape == x.shape and float(dw.abs().max()) == 0


def test_second_derivatives_are_refused(layers, gpu):
    x = rand((1, 4, 8), 1, torch.float32, gpu).requires_grad_()
    y, _ = layers.gated_linear_scan(x, x)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(layers, gpu):
    x = torch.zeros(2, 3, 4, device=gpu)
    cases = [
        (ValueError, lambda: layers.gated_linear_scan(x, x[:, :2])),
        (ValueError, lambda: layers.gated_linear_scan(x[0, 0], x[0, 0])),
        (TypeError, lambda: layers.gated_linear_scan(x, x.half())),
        (TypeError, lambda: layers.gated_linear_scan(x.double(), x.double())),
        (TypeError, lambda: layers.gated_linear_scan(x, None)),
        (TypeError, lambda: layers.gated_linear_scan(x, x, torch.zeros(2, 4, device=gpu, dtype=torch.bfloat16))),
        (ValueError, lambda: layers.gated_linear_scan(x, x, torch.zeros(2, 5, device=gpu))),
        (RuntimeError, lambda: layers.gated_linear_scan(x, x, torch.zeros(2, 4))),
        (TypeError, lambda: layers.gated_linear_scan(x, x, lengths=torch.zeros(2, device=gpu, dtype=torch.int64))),
        (ValueError, lambda: layers.gated_linear_scan(x, x, lengths=torch.zeros(3, device=gpu, dtype=torch.int32))),
        (ValueError, lambda: layers.gated_linear_step(x[:, 0], x[:, 0], torch.zeros(4, 2, device=gpu).t(), inplace=True)),
        (ValueError, lambda: layers.counter_dropout(x, 1.5, 1)),
        (ValueError, lambda: layers.counter_dropout(x, float("nan"), 1)),
        (ValueError, lambda: layers.counter_dropout(x, 0.5, -1)),
        (ValueError, lambda: layers.counter_dropout(x, 0.5, 1 << 64)),
        (ValueError, lambda: layers.counter_dropout(x, 0.5, 1, residual=x[0])),
        (TypeError, lambda: layers.counter_dropout(x, 0.5, 1, offset=torch.zeros(1, device=gpu))),
        (ValueError, lambda: layers.counter_dropout(x, 0.5, 1, offset=torch.zeros(2, device=gpu, dtype=torch.int64))),
        (ValueError, lambda: layers.group_norm_act(x, 1)),
        (ValueError, lambda: layers.group_norm_act(x[None], 4)),
        (ValueError, lambda: layers.group_norm_act(x[None], 0)),
        (ValueError, lambda: layers.group_norm_act(x[None], 1, act="gelu")),
        (ValueError, lambda: layers.group_norm_act(x[None], 1, torch.ones(3, device=gpu))),
        (TypeError, lambda: layers.group_norm_act(x[None], 1, torch.ones(2, device=gpu).half())),
        (ValueError, lambda: layers.group_norm_act(x[None], 1, eps=-1.0)),
    ]
    for k, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {k} was not refused")


def test_offsets_beyond_32_bits(layers, gpu):
    """More than 2^31 elements: the ends of the tensors against the same calls on their slices."""
    n = (1 << 31) + 1003
    x = torch.ones(n, dtype=torch.bfloat16, device=gpu)
    y = layers.counter_dropout(x, 0.5, 77, 5)
    tail = n - 4096 - n % 8
    j = R.np.arange(tail // 8, (n + 7) // 8, dtype=R.np.uint64)
    w = R.philox([j & R.np.uint64(0xFFFFFFFF), j >> R.np.uint64(32), R.np.full_like(j, 5), R.np.full_like(j, 0)], (77, 0))
    u16 = R.np.stack([w[i // 2] >> R.np.uint64(16 * (i % 2)) & R.np.uint64(0xFFFF) for i in range(8)], 1).reshape(-1)[:n - tail]
    assert torch.equal(y[tail:] != 0, torch.from_numpy(u16 >= 32768).to(gpu))
    del x, y
    D = (1 << 31) + 24
    x = torch.full((1, 2, D), 0.5, dtype=torch.bfloat16, device=gpu)
    f = torch.zeros(1, 2, D, dtype=torch.bfloat16, device=gpu)
    x[0, :, -100:], f[0, :, -100:] = rand((2, 100), 1, torch.bfloat16, gpu), rand((2, 100), 2, torch.bfloat16, gpu)
    y, h = layers.gated_linear_scan(x, f)
    a, b = layers.gated_linear_scan(x[:, :, -100:].contiguous(), f[:, :, -100:].contiguous())
    assert torch.equal(y[:, :, -100:], a) and torch.equal(h[:, -100:], b) and float(h[0, 0]) == 0.375
    del x, f, y, h
    torch.cuda.empty_cache()
    shape = (3, 4700, 4800, 32)
    x = torch.empty(shape, dtype=torch.bfloat16, device=gpu).normal_().permute(0, 3, 1, 2)
    y = layers.group_norm_act(x, 4, act="relu")
    assert torch.equal(y[2:], layers.group_norm_act(x[2:], 4, act="relu"))
    z = layers.group_norm_act(x, 4, act="relu", p=0.5, seed=1)[2].permute(1, 2, 0).reshape(-1)
    keep = layers.counter_dropout(torch.ones(3 * 4700 * 4800 * 32, dtype=torch.bfloat16, device=gpu), 0.5, 1)[-z.numel():] != 0
    assert float(z[~keep].abs().max()) == 0 and torch.equal(z[keep], (y[2].permute(1, 2, 0).reshape(-1)[keep].float() * 2).to(torch.bfloat16))


def test_large_tensors_streamed_past_the_caches(layers, gpu):
    """Sizes at which inputs are read past the caches: the bits of the calls that keep them there."""
    x, f = rand((1, 10, 6000008), 1, torch.bfloat16, gpu), rand((1, 10, 6000008), 2, torch.bfloat16, gpu)
    y, h = layers.gated_linear_scan(x, f)
    g = x.detach().requires_grad_()                       # (a training pass does not stream)
    y2, h2 = layers.gated_linear_scan(g, f)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    # dropout: fp32 tensors are never streamed; same mask, the same product, rounded once
    out = layers.counter_dropout(x, 0.3, 5, 6, residual=f)
    assert torch.equal(out, layers.counter_dropout(x.float(), 0.3, 5, 6, residual=f.float()).bfloat16())
    out = layers.counter_dropout(x, 0.3, 5, 6)
    assert torch.equal(out, layers.counter_dropout(x.float(), 0.3, 5, 6).bfloat16())
