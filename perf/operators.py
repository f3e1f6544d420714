"""The operators around the recurrence that are measured: the gated linear recurrence, group norm with an activation
(channels last), and dropout from a counter-based generator; their cases, plain forms and 64-bit values.

``own`` false: the plain form, elementary torch operations in 32 bits, rounded once.  ``own`` true: the calls a user
makes of ``pl_convlstm_gan_amd.layers``.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MASK32 = 0xFFFFFFFF


# --------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one frame of the 15 x 12 basin grid with 32 channels arrives at a serving program: latency
        dict(name="scan step basin", op="scan_step", dtype="float32", B=1, D=15 * 12 * 32, coupled=True),
        # inference over the 128 x 128, T = 10, batch 8 workload, 32 hidden channels
        dict(name="scan forward 128x128", op="scan_forward", dtype="bfloat16", B=8, T=10, D=128 * 128 * 32, coupled=True, ragged=False),
        # a training pass over the per-GPU shard of the 256 x 256 workload (B = 4, T = 10, 32 channels)
        dict(name="scan train 256x256", op="scan_train", dtype="bfloat16", B=4, T=10, D=256 * 256 * 32, coupled=True, ragged=False),
        # gauge series: ten years of days, 48 features per step, batch 8
        dict(name="scan train gauge series", op="scan_train", dtype="float32", B=8, T=3653, D=48, coupled=True, ragged=False),
        # long series of different lengths in one padded batch
        dict(name="scan forward long ragged", op="scan_forward", dtype="bfloat16", B=4, T=32768, D=96, coupled=False, ragged=True),
        # the five frames of one basin sample: latency
        dict(name="norm forward basin", op="norm_forward", dtype="float32", N=5, C=32, G=8, H=15, W=12, act="silu", p=0.0),
        # inference over the 40 frames of the 256 x 256 shard
        dict(name="norm forward 256x256", op="norm_forward", dtype="bfloat16", N=40, C=32, G=8, H=256, W=256, act="relu", p=0.0),
        # training over the 80 frames of the 128 x 128 workload, dropout in the same pass
        dict(name="norm train 128x128 dropout", op="norm_train", dtype="bfloat16", N=80, C=32, G=4, H=128, W=128, act="silu", p=0.1),
        # wide features on a coarse grid
        dict(name="norm train wide", op="norm_train", dtype="float16", N=8, C=512, G=32, H=32, W=32, act="silu", p=0.0),
        # a width that is no multiple of eight on an odd grid
        dict(name="norm train odd", op="norm_train", dtype="float32", N=16, C=20, G=5, H=61, W=47, act="relu", p=0.0),
        # dropout on the features of the 256 x 256 shard, both directions
        dict(name="dropout train 256x256", op="dropout_train", dtype="bfloat16", n=40 * 32 * 256 * 256, p=0.1, residual=False),
        # dropout added to a skip connection, odd size
        dict(name="dropout residual odd", op="dropout_forward", dtype="float16", n=1000003, p=0.25, residual=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan_step", "scan_forward", "scan_forward", "scan_train", "scan_train", "norm_forward", "norm_train",
                     "norm_train", "dropout_forward", "dropout_train"])
    dtype = rng.choice(sorted(DTYPES))
    most = 1 << 25                      # elements of a drawn case's largest tensor
    if op == "scan_step":
        B = _log_int(rng, 1, 64)
        return dict(op=op, dtype=dtype, B=B, D=_log_int(rng, 16, (1 << 22) // B), coupled=rng.random() < 0.7)
    if op.startswith("scan"):
        B = _log_int(rng, 1, 32)
        T = _log_int(rng, 2, 16384)
        D = _log_int(rng, 8, max(9, min(1 << 20, most // (B * T))))
        return dict(op=op, dtype=dtype, B=B, T=T, D=D, coupled=rng.random() < 0.7, ragged=rng.random() < 0.3)
    if op.startswith("norm"):
        G = rng.choice([1, 2, 3, 4, 8, 16, 32])
        C = G * _log_int(rng, 1, 512 // G)
        H, W = _log_int(rng, 4, 256), _log_int(rng, 4, 256)
        N = _log_int(rng, 1, max(2, min(320, most // (C * H * W))))
        return dict(op=op, dtype=dtype, N=N, C=C, G=G, H=H, W=W, act=rng.choice(["none", "relu", "silu"]),
                    p=rng.choice([0.0, 0.0, round(rng.uniform(0.02, 0.6), 3)]))
    return dict(op=op, dtype=dtype, n=_log_int(rng, 100, most), p=round(rng.uniform(0.02, 0.9), 3), residual=rng.random() < 0.5)


def work(case):
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    op = case["op"]
    if op == "scan_step":
        n = case["B"] * case["D"]
        return {"bytes": n * (3 * e + 8), "flops": 8 * n}
    if op.startswith("scan"):
        n, s = case["B"] * case["T"] * case["D"], case["B"] * case["D"]
        if op == "scan_forward":
            return {"bytes": 3 * n * e + 8 * s, "flops": 8 * n}
        return {"bytes": (3 + 5) * n * e + 4 * 4 * s, "flops": 24 * n}       # x, f, y; then x, f, dy, dx, df; the four states
    if op.startswith("norm"):
        n = case["N"] * case["C"] * case["H"] * case["W"]
        if op == "norm_forward":
            return {"bytes": 2 * n * e + 8 * case["C"], "flops": 10 * n}
        return {"bytes": (2 + 3) * n * e + 16 * case["C"], "flops": 30 * n}
    passes = 1 if op == "dropout_forward" else 2
    return {"bytes": (2 * passes + (1 if case["residual"] else 0)) * case["n"] * e, "flops": 3 * case["n"] * passes}


# --------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)

    s = {"case": case, "op": case["op"]}
    if case["op"].startswith("scan"):
        B, D, step = case["B"], case["D"], case["op"] == "scan_step"
        shape = (B, D) if step else (B, case["T"], D)
        train = case["op"] == "scan_train"
        s["x"] = normal(*shape).requires_grad_(train)
        s["f"] = normal(*shape, scale=1.5, shift=2.0).requires_grad_(train)      # forget gates mostly open, some far open
        s["h0"] = normal(B, D, dtype=torch.float32).requires_grad_(train)
        s["lengths"] = None
        if not step and case["ragged"]:
            n = torch.randint(1, case["T"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            n[0] = case["T"]
            if B > 2:
                n[B // 2] = 0                                                    # a sample with no step at all
            s["lengths"] = n
        if train:
            s["dy"] = normal(*shape)
            s["dh"] = normal(B, D, dtype=torch.float32)
    elif case["op"].startswith("norm"):
        N, C, H, W = case["N"], case["C"], case["H"], case["W"]
        train = case["op"] == "norm_train"
        nhwc = lambda **kw: normal(N, H, W, C, **kw).permute(0, 3, 1, 2)  # noqa: E731
        s["x"] = nhwc(scale=0.7, shift=0.3).requires_grad_(train)
        s["w"] = normal(C, dtype=torch.float32, scale=0.2, shift=1.0).requires_grad_(train)
        s["b"] = normal(C, dtype=torch.float32, scale=0.2).requires_grad_(train)
        if train:
            s["dy"] = nhwc()
    else:
        train = case["op"] == "dropout_train"
        s["x"] = normal(case["n"]).requires_grad_(train)
        s["r"] = normal(case["n"]).requires_grad_(train) if case["residual"] else None
        if train:
            s["dy"] = normal(case["n"])
    s["seed"] = int(torch.randint(0, 1 << 62, (1,), generator=g, device="cuda"))
    s["offset"] = int(torch.randint(0, 1 << 40, (1,), generator=g, device="cuda"))
    return s


# --------------------------------------------------------------------------------------------------- plain forms
def _scan(a, b):
    """h[:, t] = a[:, t] h[:, t - 1] + b[:, t] (h before the first step is 0) by doubling the reach of each step."""
    d, T = 1, a.shape[1]
    while d < T:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _plain_scan(s):
    c, dt = s["case"], s["x"].dtype
    x, f, h0 = (s[k].detach().float() for k in ("x", "f", "h0"))
    a, q = torch.sigmoid(f), torch.sigmoid(-f)
    if c["op"] == "scan_step":
        h = a * h0 + (q * x if c["coupled"] else x)
        return h.to(dt), h
    b = q * x if c["coupled"] else x
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(c["T"], device=x.device)[None, :] < s["lengths"][:, None])[:, :, None]
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)       # behind its length a sample's state stands still
    b = torch.cat([b[:, :1] + a[:, :1] * h0[:, None], b[:, 1:]], 1)
    h = _scan(a, b)
    y = (h if live is None else torch.where(live, h, 0.0)).to(dt)
    last = h[:, -1].clone()
    if c["op"] == "scan_forward":
        return y, last
    dy, dh = s["dy"].float(), s["dh"]
    if live is not None:
        dy = torch.where(live, dy, 0.0)
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + dh[:, None]], 1)
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)            # g_t = dy_t + a_{t+1} g_{t+1}
    g = _scan(nxt.flip(1), dy.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    dx = g * q if c["coupled"] else g
    df = g * (before - x if c["coupled"] else before) * torch.sigmoid(f) * q
    if live is not None:
        dx, df = torch.where(live, dx, 0.0), torch.where(live, df, 0.0)
    return y, last, dx.to(dt), df.to(dt), a[:, 0] * g[:, 0]


def _philox_keep(n, p, seed, offset, device):
    """keep[e]: the 16-bit value e of Philox4x32-10 (counter = (e >> 3, offset), key = seed) is at least round(p 2^16)."""
    j = torch.arange((n + 7) // 8, device=device, dtype=torch.int64)
    c0, c1 = j & MASK32, j >> 32
    c2, c3 = torch.full_like(j, offset & MASK32), torch.full_like(j, (offset >> 32) & MASK32)
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    for _ in range(10):
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((m1 >> 32) & MASK32) ^ c1 ^ k0, m1 & MASK32, ((m0 >> 32) & MASK32) ^ c3 ^ k1, m0 & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    words = torch.stack([c0, c1, c2, c3], 1)
    u16 = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return u16 >= _threshold(p)


def _threshold(p):
    return int(math.floor(p * 65536.0 + 0.5))


def _scale(p):
    return 65536.0 / (65536.0 - _threshold(p))


def _plain_dropout(v, p, seed, offset):
    keep = _philox_keep(v.numel(), p, seed, offset, v.device).view(v.shape)
    return torch.where(keep, v * float(np.float32(_scale(p))), 0.0), keep


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    x = s["x"].detach().float()
    w, b = (s[k].detach()[None, :, None, None] for k in ("w", "b"))
    xg = x.unflatten(1, (c["G"], -1))
    d = xg - xg.mean((2, 3, 4), keepdim=True)
    r = torch.rsqrt((d * d).mean((2, 3, 4), keepdim=True) + 1e-5)
    xh = (d * r).flatten(1, 2)
    z = xh * w + b
    y = z if c["act"] == "none" else torch.relu(z) if c["act"] == "relu" else z * torch.sigmoid(z)
    keep = None
    if c["p"] > 0:
        y, keep = _plain_dropout(y.permute(0, 2, 3, 1), c["p"], s["seed"], s["offset"])     # counted in memory order
        y, keep = y.permute(0, 3, 1, 2), keep.permute(0, 3, 1, 2)
    if c["op"] == "norm_forward":
        return y.to(dt)
    dz = s["dy"].float()
    if keep is not None:
        dz = torch.where(keep, dz * float(np.float32(_scale(c["p"]))), 0.0)
    if c["act"] == "relu":
        dz = torch.where(z > 0, dz, 0.0)
    elif c["act"] == "silu":
        sg = torch.sigmoid(z)
        dz = dz * sg * (1 + z * (1 - sg))
    db, dw = dz.sum((0, 2, 3)), (dz * xh).sum((0, 2, 3))
    t, xhg = (dz * w).unflatten(1, (c["G"], -1)), xh.unflatten(1, (c["G"], -1))
    dx = r * (t - t.mean((2, 3, 4), keepdim=True) - xhg * (t * xhg).mean((2, 3, 4), keepdim=True))
    return y.to(dt), dx.flatten(1, 2).to(dt), dw, db


def run(state):
    s, c, op = state, state["case"], state["op"]
    if own:
        from pl_convlstm_gan_amd import layers

        if op == "scan_step":
            return layers.gated_linear_step(s["x"], s["f"], s["h0"], coupled=c["coupled"])
        if op == "scan_forward":
            return layers.gated_linear_scan(s["x"], s["f"], s["h0"], lengths=s["lengths"], coupled=c["coupled"])
        if op == "scan_train":
            y, last = layers.gated_linear_scan(s["x"], s["f"], s["h0"], lengths=s["lengths"], coupled=c["coupled"])
            return (y, last) + torch.autograd.grad((y, last), (s["x"], s["f"], s["h0"]), (s["dy"], s["dh"]))
        if op.startswith("norm"):
            y = layers.group_norm_act(s["x"], c["G"], s["w"], s["b"], eps=1e-5, act=c["act"], p=c["p"], seed=s["seed"],
                                      offset=s["offset"])
            return y if op == "norm_forward" else (y,) + torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        y = layers.counter_dropout(s["x"], c["p"], s["seed"], offset=s["offset"], residual=s["r"])
        if op == "dropout_forward":
            return y
        leaves = (s["x"],) if s["r"] is None else (s["x"], s["r"])
        return (y,) + torch.autograd.grad(y, leaves, s["dy"])
    if op.startswith("scan"):
        return _plain_scan(s)
    if op.startswith("norm"):
        return _plain_norm(s)
    y, keep = _plain_dropout(s["x"].detach().float(), c["p"], s["seed"], s["offset"])
    y = y if s["r"] is None else y + s["r"].detach().float()
    if op == "dropout_forward":
        return y.to(s["x"].dtype)
    dx = torch.where(keep, s["dy"].float() * float(np.float32(_scale(c["p"]))), 0.0).to(s["x"].dtype)
    return (y.to(s["x"].dtype), dx) if s["r"] is None else (y.to(s["x"].dtype), dx, s["dy"])


# --------------------------------------------------------------------------------------------------- 64-bit values
def _exact_scan(s):
    c = s["case"]
    x, f, h = (s[k].detach().double() for k in ("x", "f", "h0"))
    if c["op"] == "scan_step":
        x, f = x[:, None], f[:, None]
    B, T, D = x.shape
    n = [T] * B if s["lengths"] is None else [int(v) for v in s["lengths"]]
    gate = lambda t: 1.0 / (1.0 + torch.exp(-f[:, t]))  # noqa: E731
    alive = torch.tensor(n, device=x.device)[:, None]
    ys, before = torch.zeros(B, T, D, dtype=torch.float64, device=x.device), []
    train = c["op"] == "scan_train"
    hs = torch.empty(B, T, D, dtype=torch.float64, device=x.device) if train else None
    for t in range(T):
        if train:
            hs[:, t] = h
        a = gate(t)
        new = a * h + ((1.0 - a) * x[:, t] if c["coupled"] else x[:, t])
        if s["lengths"] is None:
            h = new
            ys[:, t] = h
        else:
            on = t < alive
            h = torch.where(on, new, h)
            ys[:, t] = torch.where(on, h, 0.0)
    if c["op"] == "scan_step":
        return ys[:, 0], h
    if not train:
        return ys, h
    last, dy, g = h, s["dy"].double(), s["dh"].double()
    dx, df = torch.zeros_like(ys), torch.zeros_like(ys)
    for t in range(T - 1, -1, -1):              # g: the gradient of the state behind step t
        a = gate(t)
        on = t < alive
        full = g + dy[:, t]
        if c["coupled"]:
            dx[:, t] = torch.where(on, full * (1.0 - a), 0.0)
            df[:, t] = torch.where(on, full * (hs[:, t] - x[:, t]) * a * (1.0 - a), 0.0)
        else:
            dx[:, t] = torch.where(on, full, 0.0)
            df[:, t] = torch.where(on, full * hs[:, t] * a * (1.0 - a), 0.0)
        g = torch.where(on, full * a, g)
    return ys, last, dx, df, g


def _exact_keep(n, p, seed, offset, device):
    """The generator once more, on the host in unsigned 64-bit integers."""
    out = np.empty((n + 7) // 8 * 8, dtype=bool)
    low, s32 = np.uint64(MASK32), np.uint64(32)
    piece = 1 << 20
    for at in range(0, (n + 7) // 8, piece):
        j = np.arange(at, min(at + piece, (n + 7) // 8), dtype=np.uint64)
        ctr = [j & low, j >> s32, np.full_like(j, offset & MASK32), np.full_like(j, offset >> 32)]
        key = [seed & MASK32, seed >> 32]
        for _ in range(10):
            lo_hi = [(np.uint64(m) * v & low, np.uint64(m) * v >> s32) for m, v in ((0xD2511F53, ctr[0]), (0xCD9E8D57, ctr[2]))]
            (l0, h0), (l1, h1) = lo_hi
            ctr = [h1 ^ ctr[1] ^ np.uint64(key[0]), l1, h0 ^ ctr[3] ^ np.uint64(key[1]), l0]
            key = [(key[0] + 0x9E3779B9) & MASK32, (key[1] + 0xBB67AE85) & MASK32]
        limit = math.floor(p * 65536.0 + 0.5)
        for k in range(8):
            out[at * 8 + k:(at + len(j)) * 8:8] = ((ctr[k // 2] >> np.uint64(16 * (k % 2))) & np.uint64(0xFFFF)) >= limit
    return torch.from_numpy(out[:n]).to(device)


def _exact_norm(s):
    c = s["case"]
    N, C, G, H, W = (c[k] for k in ("N", "C", "G", "H", "W"))
    rows = lambda t: t.detach().double().permute(0, 2, 3, 1).reshape(N, H * W, G, C // G)  # noqa: E731
    x, w, b = rows(s["x"]), s["w"].detach().double().view(G, C // G), s["b"].detach().double().view(G, C // G)
    var, mu = torch.var_mean(x, dim=(1, 3), unbiased=False, keepdim=True)
    inv = 1.0 / torch.sqrt(var + 1e-5)
    xh = (x - mu) * inv
    z = xh * w + b
    sg = 1.0 / (1.0 + torch.exp(-z))
    y, slope = {"none": (z, None), "relu": (z.clamp(min=0), (z > 0).double()), "silu": (z * sg, sg + z * sg * (1 - sg))}[c["act"]]
    factor = None
    if c["p"] > 0:
        limit = math.floor(c["p"] * 65536.0 + 0.5)
        factor = _exact_keep(x.numel(), c["p"], s["seed"], s["offset"], x.device).double().view(x.shape) * (65536.0 / (65536.0 - limit))
        y = y * factor
    back = lambda t: t.reshape(N, H, W, C).permute(0, 3, 1, 2)  # noqa: E731
    if c["op"] == "norm_forward":
        return back(y)
    dz = rows(s["dy"])
    dz = dz if factor is None else dz * factor
    dz = dz if slope is None else dz * slope
    m = H * W * (C // G)
    t = dz * w
    dx = inv * (t - t.sum((1, 3), keepdim=True) / m - xh * ((t * xh).sum((1, 3), keepdim=True) / m))
    return back(y), back(dx), (dz * xh).sum((0, 1)).reshape(C), dz.sum((0, 1)).reshape(C)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("scan"):
        return _exact_scan(s)
    if case["op"].startswith("norm"):
        return _exact_norm(s)
    limit = math.floor(case["p"] * 65536.0 + 0.5)
    factor = _exact_keep(case["n"], case["p"], s["seed"], s["offset"], "cuda").double() * (65536.0 / (65536.0 - limit))
    y = s["x"].detach().double() * factor
    y = y if s["r"] is None else y + s["r"].detach().double()
    if case["op"] == "dropout_forward":
        return y
    dx = s["dy"].double() * factor
    return (y, dx) if s["r"] is None else (y, dx, s["dy"].double())
