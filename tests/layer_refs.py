"""64-bit references of the layer operators, with a bound on how far an fp32 evaluation may be from them.

u = 2^-24 is half a step of fp32.  Each elementary operation of a kernel is off by at most a few u of its result (the
exponential, the reciprocal and their product by at most 8 u together); the bounds below follow the operations and
allow 16 u per step of the recurrence, 32 u for a normalised value, 64 u of the sum of absolute values for a sum (a sum of
n terms in a tree of depth log2 n, with at most a few dozen terms added in sequence at each level).  A result that
leaves in a 16-bit type is off by half a step of that type on top (torch.finfo(t).eps / 2, relative; half the smallest
subnormal near 0)."""
import numpy as np
import torch

U = 2.0 ** -24


def rounding(value, dtype):
    fi = torch.finfo(dtype)
    return value.abs() * (fi.eps / 2) + fi.smallest_normal * fi.eps / 2


def scan(x, f, h0, lengths, coupled, dy=None, dh=None):
    """Everything on the CPU in float64: ({name: value}, {name: bound before the final rounding})."""
    dev = x.device
    x, f = x.detach().cpu().double(), f.detach().cpu().double()
    B, T = x.shape[:2]
    h = torch.zeros(x.shape[:1] + x.shape[2:], dtype=torch.float64) if h0 is None else h0.detach().cpu().double()
    n = torch.full((B,), T) if lengths is None else lengths.cpu().clamp(0, T).long()
    alive = lambda t: (t < n).view((B,) + (1,) * (x.dim() - 2))  # noqa: E731
    E = torch.zeros_like(h)
    y, Ey = torch.zeros_like(x), torch.zeros_like(x)
    before, Eb = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        s = torch.sigmoid(f[:, t])
        before[:, t], Eb[:, t] = h, E
        new = s * h + ((1 - s) * x[:, t] if coupled else x[:, t])
        En = s * E + 16 * U * (h.abs() + x[:, t].abs())
        on = alive(t)
        h, E = torch.where(on, new, h), torch.where(on, En, E)
        y[:, t], Ey[:, t] = torch.where(on, h, 0.0), torch.where(on, E, 0.0)
    val, err = {"y": y, "h_last": h}, {"y": Ey, "h_last": E}
    if dy is not None or dh is not None:
        dy = torch.zeros_like(x) if dy is None else dy.cpu().double()
        g = torch.zeros_like(h) if dh is None else dh.cpu().double()
        Eg = torch.zeros_like(h)
        dx, df, Ex, Ef = (torch.zeros_like(x) for _ in range(4))
        for t in range(T - 1, -1, -1):
            s = torch.sigmoid(f[:, t])
            q, on = torch.sigmoid(-f[:, t]), alive(t)
            full, Efull = g + dy[:, t], Eg + 2 * U * (g.abs() + dy[:, t].abs())
            m = before[:, t] - x[:, t] if coupled else before[:, t]
            Em = Eb[:, t] + 2 * U * (before[:, t].abs() + (x[:, t].abs() if coupled else 0))
            k = q if coupled else torch.ones_like(q)
            dx[:, t] = torch.where(on, full * k, 0.0)
            df[:, t] = torch.where(on, full * m * s * q, 0.0)
            Ex[:, t] = torch.where(on, k * (Efull + 16 * U * full.abs()), 0.0)
            Ef[:, t] = torch.where(on, s * q * (Efull * m.abs() + full.abs() * (Em + 32 * U * m.abs())), 0.0)
            g, Eg = torch.where(on, s * full, g), torch.where(on, s * (Efull + 16 * U * full.abs()), Eg)
        val.update(dx=dx, df=df, dh0=g)
        err.update(dx=Ex, df=Ef, dh0=Eg)
    return {k: v.to(dev) for k, v in val.items()}, {k: v.to(dev) for k, v in err.items()}


def _linear(a, b):
    """h[:, t] = a[:, t] h[:, t - 1] + b[:, t], h before the first step 0, by doubling the reach of each step."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def scan_long(x, f, h0, lengths, coupled, dy, dh):
    """scan() for sequences of which a loop over the steps takes too long: values and bounds are linear recurrences all."""
    dev = x.device
    x, f, h0, dy, dh = (t.detach().cpu().double() for t in (x, f, h0, dy, dh))
    B, T = x.shape[:2]
    n = torch.full((B,), T) if lengths is None else lengths.cpu().clamp(0, T).long()
    on = (torch.arange(T)[None] < n[:, None]).view((B, T) + (1,) * (x.dim() - 2))
    zero = torch.zeros((), dtype=torch.float64)
    s, q = torch.sigmoid(f), torch.sigmoid(-f)
    a = torch.where(on, s, 1.0)
    start = lambda b, v: torch.cat([b[:, :1] + a[:, :1] * v[:, None], b[:, 1:]], 1)  # noqa: E731
    h = _linear(a, start(torch.where(on, q * x if coupled else x, zero), h0))
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    E = _linear(a, torch.where(on, 16 * U * (before.abs() + x.abs()), zero))
    Eb = torch.cat([torch.zeros_like(E[:, :1]), E[:, :-1]], 1)
    back = lambda b: _linear(a.flip(1), b.flip(1)).flip(1)  # noqa: E731
    behind = lambda c, last: torch.cat([c[:, 1:], last[:, None]], 1)  # noqa: E731
    inner = torch.where(on, a * dy, zero)
    g = back(torch.cat([inner[:, :-1], inner[:, -1:] + a[:, -1:] * dh[:, None]], 1))          # what a step passes to the one in front of it
    full = behind(g, dh) + dy
    step = 2 * U * (behind(g, dh).abs() + dy.abs())
    Eg = back(torch.where(on, a * (step + 16 * U * full.abs()), zero))
    Efull = behind(Eg, torch.zeros_like(dh)) + step
    m = before - x if coupled else before
    Em = Eb + 2 * U * (before.abs() + (x.abs() if coupled else 0))
    k = q if coupled else torch.ones_like(q)
    val = {"y": torch.where(on, h, zero), "h_last": h[:, -1], "dx": torch.where(on, full * k, zero), "df": torch.where(on, full * m * s * q, zero), "dh0": g[:, 0]}
    err = {"y": torch.where(on, E, zero), "h_last": E[:, -1], "dx": torch.where(on, k * (Efull + 16 * U * full.abs()), zero),
           "df": torch.where(on, s * q * (Efull * m.abs() + full.abs() * (Em + 32 * U * m.abs())), zero), "dh0": Eg[:, 0]}
    return {k: v.to(dev) for k, v in val.items()}, {k: v.to(dev) for k, v in err.items()}


def philox(ctr, key):
    """Philox4x32-10 on arrays of 32-bit words held in uint64: ctr four arrays, key two integers -> four arrays."""
    low, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c, k = [np.asarray(w, dtype=np.uint64) for w in ctr], [int(v) for v in key]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(n, p, seed, offset):
    j = np.arange((n + 7) // 8, dtype=np.uint64)
    w = philox([j & np.uint64(0xFFFFFFFF), j >> np.uint64(32), np.full_like(j, offset & 0xFFFFFFFF), np.full_like(j, offset >> 32)],
               (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack([w[i // 2] >> np.uint64(16 * (i % 2)) & np.uint64(0xFFFF) for i in range(8)], 1).reshape(-1)[:n]
    return torch.from_numpy(halves >= int(p * 65536.0 + 0.5))


def keep_scale(p):
    return 65536.0 / (65536.0 - int(p * 65536.0 + 0.5))


def norm(x, groups, w, b, eps, act, p=0.0, seed=0, offset=0, dy=None):
    """As scan(): x, dy logical [N, C, H, W]."""
    dev = x.device
    N, C, H, W = x.shape
    rows = lambda t: t.detach().cpu().double().permute(0, 2, 3, 1).reshape(N, H * W, groups, C // groups)  # noqa: E731
    back = lambda t: t.reshape(N, H, W, C).permute(0, 3, 1, 2).to(dev)  # noqa: E731
    par = lambda t, v: torch.full((groups, C // groups), v, dtype=torch.float64) if t is None else t.detach().cpu().double().view(groups, -1)  # noqa: E731
    X, wt, bt = rows(x), par(w, 1.0), par(b, 0.0)
    avg = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    mu = avg(X)
    r = ((X - mu).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    xh = (X - mu) * r
    Exh = 32 * U * (xh.abs() + r * avg(X.abs()))
    z = xh * wt + bt
    Ez = wt.abs() * Exh + 4 * U * (z.abs() + bt.abs())
    s = torch.sigmoid(z)
    if act == "none":
        y, Ey, slope, Es = z, Ez, torch.ones_like(z), torch.zeros_like(z)
    elif act == "relu":      # (nothing but the sign of z decides the slope: it is open where z is within its own error of 0)
        y, Ey, slope, Es = z.clamp(min=0), Ez, (z > 0).double(), (z.abs() <= Ez).double()
    else:                    # |silu'| <= 1.1, |silu''| <= 0.5
        y, Ey, slope, Es = z * s, 1.1 * Ez + 16 * U * (z * s).abs(), s + z * s * (1 - s), 0.5 * Ez + 32 * U
    keep = torch.ones_like(X) if p == 0 else keep_mask(X.numel(), p, seed, offset).view(X.shape).double() * keep_scale(p)
    y, Ey = y * keep, Ey * keep + 2 * U * (y * keep).abs()
    val, err = {"y": back(y)}, {"y": back(Ey)}
    if dy is not None:
        g = rows(dy) * keep
        dz, Edz = g * slope, g.abs() * (Es + 4 * U * slope.abs())
        t, Et = wt * dz, wt.abs() * (Edz + 2 * U * dz.abs())
        tx, Etx = t * xh, Et * xh.abs() + t.abs() * Exh
        c1, c2 = avg(t), avg(tx)
        Ec1, Ec2 = avg(Et) + 64 * U * avg(t.abs()), avg(Etx) + 64 * U * avg(tx.abs())
        dx = r * (t - c1 - xh * c2)
        Edx = r * (Et + Ec1 + xh.abs() * Ec2 + Exh * c2.abs() + 8 * U * (t.abs() + c1.abs() + (xh * c2).abs())) + 40 * U * dx.abs()
        val.update(dx=back(dx), dw=(dz * xh).sum((0, 1)).reshape(C).to(dev), db=dz.sum((0, 1)).reshape(C).to(dev))
        err.update(dx=back(Edx), dw=(Edz * xh.abs() + dz.abs() * Exh + 64 * U * (dz * xh).abs()).sum((0, 1)).reshape(C).to(dev),
                   db=(Edz + 64 * U * dz.abs()).sum((0, 1)).reshape(C).to(dev))
    return val, err


def check(got, val, err, what=""):
    """got within err + the rounding of its own type of val, element by element; NaN and infinities in the same places."""
    assert got.shape == val.shape, (what, got.shape, val.shape)
    g = got.detach().double()
    tol = err + rounding(val, got.dtype)
    bad = ~((g - val).abs() <= tol) & ~(torch.isnan(g) & torch.isnan(val)) & ~(g == val)
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, first at {i}: "
                             f"{float(g[i])} for {float(val[i])}, allowed {float(tol[i]):.3e}")
