"""CPU oracle for the ConvLSTM rollout + generator conv stack.

TEST INFRASTRUCTURE ONLY.  This file is a functional CPU restatement (PyTorch CPU
ops, fp32) of the reference algorithm.  Only tests/, __graft_entry__.smoke() and the
cpu_baseline leg of bench.py may import it; the product path never does.

Parity status: PINNED.  tests/test_oracle_golden.py checks every function here against
golden vectors generated by importing the reference on CPU (tests/golden/make_golden.py).

Each function cites the reference lines it restates.  Parameters are passed as a flat
dict keyed by the reference's state_dict names (init_conv.weight, cell1.conv.weight,
dem_attn.conv.0.weight, ..., upsample_blocks.0.conv.weight, post_process.2.bias).

`emulate="bf16"` mirrors the storage-rounding points of the HIP bf16 pipeline (operands
of every MFMA product rounded to bf16, fp32 accumulation, fp32 cell state, hidden state /
feature maps stored as bf16) so the GPU result can be compared at a tight tolerance.
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

Params = Dict[str, torch.Tensor]


# --------------------------------------------------------------------------------------
# rounding helpers
# --------------------------------------------------------------------------------------
def bf16_round(t: torch.Tensor) -> torch.Tensor:
    """Round-to-nearest-even fp32 -> bf16 -> fp32 (value-preserving container)."""
    return t.to(torch.bfloat16).to(torch.float32)


def fp8_round(t: torch.Tensor) -> torch.Tensor:
    """fp32 -> OCP e4m3 (round to nearest even, clamped to +-448) -> fp32.  Straight-through for
    autograd (the engine's backward pass runs in bf16 on the saved activations)."""
    q = t.detach().clamp(-448.0, 448.0).to(torch.float8_e4m3fn).to(torch.float32)
    return t + (q - t.detach())


def fp8_weight_exponent(w: torch.Tensor) -> int:
    """The power of two the fp8 path multiplies a conv weight by before rounding it to e4m3:
    max|w| = 1.m * 2^k  ->  e = 7 - k (largest scaled magnitude in [128, 256))."""
    import math
    amax = float(w.detach().abs().max())
    if not (amax > 0.0 and math.isfinite(amax)):
        return 0
    _, ex = math.frexp(amax)            # amax = m * 2^ex with m in [0.5, 1)
    return max(-100, min(100, 7 - (ex - 1)))


def fp8_weight(w: torch.Tensor) -> torch.Tensor:
    e = fp8_weight_exponent(w)
    return fp8_round(w * (2.0 ** e)) * (2.0 ** -e)


def _q(emulate: Optional[str]):
    if emulate is None:
        return lambda t: t
    if emulate in ("bf16", "fp8"):      # "fp8": only the gate convs' operands are e4m3, the rest is the bf16 pipeline
        return bf16_round
    raise ValueError(f"unknown emulate mode {emulate!r}")


# --------------------------------------------------------------------------------------
# coordconv.py:3-10
# --------------------------------------------------------------------------------------
def coord_tables(H: int, W: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Row / column coordinate tables: linspace(0,1,H), linspace(0,1,W)."""
    return torch.linspace(0, 1, H), torch.linspace(0, 1, W)


def coord_channels(x: torch.Tensor) -> torch.Tensor:
    """[B,C,H,W] -> [B,C+2,H,W]; appended channels are (row, col) in that order."""
    B, _, H, W = x.shape
    row, col = coord_tables(H, W)
    rr = row.view(1, 1, H, 1).expand(B, 1, H, W)
    cc = col.view(1, 1, 1, W).expand(B, 1, H, W)
    return torch.cat((x, rr, cc), dim=1)


# --------------------------------------------------------------------------------------
# convlstm.py:16-28
# --------------------------------------------------------------------------------------
def convlstm_cell(x, h, c, weight, bias, emulate: Optional[str] = None):
    """One ConvLSTM step.  weight [4Ch, Cin+Ch, k, k] acts on cat([x, h]); gate order
    along the output channels is i, f, o, g.  Returns (h', c')."""
    q = _q(emulate)
    Ch = h.shape[1]
    k = weight.shape[-1]
    if emulate == "fp8":
        # operands of the gate conv as the fp8 path sees them: activations bf16-stored, then e4m3;
        # weights scaled by a power of two, e4m3, scaled back (exact); fp32 accumulation and bias
        z = F.conv2d(torch.cat((fp8_round(q(x)), fp8_round(q(h))), dim=1), fp8_weight(weight), bias, padding=k // 2)
    else:
        z = F.conv2d(torch.cat((q(x), q(h)), dim=1), q(weight), bias, padding=k // 2)
    zi, zf, zo, zg = z[:, 0:Ch], z[:, Ch:2 * Ch], z[:, 2 * Ch:3 * Ch], z[:, 3 * Ch:4 * Ch]
    c_new = torch.sigmoid(zf) * c + torch.sigmoid(zi) * torch.tanh(zg)
    h_new = torch.sigmoid(zo) * torch.tanh(c_new)
    return h_new, c_new


# --------------------------------------------------------------------------------------
# generator.py:73-92  (how many PixelShuffle(2) blocks a scale needs + residual factor)
# --------------------------------------------------------------------------------------
def upsample_plan(scale_factor: int) -> Tuple[int, float]:
    s = int(scale_factor)
    if s <= 1:
        return 0, 1
    n, cur = 0, s
    while cur > 1 and cur >= 2:
        n += 1
        cur //= 2
    return n, s / (2 ** n)


def resolve_geometry(H, W, scale_factor=None, target_grid_size=None, input_grid_size=None):
    """generator.py:106-140 -> (scale, target_size_or_None, final_H, final_W)."""
    if target_grid_size is not None and input_grid_size is not None:
        gx, gy = input_grid_size
        tx, ty = target_grid_size
        sw, sh = gx / tx, gy / ty
        target = (int(H * sh), int(W * sw))
        return max(sh, sw), target, target[0], target[1]
    if scale_factor is not None:
        return scale_factor, None, int(H * scale_factor), int(W * scale_factor)
    return 1, None, int(H), int(W)


# --------------------------------------------------------------------------------------
# attention.py:6-13, 19-26
# --------------------------------------------------------------------------------------
def attention_gate(aux, w0, b0, w1, b1, emulate: Optional[str] = None):
    """sigmoid(conv1x1(relu(conv3x3(aux)))) -> [B, C2, Hh, Wh]."""
    q = _q(emulate)
    mid = q(F.relu(F.conv2d(q(aux), q(w0), b0, padding=1)))
    return torch.sigmoid(F.conv2d(mid, q(w1), b1))


# --------------------------------------------------------------------------------------
# generator.py:94-205
# --------------------------------------------------------------------------------------
def generator_forward(p: Params, rain_lr, dem, lu, *, scale_factor=None, target_grid_size=None,
                      input_grid_size=None, emulate: Optional[str] = None,
                      return_states: bool = False, feature_head=None):
    """Whole rollout.  rain_lr [B,T,1,H,W], dem [B,1,.,.], lu [B,L,.,.] -> [B,T,1,Hh,Wh].

    The two attention gates do not depend on t, so they are evaluated once and their
    product is applied every step (generator.py:198-199 evaluates them inside the loop;
    the values are identical).  The number of upsample blocks is read from the params
    dict (they must have been materialised, generator.py:129-132).
    ``feature_head(h2, t)``: what the engine's optional feature head does to the features of step t (not in the reference).
    """
    q = _q(emulate)
    B, T, _, H, W = rain_lr.shape
    scale, target, fH, fW = resolve_geometry(H, W, scale_factor, target_grid_size, input_grid_size)
    n_blocks = 0
    while f"upsample_blocks.{n_blocks}.conv.weight" in p:
        n_blocks += 1
    remaining = scale / (2 ** n_blocks)

    dem_hr = F.interpolate(dem, size=(fH, fW), mode="bilinear", align_corners=False)
    lu_hr = F.interpolate(lu, size=(fH, fW), mode="nearest")
    g_dem = attention_gate(dem_hr, p["dem_attn.conv.0.weight"], p["dem_attn.conv.0.bias"],
                           p["dem_attn.conv.2.weight"], p["dem_attn.conv.2.bias"], emulate)
    g_lu = attention_gate(lu_hr, p["lu_attn.conv.0.weight"], p["lu_attn.conv.0.bias"],
                          p["lu_attn.conv.2.weight"], p["lu_attn.conv.2.bias"], emulate)
    if emulate is None:
        gate = None
    else:
        # HIP pipeline stores sigma(dem) as bf16, multiplies sigma(lu) by it, stores bf16.
        gate = q(q(g_dem) * g_lu)

    C1 = p["cell1.conv.weight"].shape[0] // 4
    C2 = p["cell2.conv.weight"].shape[0] // 4
    h1 = torch.zeros(B, C1, H, W)
    c1 = torch.zeros_like(h1)
    h2 = torch.zeros(B, C2, H, W)
    c2 = torch.zeros_like(h2)
    outs = []
    states = []
    for t in range(T):
        x = coord_channels(rain_lr[:, t])
        x = q(F.relu(F.conv2d(q(x), q(p["init_conv.weight"]), p["init_conv.bias"], padding=1)))
        h1, c1 = convlstm_cell(x, h1, c1, p["cell1.conv.weight"], p["cell1.conv.bias"], emulate)
        h1 = q(h1)
        h2, c2 = convlstm_cell(h1, h2, c2, p["cell2.conv.weight"], p["cell2.conv.bias"], emulate)
        h2 = q(h2)
        if return_states:
            states.append((h1, c1, h2, c2))
        feat = h2 if feature_head is None else q(feature_head(h2, t))
        for k in range(n_blocks):
            w = p[f"upsample_blocks.{k}.conv.weight"]
            b = p[f"upsample_blocks.{k}.conv.bias"]
            feat = q(F.relu(F.pixel_shuffle(F.conv2d(q(feat), q(w), b, padding=1), 2)))
        if remaining > 1:
            feat = q(F.interpolate(feat, scale_factor=remaining, mode="bilinear", align_corners=False))
        if target is not None:
            feat = q(F.interpolate(feat, size=target, mode="bilinear", align_corners=False))
        if gate is None:
            feat = (feat * g_dem) * g_lu
        else:
            feat = q(feat * gate)
        mid = q(F.relu(F.conv2d(feat, q(p["post_process.0.weight"]), p["post_process.0.bias"], padding=1)))
        out = F.conv2d(mid, q(p["post_process.2.weight"]), p["post_process.2.bias"], padding=1)
        outs.append(out.unsqueeze(1))
    y = torch.cat(outs, dim=1)
    if return_states:
        return y, states
    return y


# --------------------------------------------------------------------------------------
# combined_loss.py:23-191
# --------------------------------------------------------------------------------------
def sample_weights(obs, use_weighted=True, strategy="log"):
    """combined_loss.py:23-59."""
    if not use_weighted:
        return torch.ones_like(obs)
    if strategy == "log":
        return 1.0 + torch.log1p(obs)
    if strategy == "stratified":
        w = torch.ones_like(obs)
        for thr, val in ((10, 2.0), (25, 3.0), (50, 5.0)):
            w = torch.where(obs >= thr, torch.full_like(obs, val), w)
        return w
    if strategy == "sqrt":
        return 1.0 + torch.sqrt(obs)
    return torch.ones_like(obs)


def loss_conserve(pred, lr_input):
    """combined_loss.py:64-74: area-average pred back to the LR grid, L1 to the input."""
    B, T, C, H, W = pred.shape
    Hl, Wl = lr_input.shape[-2:]
    pooled = F.interpolate(pred.reshape(B * T, C, H, W), size=(Hl, Wl), mode="area")
    return (pooled.reshape(B, T, C, Hl, Wl) - lr_input).abs().mean()


def station_pixels(s_coords, scale_factor, H, W):
    """combined_loss.py:90-104 / trainer.py:237-243: LR station (row, col) -> HR pixel,
    truncating; returns (rows, cols, in_bounds_mask).  Batched coords use sample 0."""
    coords = s_coords[0] if s_coords.dim() == 3 else s_coords
    sc = ((coords.float() + 0.5) * scale_factor - 0.5).long()
    r, c = sc[:, 0], sc[:, 1]
    ok = (r >= 0) & (r < H) & (c >= 0) & (c < W)
    return r, c, ok


def loss_point(pred, s_coords, s_values, scale_factor=1.0, use_weighted=True, strategy="log"):
    """combined_loss.py:79-141."""
    if s_values is None or s_coords.numel() == 0:
        return torch.tensor(0.0)
    B, T, _, H, W = pred.shape
    r, c, ok = station_pixels(s_coords, scale_factor, H, W)
    r, c = r[ok], c[ok]
    if r.numel() == 0:
        return torch.tensor(0.0)
    at = pred[:, :, 0][:, :, r, c]                      # [B,T,N]
    if s_values.dim() == 3:
        obs = s_values[:, :, ok]
    else:
        obs = s_values[:, ok].unsqueeze(0).expand(B, -1, -1)
    valid = ~torch.isnan(obs)
    if int(valid.sum()) == 0:
        return torch.tensor(0.0)
    o = obs[valid]
    return ((at[valid] - o).abs() * sample_weights(o, use_weighted, strategy)).mean()


def loss_smooth(pred):
    """combined_loss.py:146-155."""
    dx = (pred[..., :, :-1] - pred[..., :, 1:]).abs().mean()
    dy = (pred[..., :-1, :] - pred[..., 1:, :]).abs().mean()
    return dx + dy


def loss_temporal(pred):
    """combined_loss.py:160-168 (T == 1 gives the mean of an empty tensor = NaN)."""
    return (pred[:, :-1] - pred[:, 1:]).abs().mean()


def combined_loss(pred, lr_input, s_coords, s_values, scale_factor=1.0, *, lambda_point=1.0,
                  lambda_conserve=1.0, lambda_smooth=0.1, lambda_temporal=0.05,
                  use_weighted=True, strategy="log"):
    """combined_loss.py:173-191 -> (total, dict)."""
    lp = loss_point(pred, s_coords, s_values, scale_factor, use_weighted, strategy)
    lc = loss_conserve(pred, lr_input)
    ls = loss_smooth(pred)
    lt = loss_temporal(pred)
    total = lambda_point * lp + lambda_conserve * lc + lambda_smooth * ls + lambda_temporal * lt
    return total, {"point": lp, "conserve": lc, "smooth": ls, "temporal": lt}


# --------------------------------------------------------------------------------------
# trainer.py:225-272
# --------------------------------------------------------------------------------------
def station_rmse(pred, s_coords, s_values, scale_factor=1.0):
    """RMSE between pred at station pixels and non-NaN observations."""
    B, T, _, H, W = pred.shape
    r, c, ok = station_pixels(s_coords, scale_factor, H, W)
    r, c = r[ok], c[ok]
    at = pred[:, :, 0][:, :, r, c]
    obs = s_values[:, :, ok]
    valid = ~torch.isnan(obs)
    if int(valid.sum()) == 0:
        return 0.0
    return float(torch.sqrt(((at[valid] - obs[valid]) ** 2).mean()))


# --------------------------------------------------------------------------------------
# trainer.py:290-315 (one optimisation step; Adam over a chosen subset of the params)
# --------------------------------------------------------------------------------------
def grads_of(p: Params, rain_lr, dem, lu, s_coords, s_values, *, fwd_kw=None, loss_kw=None):
    """Forward + CombinedLoss + backward via autograd on the restatement.
    Returns (loss, {name: grad}, pred)."""
    fwd_kw = dict(fwd_kw or {})
    loss_kw = dict(loss_kw or {})
    leaf = {k: v.detach().clone().requires_grad_(True) for k, v in p.items()}
    pred = generator_forward(leaf, rain_lr, dem, lu, **fwd_kw)
    sf = pred.shape[-2] / rain_lr.shape[-2]
    loss, _ = combined_loss(pred, rain_lr, s_coords, s_values, sf, **loss_kw)
    loss.backward()
    return loss.detach(), {k: v.grad for k, v in leaf.items()}, pred.detach()


def clip_coef(grads: Sequence[torch.Tensor], max_norm: float) -> float:
    """torch.nn.utils.clip_grad_norm_ semantics (trainer.py:311-314): L2 over all grads,
    coefficient = min(1, max_norm / (norm + 1e-6))."""
    total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    return min(1.0, max_norm / (total + 1e-6))
