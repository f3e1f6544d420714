"""The Generator's optional feature head (group norm + activation + dropout on the recurrence's features): inside the
rollout against the 64-bit reference of the operator on the rollout's own features, the whole model against the oracle
with the same head, dropout, HIP graph, Trainer."""
import ctypes as C

import numpy as np
import pytest
import torch

import layer_refs as R
from conftest import master_params
from oracle import cpu_oracle as O

pytestmark = pytest.mark.gpu


def make(gpu, s=1, groups=8, act="silu", p=0.0, dims=(16, 32), **kw):
    from pl_convlstm_gan_amd import Generator
    from pl_convlstm_gan_amd.models import UpsampleBlock
    nb, _ = O.upsample_plan(s)
    m = Generator(hidden_dims=list(dims), lu_channels=5, scale_factor=s)
    m.upsample_blocks = torch.nn.ModuleList([UpsampleBlock(dims[1], 2) for _ in range(nb)])
    if dims == (16, 32):
        m.load_state_dict(master_params(nb), strict=True)
    m.set_feature_head(groups, act, p, **kw)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        m.feature_norm.weight.copy_(1 + 0.2 * torch.randn(dims[1], generator=g))
        m.feature_norm.bias.copy_(0.2 * torch.randn(dims[1], generator=g))
    return m.to(gpu)


def inputs(gpu, B=2, T=3, H=24, W=40, s=1, seed=1):
    g = torch.Generator().manual_seed(seed)
    rain = 10 * torch.rand(B, T, 1, H, W, generator=g) * (torch.rand(B, T, 1, H, W, generator=g) > 0.7)
    dem = torch.rand(B, 1, H * s, W * s, generator=g)
    lu = torch.nn.functional.one_hot(torch.randint(0, 5, (B, H * s, W * s), generator=g), 5).permute(0, 3, 1, 2).float().contiguous()
    return rain.to(gpu), dem.to(gpu), lu.to(gpu)


def internal(m, rain, dem, lu, save):
    """The features before and behind the head, [T * B, C, H, W] bf16, from the rollout's workspace."""
    from pl_convlstm_gan_amd import _lib
    from pl_convlstm_gan_amd.autograd import _param_list
    out, d, (ws, _) = m._forward_impl(rain, dem, lu, None, save, [p.detach() for p in _param_list(m)])
    torch.cuda.synchronize()
    n, ch, H, W = d.T * d.B, d.C2, d.H, d.W

    def at(name, skip):
        o = _lib.lib().plc_generator_workspace_offset(C.byref(d), name) + skip * ch * H * W * 2
        cb8 = ws[o:o + n * ch * H * W * 2].view(torch.bfloat16).view(n, ch // 8, H, W, 8)
        return cb8.permute(0, 1, 4, 2, 3).reshape(n, ch, H, W)
    return at(b"h2s", d.B), at(b"head", 0), out


@pytest.mark.parametrize("groups,act,dims,shape", [(8, "silu", (16, 32), (2, 3, 24, 40)), (4, "relu", (16, 32), (1, 2, 15, 12)), (32, "none", (16, 32), (2, 2, 64, 64)),
                                                   (1, "silu", (16, 32), (1, 4, 33, 17)), (3, "relu", (16, 24), (1, 2, 20, 20)), (2, "silu", (16, 64), (1, 2, 20, 36)),
                                                   (8, "relu", (16, 32), (1, 2, 256, 256))])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_head_inside_the_rollout(gpu, groups, act, dims, shape, p):
    B, T, H, W = shape
    m = make(gpu, 1, groups, act, p, dims, seed=21)
    for save in (False, True):
        h2, head, _ = internal(m, *inputs(gpu, B, T, H, W), save)
        val, err = R.norm(h2, groups, m.feature_norm.weight, m.feature_norm.bias, 1e-5, act, p, 21, 0)
        R.check(head, val["y"], err["y"], f"head {groups} {act} {dims} {shape} p={p}")


@pytest.mark.parametrize("groups,act,p", [(8, "silu", 0.0), (4, "relu", 0.3), (2, "silu", 0.2), (1, "none", 0.0), (32, "silu", 0.0)])
@pytest.mark.parametrize("N,ch,H,W", [(3, 32, 15, 12), (2, 64, 40, 24), (1, 32, 130, 130), (5, 96, 7, 9)])
def test_norm_on_the_engines_layout(gpu, N, ch, H, W, groups, act, p):
    """plc_group_norm_fwd / _bwd on CB8 tensors, element by element, masks as on channels-last ones."""
    from pl_convlstm_gan_amd import _lib, ops
    L, st = _lib.lib(), ops._stream()
    g = torch.Generator().manual_seed(ch + H)
    x, dy = (torch.randn(N, ch, H, W, generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    w, b = (torch.randn(ch, generator=g).to(gpu) for _ in range(2))
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
        R.check(v, val[k], err[k], f"{k} {N} {ch} {H} {W} {groups} {act} {p}")


@pytest.mark.parametrize("s", [1, 2, 3])
def test_model_with_head_against_the_oracle(gpu, s):
    """Forward within 2e-2 of the largest output, gradients of a linear functional against autograd on the bf16
    restatement.  The functional's weights are random signs, so a gradient is a sum that mostly cancels, and what the bf16
    pipeline does to it is measured rather than guessed: e_k = |g_bf16 - g_fp32| / |g_fp32| of the restatement itself is the effect
    of ONE rounding (half a step, 2^-9) of every stored tensor of the forward pass.  The engine shares those roundings
    (up to the ones that another summation order turns over) and adds one of the same size to every stored tensor of the
    backward pass, of which there are as many, so to first order it is e_k from the restatement; where that is smaller, the model's own
    bound of 3e-2 holds.  (The operator inside is checked element by element above.)"""
    m = make(gpu, s)
    rain, dem, lu = inputs(gpu, s=s)
    out = m(rain, dem, lu)
    r = torch.randn(out.shape, generator=torch.Generator().manual_seed(3))
    names = [k for k, _ in m.named_parameters()]
    grads = dict(zip(names, torch.autograd.grad(out, [p for _, p in m.named_parameters()], r.to(gpu))))
    ref = {}
    for emulate in ("bf16", None):
        leaf = {k: v.detach().cpu().clone().requires_grad_() for k, v in m.state_dict().items() if k != "feature_norm.offset"}

        def head(h2, t):
            z = torch.nn.functional.group_norm(h2, 8, leaf["feature_norm.weight"], leaf["feature_norm.bias"], 1e-5)
            return z * torch.sigmoid(z)
        y = O.generator_forward({k: v for k, v in leaf.items() if not k.startswith("feature_norm")}, rain.cpu(), dem.cpu(), lu.cpu(),
                                scale_factor=s, emulate=emulate, feature_head=head)
        (y * r).sum().backward()
        ref[emulate] = (y.detach(), {k: v.grad for k, v in leaf.items()})
    want = ref["bf16"][0]
    assert float((out.detach().cpu() - want).abs().max()) <= 2e-2 * float(want.abs().max())
    for k in names:
        b, f = ref["bf16"][1][k], ref[None][1][k]
        allowed = max(3e-2, float((b - f).norm() / f.norm()))
        e = float((grads[k].cpu() - b).norm() / b.norm())
        assert e <= allowed, (k, e, allowed)


def test_head_off_is_the_reference_model(gpu):
    m = make(gpu)
    args = inputs(gpu)
    with torch.no_grad():
        with_head = m(*args)
        off = m.set_feature_head(0)(*args)
    plain = make(gpu).set_feature_head(0)
    assert "feature_norm.weight" not in plain.state_dict() and torch.equal(plain(*args).detach(), off) and not torch.equal(off, with_head)


def test_head_dropout_and_offsets(gpu):
    m = make(gpu, p=0.4, seed=7)
    args = inputs(gpu)
    with torch.no_grad():
        a, b = m(*args), m(*args)
        assert int(m.feature_norm.offset) == 2 and not torch.equal(a, b)
        m.feature_norm.offset.zero_()
        assert torch.equal(m(*args), a)
        m.eval()
        e = m(*args)
        assert torch.equal(m(*args), e) and int(m.feature_norm.offset) == 1
        h2, head, _ = internal(m, *args, False)
        assert float((head == 0).float().mean()) < 0.01
        m.train()
        m.feature_norm.offset.fill_(3)
        _, head, _ = internal(m, *args, False)
    keep = R.keep_mask(head.numel(), 0.4, 7, 3).view(head.permute(0, 2, 3, 1).shape).permute(0, 3, 1, 2).to(gpu)
    assert float(head[~keep].abs().max()) == 0 and torch.equal(head != 0, keep & (head != 0)) and float((head[keep] != 0).float().mean()) > 0.99
    # the backward pass takes the offset its forward pass used, whatever the buffer says by then
    m.feature_norm.offset.fill_(5)
    out = m(*args)
    r = torch.ones_like(out)
    ps = list(m.parameters())
    g1 = torch.autograd.grad(out, ps, r)
    m.feature_norm.offset.fill_(5)
    out2 = m(*args)
    m.feature_norm.offset.fill_(1000)
    g2 = torch.autograd.grad(out2, ps, r)
    assert torch.equal(out, out2) and all(torch.equal(x, y) for x, y in zip(g1, g2))


def _batch(seed, dev, B=4, T=3, H=15, W=12, s=2, N=6):
    rain, dem, lu = inputs(dev, B, T, H, W, s, seed)
    g = torch.Generator().manual_seed(seed)
    coords = torch.randint(0, min(H, W), (N, 2), generator=g).unsqueeze(0).repeat(B, 1, 1)
    return [rain, dem, lu, coords.to(dev), (20 * torch.rand(B, T, N, generator=g)).to(dev)]


def test_graphed_step_with_head_equals_eager(gpu):
    from pl_convlstm_gan_amd.losses import CombinedLoss
    from pl_convlstm_gan_amd.optim import FusedAdam
    from pl_convlstm_gan_amd.training import GraphedTrainStep, train_step
    seeds = [10, 20, 30, 40]

    def setup():
        m = make(gpu, 2, p=0.2, seed=3)
        return m, CombinedLoss(), FusedAdam(m.parameters(), lr=5e-4)
    m, loss_mod, opt = setup()
    ref = []
    for k in seeds:
        loss = train_step(m, loss_mod, opt, *_batch(k, gpu), max_norm=0.5, nan_check="device")[0]
        ref.append((float(loss.detach()), torch.cat([p.detach().reshape(-1) for p in m.parameters()]).clone()))
    del loss
    assert int(m.feature_norm.offset) == len(seeds)
    m, loss_mod, opt = setup()
    step = GraphedTrainStep(m, loss_mod, opt, _batch(99, gpu), max_norm=0.5)
    assert int(m.feature_norm.offset) == 0                       # the warm-up left no trace
    for k, (l, p) in zip(seeds, ref):
        loss = step(*_batch(k, gpu))[0]
        assert float(loss) == l and torch.equal(torch.cat([q.detach().reshape(-1) for q in m.parameters()]), p)
    assert int(m.feature_norm.offset) == len(seeds)


def test_trainer_with_feature_head(gpu, tmp_path, monkeypatch):
    from pl_convlstm_gan_amd.host import config as C
    from pl_convlstm_gan_amd.host.datasets import write_synthetic_dataset
    paths = write_synthetic_dataset(str(tmp_path / "basin"), start_year=2012, end_year=2013, lr_hw=(15, 12), scale=2, n_stations=10)
    cfg = C.Config()
    for k, v in paths.items():
        setattr(cfg.data, k, v)
    cfg.model.scale_factor, cfg.model.feature_groups, cfg.model.feature_act, cfg.model.feature_dropout = 2, 4, "relu", 0.1
    cfg.training.batch_size, cfg.training.epochs = 32, 1
    cfg.training.train_years, cfg.training.val_years, cfg.training.test_years = [2012, 2012], [2013, 2013], [2013, 2013]
    cfg.output.output_dir = str(tmp_path / "out")
    cfg.to_yaml(str(tmp_path / "configs" / "synthetic.yaml"))
    monkeypatch.setattr(C, "CONFIG_DIR", str(tmp_path / "configs"))
    from src.training.trainer import Trainer
    t = Trainer("synthetic")
    t.train()
    head = t.model.feature_norm
    assert (head.num_groups, head.act, head.p) == (4, "relu", 0.1) and int(head.offset) > 0
    assert all(np.isfinite(t.history["total_loss"])) and all(np.isfinite(t.history["rmse"]))
    assert float((head.weight.detach() - 1).abs().max()) > 0 and len(t.optimizer.param_groups[0]["params"]) == 20
