"""How the layer operators meet the rest of PyTorch's differentiation: what they cannot do raises instead of giving a
wrong derivative.  The checks come before anything is launched, so they run without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD


def calls(x, image, x2=None, image2=None):
    """One call of every operator; x [B, T, D] and image [N, C, H, W] are what a derivative is asked of,
    x2 and image2 the other arguments of the same shapes."""
    from pl_convlstm_gan_amd import layers
    x2, image2 = x if x2 is None else x2, image if image2 is None else image2
    return {"scan": lambda: layers.gated_linear_scan(x, x2), "scan, gate": lambda: layers.gated_linear_scan(x2, x),
            "step": lambda: layers.gated_linear_step(x[:, 0], x2[:, 0], x2[:, 1]), "step, state": lambda: layers.gated_linear_step(x2[:, 0], x2[:, 0], x[:, 1]),
            "scan, state": lambda: layers.gated_linear_scan(x2, x2, x[:, 0]),
            "dropout": lambda: layers.counter_dropout(x, 0.5, 1), "residual": lambda: layers.counter_dropout(x2, 0.5, 1, residual=x),
            "norm": lambda: layers.group_norm_act(image, 2), "norm, weight": lambda: layers.group_norm_act(image2, 2, image[0, :, 0, 0]),
            "norm, bias": lambda: layers.group_norm_act(image2, 2, None, image[0, :, 0, 0])}


@pytest.mark.parametrize("mode", ["grad", "no_grad"])
def test_forward_mode_derivatives_are_refused(mode):
    """A dual tensor that needs no gradient would come back without its tangent, as a constant."""
    x, image = torch.randn(2, 3, 4), torch.randn(2, 4, 3, 3)
    with fwAD.dual_level(), torch.set_grad_enabled(mode == "grad"):
        dual = [fwAD.make_dual(t, torch.ones_like(t)) for t in (x, image)]
        for call in calls(*dual, x, image).values():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        # a dual level without a tangent is in nobody's way (the CPU tensors are the complaint)
        for call in calls(x, image).values():
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                call()


@pytest.mark.filterwarnings("ignore")
def test_recorders_that_cannot_see_a_kernel_are_refused():
    """torch.jit.trace and make_fx record PyTorch's own operations: of a call of these operators they would keep the
    allocation of the result and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from pl_convlstm_gan_amd import ops
    x, image = torch.randn(2, 3, 4), torch.randn(2, 4, 3, 3)
    one = lambda k: lambda x, image: calls(x, image)[k]()  # noqa: E731
    for grad in (False, True):
        for call in {**{k: one(k) for k in calls(x, image)},
                           "scan pass": lambda x, image: ops.gated_scan_forward(x, x),
                           "scan backward pass": lambda x, image: ops.gated_scan_backward(x, x, None, None, True, None, x, None),
                           "dropout pass": lambda x, image: ops.dropout_forward(x, 0.5, 1),
                           "norm pass": lambda x, image: ops.group_norm_forward(image, 2),
                           "norm backward pass": lambda x, image: ops.group_norm_backward(image, 2, None, None, 1e-5, "none", 0.0, 0, 0, x, image)}.values():
            a, b = x.clone().requires_grad_(grad), image.clone().requires_grad_(grad)
            with pytest.raises(RuntimeError, match="record"):
                torch.jit.trace(call, (a, b), check_trace=False)
            with pytest.raises(RuntimeError, match="record"):
                make_fx(call)(a, b)


@pytest.fixture
def cpu_stand_ins(monkeypatch):
    """The two operators with a mask, computed by the 64-bit references' generator on the CPU."""
    import layer_refs as R
    from pl_convlstm_gan_amd import layers

    def mask(x, p, seed, offset):
        return (R.keep_mask(x.numel(), p, int(seed), int(offset)).float() * R.keep_scale(p)).view(x.shape) if p > 0 else torch.ones(x.shape)

    def dropout(x, p, seed, offset=0, residual=None):
        y = x * mask(x, p, seed, offset)
        return y if residual is None else y + residual

    def norm(x, groups, w=None, b=None, eps=1e-5, act="none", p=0.0, seed=0, offset=0):
        y = torch.nn.functional.group_norm(x, groups, w, b, eps)
        return y * mask(y.permute(0, 2, 3, 1), p, seed, offset).permute(0, 3, 1, 2)
    monkeypatch.setattr(layers, "counter_dropout", dropout)
    monkeypatch.setattr(layers, "group_norm_act", norm)
    return layers


def recomputed(layers, dev, reentrant):
    """Activation recomputation runs a module's forward a second time inside the backward pass, when its own offset has moved on:
    refused, and right with an offset that the caller gives."""
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(2, 8, 6, 5, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_()
    for m in (layers.CounterDropout(0.5, seed=1).to(dev), layers.GroupNormAct(4, 8, p=0.5, seed=1).to(dev)):
        y = checkpoint(lambda v: m(v).square(), x, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="offset"):
            y.sum().backward()
        before = int(m.offset)
        for offset in (7, torch.tensor([7], device=dev)):
            plain = torch.autograd.grad(m(x, offset=offset).square().sum(), x)[0]
            y = checkpoint(lambda v, k: m(v, offset=k).square(), x, offset, use_reentrant=reentrant)
            x.grad = None
            y.sum().backward()
            assert torch.equal(x.grad, plain) and int(m.offset) == before
        if isinstance(m, layers.CounterDropout):
            assert torch.equal(y == 0, x.grad == 0) and bool((y == 0).any())
        # without a mask there is nothing to keep apart
        m.eval()
        want = torch.autograd.grad(m(x).square().sum(), x)[0]
        x.grad = None
        checkpoint(lambda v: m(v).square(), x, use_reentrant=reentrant).sum().backward()
        assert torch.equal(x.grad, want)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_takes_the_same_mask_or_raises(cpu_stand_ins, reentrant):
    recomputed(cpu_stand_ins, torch.device("cpu"), reentrant)


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_on_the_gpu(gpu, reentrant):
    from pl_convlstm_gan_amd import layers
    recomputed(layers, gpu, reentrant)


def test_generator_with_a_mask_is_not_recomputed():
    """The rollout with the feature head's dropout inside a backward pass: refused before anything runs; without dropout, or
    in evaluation mode, it is not (and a machine without a GPU is the complaint)."""
    from pl_convlstm_gan_amd import Generator

    class Probe(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, call):
            ctx.call = call
            return x * 1

        @staticmethod
        def backward(ctx, g):
            ctx.call()
            return g, None
    model = Generator(hidden_dims=[16, 32], lu_channels=5, scale_factor=1)
    args = torch.zeros(1, 2, 1, 16, 16), torch.zeros(1, 1, 16, 16), torch.zeros(1, 5, 16, 16)

    def inside():
        with pytest.raises(RuntimeError) as e:
            model(*args) if not torch.cuda.is_available() else pytest.skip("needs a machine without a GPU")
        messages.append(str(e.value))
    messages = []
    for p, training in ((0.0, True), (0.3, False), (0.3, True)):
        model.set_feature_head(4, p=p, seed=3).train(training)
        Probe.apply(torch.ones(1, requires_grad=True), inside).backward()
    assert ["dropout" in m and "backward" in m for m in messages] == [False, False, True]


def test_default_modules_draw_masks_of_their_own(cpu_stand_ins):
    """Two modules that were given no seed drop different elements, from the first pass on; torch.manual_seed and a saved
    state bring the masks back; with a seed the offset counts from 0."""
    layers = cpu_stand_ins
    x = torch.ones(2, 8, 16, 16)
    image = torch.randn(x.shape, generator=torch.Generator().manual_seed(1))

    def make():
        return torch.nn.ModuleList([layers.CounterDropout(0.5), layers.CounterDropout(0.5), layers.GroupNormAct(2, 8, p=0.5), layers.GroupNormAct(2, 8, p=0.5)])

    def masks(ms):                                         # (of three passes; elements in the order the masks count them)
        return [torch.stack([ms[0](x) != 0, ms[1](x) != 0] + [(m(image) != 0).permute(0, 2, 3, 1).reshape(x.shape) for m in ms[2:]]) for _ in range(3)]
    torch.manual_seed(11)
    a, b = make(), make()
    got = torch.cat(masks(a) + masks(b)).flatten(1)
    # 4096 independent fair elements each: the number two masks agree on is 2048 +- 32, 8 deviations allowed
    agree = (got[:, None] == got[None]).sum(2)
    agree.fill_diagonal_(2048)
    assert int((agree - 2048).abs().max()) <= 256
    torch.manual_seed(11)
    again = make()
    assert torch.equal(torch.cat(masks(again)).flatten(1), got[:12])
    state = {k: v.clone() for k, v in again.state_dict().items()}
    went_on = torch.cat(masks(again))
    torch.manual_seed(12)
    other = make()
    assert not torch.equal(torch.cat(masks(other)).flatten(1), got[:12])
    other.load_state_dict(state)
    assert torch.equal(torch.cat(masks(other)), went_on)
    for m in (layers.CounterDropout(0.5, seed=0), layers.CounterDropout(0.5, seed=7), layers.GroupNormAct(2, 8, p=0.5, seed=0), layers.CounterDropout(0.0), layers.GroupNormAct(2, 8)):
        assert int(m.offset) == 0
    # (nothing is drawn where nothing is dropped, or where a seed is given)
    torch.manual_seed(3)
    layers.CounterDropout(0.0), layers.GroupNormAct(2, 8), layers.CounterDropout(0.5, seed=1)
    drawn = torch.rand(1)
    torch.manual_seed(3)
    assert torch.equal(torch.rand(1), drawn)


def test_default_feature_heads_draw_masks_of_their_own():
    from pl_convlstm_gan_amd import Generator
    make = lambda **kw: Generator(hidden_dims=[16, 32], lu_channels=5, scale_factor=1).set_feature_head(4, p=0.2, **kw).feature_norm  # noqa: E731
    torch.manual_seed(5)
    a, b = make(), make()
    torch.manual_seed(5)
    assert int(a.offset) != int(b.offset) and int(make().offset) == int(a.offset) and a.seed == b.seed == 0
    assert int(make(seed=3).offset) == 0 and make(seed=3).seed == 3


@pytest.mark.gpu
def test_default_modules_on_the_gpu(gpu):
    from pl_convlstm_gan_amd import layers
    a, b = layers.CounterDropout(0.5).to(gpu), layers.CounterDropout(0.5).to(gpu)
    x = torch.ones(4096, device=gpu)
    first, start = int(a.offset), a(x)
    assert not torch.equal(start, b(x)) and int(a.offset) == first + 1
    assert torch.equal(start, layers.counter_dropout(x, 0.5, 0, first))


def test_trainer_runs_and_ranks_draw_masks_of_their_own(monkeypatch):
    """Two runs of the Trainer draw different masks unless torch's seed is the same; ranks start at one offset (and one set of
    weights) under seeds of their own."""
    from pl_convlstm_gan_amd.host import trainer as T
    from pl_convlstm_gan_amd.host.config import Config

    class Data:
        lucc_onehot = torch.zeros(5, 4, 4)

    def head(rank=0, world=1, dropout=0.2):
        monkeypatch.setattr(T, "_rank_world", lambda: (rank, world))
        t = T.Trainer.__new__(T.Trainer)
        t.config, t.device = Config(), torch.device("cpu")
        t.config.model.feature_groups, t.config.model.feature_dropout = 4, dropout
        t._make_optimizer = lambda params, lr: torch.optim.Adam(params, lr=lr)
        t.setup_model(Data())
        return t.model.feature_norm.seed, int(t.model.feature_norm.offset), t.model.init_conv.weight.detach().clone()
    torch.manual_seed(1)
    (s0, o0, _), (s1, o1, _) = head(), head()
    assert o0 != o1 and s0 == s1 == 0
    torch.manual_seed(1)
    assert head()[1] == o0
    (s0, o0, w0), (s1, o1, w1) = head(0, 2), head(1, 2)
    assert (s0, s1) == (0, 1) and o0 == o1 and torch.equal(w0, w1)
    assert head(dropout=0.0)[:2] == (0, 0)
