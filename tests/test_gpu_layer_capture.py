"""Training passes over the layer operators captured into a HIP graph beside autograd graphs that are still alive."""
import pytest
import torch

from test_gpu_layers import rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from pl_convlstm_gan_amd import layers as m
    return m


def replays(graph, got, want, what=""):
    """Every replay gives the eager pass's results, with eager work and synchronisations in between."""
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(got, want)):
            assert torch.equal(p, q), (what, k, i)
        torch.randn(1000, device="cuda").sum().item()


def test_warm_up_on_a_side_stream_may_stay_alive(layers, gpu):
    """PyTorch's own recipe of a captured training pass: a warm-up on a side stream, whose last loss is still referenced when the
    capture begins."""
    norm = layers.GroupNormAct(4, 16, act="silu").to(gpu)
    image = rand((2, 16, 8, 8), 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last).requires_grad_()
    x, f, r = (rand((2, 20, 12), k, torch.float32, gpu).requires_grad_() for k in (2, 3, 4))
    leaves = [norm.weight, norm.bias, image, x, f, r]

    def step():
        y, h = layers.gated_linear_scan(x, f)
        loss = (norm(image) ** 2).sum() + (layers.counter_dropout(y, 0.3, 5, 6, residual=r) ** 2).sum() + (h ** 2).sum()
        return loss, torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            loss, _ = step()
    torch.cuda.current_stream().wait_stream(side)
    assert loss.requires_grad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, got = step()
    replays(graph, got, [g.detach() for g in step()[1]])


def test_leaves_behind_other_operations(layers, gpu):
    """The leaf that an earlier pass on the default stream still holds reaches the operator through a cast, a view or another
    operation: refused like a leaf that is its argument.  Without that pass the capture works."""
    image = rand((2, 16, 8, 8), 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last)
    w, s = torch.ones(16, device=gpu, dtype=torch.bfloat16, requires_grad=True), rand((2, 20, 12), 3, torch.float32, gpu).requires_grad_()
    for name, leaf, call in (("cast weight", w, lambda: layers.group_norm_act(image, 4, w.float())), ("scaled input", s, lambda: layers.gated_linear_scan(s * 2, s.detach())[0]),
                             ("view", s, lambda: layers.counter_dropout(s[:, 3:], 0.5, 1)), ("gate of a gate", s, lambda: layers.gated_linear_scan(s.detach(), layers.counter_dropout(s, 0.5, 2))[0])):
        call()
        (want,) = torch.autograd.grad(call().sum(), leaf)
        alive = call()
        with pytest.raises(RuntimeError, match="earlier pass over the same leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (got,) = torch.autograd.grad(call().sum(), leaf)
        replays(graph, [got], [want], name)


def test_inputs_computed_before_the_capture(layers, gpu):
    """An input with a graph of its own, made on the default stream before the capture: gradients that do not lead there are
    captured, one that does is refused in the backward pass."""
    base = rand((2, 16, 8, 8), 1, torch.float32, gpu).contiguous(memory_format=torch.channels_last).requires_grad_()
    w, dy = torch.ones(16, device=gpu, requires_grad=True), rand((2, 16, 8, 8), 2, torch.float32, gpu)
    x = base * 2
    want = torch.autograd.grad(layers.group_norm_act(x, 4, w), w, dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layers.group_norm_act(x, 4, w), w, dy)
    replays(graph, got, want)
    for into in (base, x):
        with pytest.raises(RuntimeError, match="earlier pass over the same leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(layers.group_norm_act(x, 4, w), into, dy)
    replays(graph, got, want)
