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
