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
