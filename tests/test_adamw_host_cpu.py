"""CPU: the host side of GroupedAdamW, grad_norm and clip_grad_norm_ - arguments that would be taken for others, parameter lists without
a parameter, gradients that share memory, libraries that do not fit this package."""
import pytest
import torch

from pde_amd.optim import GroupedAdamW, clip_grad_norm_


@pytest.mark.parametrize("third", [2.0, 1.0, 2, 1, float("inf"), "inf", None])
def test_a_norm_type_is_not_taken_for_error_if_nonfinite(third):
    """torch.nn.utils.clip_grad_norm_ takes the norm's type third; here it is always 2"""
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(TypeError, match="2-norm"):
        clip_grad_norm_([p], 1.0, third)
    assert torch.equal(p.grad, torch.ones(3))


def test_groups_without_any_parameter_are_refused():
    with pytest.raises(ValueError, match="no parameter"):
        GroupedAdamW([dict(params=[]), dict(params=[])])
