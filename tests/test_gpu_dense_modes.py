"""Derivatives that dense layers do not have are refused, not left out."""
import pytest
import torch

import difflogic_b200 as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(which, grad):
    given = [torch.randn(*s, device="cuda", requires_grad=grad) for s in ((5, 6), (7, 6), (7,), (5, 7))]
    with torch.autograd.forward_ad.dual_level():
        given[which] = torch.autograd.forward_ad.make_dual(given[which], torch.randn_like(given[which]))
        with pytest.raises(RuntimeError, match="forward mode"):
            D.dense(*given, activation="silu")
    given[which] = given[which].detach()
    assert D.dense(*given, activation="silu").shape == (5, 7)


def test_orthogonalize_carries_no_derivatives():
    x = torch.randn(30, 20, device="cuda", requires_grad=True)
    assert not D.ops.orthogonalize(x).requires_grad and not D.ops.orthogonalize(x.t()).requires_grad
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(torch.randn(30, 20, device="cuda"), torch.randn(30, 20, device="cuda"))
        assert torch.autograd.forward_ad.unpack_dual(D.ops.orthogonalize(x)).tangent is None
