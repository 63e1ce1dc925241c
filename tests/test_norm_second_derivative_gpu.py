"""The norm's gradient refuses to be differentiated, whatever asks for it."""
from __future__ import annotations

import pytest
import torch

import fastmoe_amd as fm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("with_residual", [False, True])
def test_a_penalty_on_the_gradient_is_refused(with_residual):
    """sum(y) has a constant gradient in y, so only the norm's own inputs carry the second derivative."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x, r, w = (torch.randn(*s, generator=g, device="cuda").requires_grad_(True)
               for s in ((4, 32), (4, 32), (32,)))
    leaves = [x, w] + ([r] if with_residual else [])
    for through in range(2):  # the gradient of x, of the weight
        y, _ = fm.add_rms_norm(x, w, r if with_residual else None)
        grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
        penalty = y.sum() + grads[through].square().sum()
        for wanted in leaves:
            with pytest.raises(RuntimeError, match="no gradient of its own"):
                torch.autograd.grad(penalty, wanted, retain_graph=True)
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            penalty.backward()
    # the first derivatives are those of a plain call
    y, _ = fm.add_rms_norm(x, w, r if with_residual else None)
    for a, b in zip(grads, torch.autograd.grad(y.sum(), leaves)):
        assert torch.equal(a, b) and not b.requires_grad
    # and a frozen weight's norm of a constant has nothing to refuse
    y, _ = fm.add_rms_norm(x.detach(), w)
    assert torch.autograd.grad(y.sum(), w, create_graph=True)[0].isfinite().all()
