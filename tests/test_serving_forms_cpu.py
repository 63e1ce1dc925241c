"""What the layers for serving refuse names the form that was asked for (CPU: before anything runs)."""
from __future__ import annotations

import pytest
import torch.nn as nn

import fastmoe_amd as fm


class Own(fm.MoEFeedForward):
    def forward(self, x):
        return super().forward(x) * 2


def make(kind=fm.MoEFeedForward):
    return kind(16, 8, 2, 1).bfloat16()


@pytest.mark.parametrize("form,other,bits", [("int8", "fp4", "8-bit"), ("fp4", "int8", "4-bit")])
def test_refusals_name_their_form(form, other, bits):
    def refusal(layer, error):
        with pytest.raises(error) as e:
            getattr(layer, form)()
        assert other not in str(e.value)
        return str(e.value)

    hooked, inner, near = make(), make(), make()
    hooked.register_forward_hook(lambda *a: None)
    inner.experts[1].register_forward_hook(lambda *a: None)
    near.experts[1][1] = nn.GELU("tanh")
    assert f"{form}() would lose" in refusal(make(Own), TypeError)
    assert f"{form}() makes" in refusal(hooked, ValueError)
    assert f"{bits} operators" in refusal(inner, ValueError)
    assert f"{bits} operators" in refusal(near, ValueError)
    block = fm.NormedMoEFeedForward(make())
    block.register_forward_hook(lambda *a: None)
    assert f"{form}() makes" in refusal(block, ValueError)
    if form == "fp4":
        block = fm.SandwichMoEFeedForward(make())
        block.register_forward_hook(lambda *a: None)
        assert "fp4() makes" in refusal(block, ValueError)
