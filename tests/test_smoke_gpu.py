"""smoke() notices a wrong gradient, whichever of the three it is."""
from __future__ import annotations

import pytest
import torch

import __graft_entry__
import flash_atten

pytestmark = pytest.mark.gpu


def test_smoke_passes(gpu, capsys):
    __graft_entry__.smoke()
    assert "backward dQ dK dV" in capsys.readouterr().out


@pytest.mark.parametrize("which", [0, 1, 2], ids=["dq", "dk", "dv"])
@pytest.mark.parametrize("wrong", [lambda g: g * 1.01, lambda g: torch.full_like(g, float("nan"))], ids=["scaled", "nan"])
def test_smoke_checks_every_gradient(gpu, monkeypatch, which, wrong):
    right = flash_atten.attention_backward

    def backward(*args, **kwargs):
        grads = list(right(*args, **kwargs))
        grads[which] = wrong(grads[which])
        return tuple(grads)

    monkeypatch.setattr(flash_atten, "attention_backward", backward)
    with pytest.raises(AssertionError, match="backward"):
        __graft_entry__.smoke()
