"""Derivatives that an operator does not have are refused, not dropped: tangents of forward mode everywhere, gradients of what only
goes forwards."""
import pytest
import torch
from torch.autograd import forward_ad

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import DEV, logits_inputs, w4_inputs

pytestmark = pytest.mark.gpu


def calls(make):
    """Each operator with each of its inputs of numbers, one at a time, through ``make``."""
    x, gate, h0 = (torch.randn(shape, device=DEV) for shape in ((10, 8), (10, 8), (2, 8)))
    off = torch.tensor([0, 4, 10], device=DEV)
    state = torch.randn((10, 8), device=DEV)
    q, scales, z, xh, b = w4_inputs(2, 16, 64, 32, torch.bfloat16, True)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=64, group=32)
    a = logits_inputs(2, 40, [3, 3], torch.float32)
    yield "scan x", lambda: lm_ops.gated_scan(make(x), gate, off)
    yield "scan gate", lambda: lm_ops.gated_scan(x, make(gate), off)
    yield "scan h0", lambda: lm_ops.gated_scan(x, gate, off, h0=make(h0))
    yield "dense scan x", lambda: lm_ops.gated_scan(make(x.view(2, 5, 8)), gate.view(2, 5, 8))
    yield "step x", lambda: lm_ops.gated_step(make(x), gate, state)
    yield "step gate", lambda: lm_ops.gated_step(x, make(gate), state)
    yield "step state", lambda: lm_ops.gated_step(x, gate, make(state))
    yield "matvec x", lambda: matrix.matvec(make(xh))
    yield "matvec bias", lambda: matrix.matvec(xh, bias=make(b))
    yield "matvec scales", lambda: lm_ops.W4Matrix(q, make(scales), z, in_features=64, group=32).matvec(xh)
    for name in ("logits", "repetition", "presence", "frequency", "bias"):
        yield "logits " + name, lambda name=name: lm_ops.process_logits(**{**a, name: make(a[name])})


def test_tangents_are_refused():
    with forward_ad.dual_level():
        for name, call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
                pytest.fail(name)
        for name, call in calls(lambda t: t):                          # (inside a level, without tangents)
            call()


def test_gradients_of_what_only_goes_forwards_are_refused():
    for name, call in calls(lambda t: t.detach().clone().requires_grad_(True)):
        if "scan" in name:
            out = call()[0]
            assert out.requires_grad
            continue
        with pytest.raises(ValueError, match="no backward pass"):
            call()
            pytest.fail(name)
        with torch.no_grad():
            call()
