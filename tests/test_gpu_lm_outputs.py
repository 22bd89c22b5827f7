"""Outputs that the caller gives: results are those without, what would be read after it was written is refused, and gradients are not
wrong in silence."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import DEV, logits_inputs, w4_inputs

pytestmark = pytest.mark.gpu


def test_outputs_that_share_places_with_inputs():
    q, scales, z, x, b = w4_inputs(4, 64, 64, 32, torch.bfloat16, True)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=64, group=32)
    want = matrix.matvec(x)
    wide = torch.cat([x, torch.zeros_like(x)], 1)
    assert torch.equal(matrix.matvec(wide[:, :64], out=wide[:, 64:]), want) and torch.equal(wide[:, :64], x)
    for out in (x, wide[:, 1:65], wide[:, :64]):
        with pytest.raises(ValueError, match="overlap"):
            matrix.matvec(x if out is x else wide[:, :64], out=out)
    with pytest.raises(ValueError, match="overlap"):
        matrix.matvec(x, out=torch.zeros((1, 64), dtype=x.dtype, device=DEV).expand(4, 64))
    a = logits_inputs(4, 96, [5, 0, 7, 2], torch.bfloat16)
    z2 = torch.zeros((5, 96), dtype=torch.bfloat16, device=DEV)
    z2[:4] = a["logits"]
    want = lm_ops.process_logits(**a)
    with pytest.raises(ValueError, match="overlap"):
        lm_ops.process_logits(**{**a, "logits": z2[:4]}, out=z2[1:])
    buffer = torch.zeros((4, 96), device=DEV)                          # float32 results over 16-bit logits
    half = buffer.view(torch.bfloat16)[:, :96]
    half.copy_(a["logits"])
    with pytest.raises(ValueError, match="overlap"):
        lm_ops.process_logits(**{**a, "logits": half}, out=buffer)
    assert torch.equal(lm_ops.process_logits(**{**a, "logits": z2[:4]}, out=z2[:4]), want)
    x1, gate, state = (torch.randn((3, 8), device=DEV) for _ in range(3))
    both = torch.randn((4, 8), device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        lm_ops.gated_step(x1, gate, both[:3], out_state=both[1:])
    y, h = lm_ops.gated_step(x1, gate, state)
    assert torch.equal(lm_ops.gated_step(x1, gate, both[:3].copy_(state), out_state=both[:3])[1], h)


def test_an_input_of_a_product_is_no_output():
    """In place even with a square matrix: other workgroups still read the rows."""
    q, scales, z, x, b = w4_inputs(4, 64, 64, 32, torch.bfloat16, True)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=64, group=32)
    with pytest.raises(ValueError, match="overlap"):
        matrix.matvec(x, out=x)


def test_gradients_through_what_was_overwritten_are_refused():
    a = logits_inputs(2, 40, [3, 3], torch.float32)
    w = a["logits"].requires_grad_(True)
    h = w * 2.0
    loss = (h * h).sum()
    with torch.no_grad():
        lm_ops.process_logits(**{**a, "logits": h}, out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with pytest.raises(ValueError, match="no backward pass"):
        lm_ops.process_logits(**{**a, "logits": a["logits"].detach()}, out=torch.zeros_like(w).requires_grad_(True))
