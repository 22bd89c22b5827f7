"""Tokens and parents of rows that begin at any place, and the tensors that reorder_rows is given."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_beam import DEV, TYPES, compare_scores, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 2, 5, 7])
def test_rows_at_any_place(shift, dtype):
    """16-bit rows that begin on no multiple of a wide load, their ties by beam, logit and token among them."""
    g = torch.Generator().manual_seed(8)
    wide = (torch.randn((8, 5011), generator=g) * 2).to(dtype)
    scores = -torch.rand((2, 4), generator=g)
    want, gap = plain(wide[:, shift:shift + 5001], scores, 6)
    assert gap > 1e-9
    got = lm_ops.beam_select(wide.to(DEV)[:, shift:shift + 5001], scores.to(DEV), 6)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    compare_scores(got[0], want[0], None)


def test_reorder_returns_what_it_was_given():
    tensors = [torch.arange(6 * n, device=DEV, dtype=torch.float32).view(6, n) for n in (1, 4, 33)]
    parents = torch.tensor([[2, 0, 1], [1, 1, 2]], dtype=torch.int32, device=DEV)
    rows = torch.tensor([2, 0, 1, 4, 4, 5], device=DEV)
    out = [torch.zeros_like(t) for t in tensors]
    got = lm_ops.reorder_rows(tensors, parents, out=out)
    assert len(got) == 3 and all(a is b for a, b in zip(got, out))
    assert all(torch.equal(o, t[rows]) for o, t in zip(out, tensors))
