"""What a beam's row adds up to: the logarithm of its sum of exponentials, wherever its largest logit lies.

A term is good to 3 u (u = 2^-24: an exponential's last place and two products of 32 bits; differences of 32-bit logits carry what they
are rounded off by), their sum is held in 64 bits, so its logarithm is off by 3 u and the score, rounded once, by half a unit of itself
more.  Asked for are 8 u, as everywhere."""
import math

import pytest
import torch

from dnatok_amd import lm_ops
from tests.support.attention_reference import U

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def scores_of(rows):
    """The best continuation of each row: its score and what that is in 64 bits."""
    got, tokens, parents = lm_ops.beam_select(rows.to(DEV), torch.zeros((rows.shape[0], 1), device=DEV), 1)
    wide = rows.double()
    want = wide.max(1).values - torch.logsumexp(wide, 1)
    assert torch.equal(tokens[:, 0].cpu(), wide.argmax(1).to(torch.int32))
    off = (got[:, 0].cpu().double() - want).abs() - (8 * U + U * want.abs())
    assert off.max().item() <= 0, off
    return got[:, 0].cpu()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [32000, 12301, 4096])
def test_a_peak_at_any_place(vocab, dtype):
    """One logit of 0 among many of -17: each of those is 2^-24.5 of the sum, all of them 1.3e-3."""
    places = [p for p in (0, 1, 3, 4, 7, 8, 31, 4095, 4096, 8191, 12300, 28675, 31999) if p < vocab]
    rows = torch.full((len(places), vocab), -17.0)
    rows[range(len(places)), places] = 0.0
    got = scores_of(rows.to(dtype))
    assert (got - got[0]).abs().max().item() <= 2 * U * abs(got[0].item())      # the same rows in another order


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups", [1, 300])
def test_beams_that_are_each_other_in_another_order(groups, dtype):
    """As many of a row's tokens as not are worth what a peak hides: the beam that is worth more by a part in 10^6 comes first."""
    g = torch.Generator().manual_seed(0)
    row = torch.full((32000,), -17.0)
    row[torch.randperm(32000, generator=g)[:3000]] = -12.0
    rows = torch.stack([row, row.flip(0), row[torch.randperm(32000, generator=g)]])
    for beam, at in enumerate((0, 31999, 17)):
        rows[beam, at] = 0.0
        rows[beam, 100:110] = -17.0
    rows = rows.to(dtype)
    values = torch.logsumexp(rows.double(), 1)
    scores = (values - values[0]).float()[None] + torch.tensor([[0.0, 1e-6, 2e-6]])
    order = [int(i) for i in (scores.double()[0] - values).argsort(descending=True)]
    assert (scores.double()[0] - values).sort().values.diff().min() > 8e-7
    got = lm_ops.beam_select(rows.repeat(groups, 1).to(DEV), scores.expand(groups, 3).contiguous().to(DEV), 3)
    assert got[2].cpu().tolist() == [order] * groups


@pytest.mark.parametrize("vocab", [32000, 1 << 20])
@pytest.mark.parametrize("gap", [8.3, 10.1, 15.9, 16.3])
def test_terms_that_are_all_rounded_the_same_way(vocab, gap):
    """The difference of two 32-bit logits is off by up to 2^-24 of 16, and all of these by the same."""
    low = torch.nextafter(torch.tensor(0.1) - gap, torch.tensor(0.0))
    rows = torch.full((2, vocab), low.item())
    rows[0, 5], rows[1, vocab - 1] = 0.1, 0.1
    scores_of(rows)


def test_rows_of_which_little_is_finite():
    """Infinities and the type's lowest value beside a peak add nothing, and NaN makes a beam none."""
    rows = torch.full((4, 9000), -math.inf)
    rows[:, 7000] = 1.5
    rows[1, :7000] = torch.finfo(torch.float32).min
    rows[2, 3:9000:2] = -17.0
    rows[2, 7000] = 1.5
    scores_of(rows)
    rows[3, 2] = math.nan
    got = lm_ops.beam_select(rows.to(DEV), torch.zeros((1, 4), device=DEV), 4)
    assert 3 not in got[2][got[1] >= 0].tolist()
    rows[3, 2] = math.inf
    got = lm_ops.beam_select(rows.to(DEV), torch.zeros((1, 4), device=DEV), 4)
    assert 3 not in got[2][got[1] >= 0].tolist()
