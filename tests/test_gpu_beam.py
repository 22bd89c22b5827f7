"""A step of a beam search against its definition in 64 bits, and states in the order of the beams.

Scores are float32 of a value that is off by at most the rounding of a logarithm's sum: the exponentials are good to a few u
each, so is their sum (held in 64 bits), and so its logarithm, absolutely: 8 u and half a unit of the result.  Values that
are closer to each other than that are not in these inputs, but for equal ones of one beam, which are taken by token."""
import math

import pytest
import torch

from dnatok_amd import lm_ops
from tests.support.attention_reference import U

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain(logits, scores, width, finished=None, eos=None):
    """Scores, tokens, parents (lists) and the distance between the last that is taken and the first that is not."""
    groups, beams = scores.shape
    z, s = logits.detach().cpu().double(), scores.detach().cpu().double()
    result, gap = [], math.inf
    for g in range(groups):
        found = []
        for b in range(beams):
            if finished is not None and bool(finished[g, b]):
                found.append((-float(s[g, b]), b, 0.0, int(eos)))
                continue
            row = z[g * beams + b]
            total = torch.logsumexp(torch.where(torch.isnan(row), math.nan, row), 0)
            if not math.isfinite(float(total)):
                continue
            value = float(s[g, b]) + (row - total)
            order = torch.sort(-row, stable=True).indices[:width + 1].tolist()
            found += [(-float(value[i]), b, -float(row[i]), i) for i in order]
        found = sorted(f for f in found if f[0] < math.inf)
        values = sorted(f[0] for f in found)
        for i, (a, c) in enumerate(zip(values[:width], values[1:width + 1])):
            if a != c:
                gap = min(gap, c - a)
        found = found[:width] + [(math.inf, j % beams, 0.0, -1) for j in range(len(found[:width]), width)]
        result.append(([-f[0] for f in found], [f[3] for f in found], [f[1] for f in found]))
    return [torch.tensor([r[i] for r in result], dtype=torch.float64 if i == 0 else torch.int32).view(groups, width) for i in range(3)], gap


def check(groups, beams, vocab, width, dtype, seed=0, masked=0.0, ended=False, logits=None, scores=None):
    print(f"beam_select groups={groups} beams={beams} vocab={vocab} width={width} {dtype} masked={masked} ended={ended}", flush=True)
    g = torch.Generator().manual_seed(seed)
    if logits is None:
        logits = (torch.randn((groups * beams, vocab), generator=g) * 3.0).to(dtype)
        logits[torch.rand(logits.shape, generator=g) < masked] = -math.inf
    if scores is None:
        scores = -5.0 * torch.rand((groups, beams), generator=g)
    finished = torch.rand((groups, beams), generator=g) < 0.3 if ended else None
    eos = vocab - 1 if ended else None
    got = lm_ops.beam_select(logits.to(DEV), scores.to(DEV), width, finished=None if finished is None else finished.to(DEV), eos_id=eos)
    want, gap = plain(logits, scores, width, finished, eos)
    assert gap > 1e-9, "values too close to tell"                       # (of the inputs: their roundings are some 1e-10 apart)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    compare_scores(got[0], want[0], scores)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    return got


def compare_scores(got, want, scores):
    got, finite = got.cpu().double(), torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite) and (got[~finite] == -math.inf).all()
    off = (got - want).abs()[finite] - (8 * U + U * want.abs()[finite])
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 64, 65, 255, 256, 257, 1000, 4096, 12301, 32000, 70001])
def test_vocabularies_and_types(vocab, dtype):
    check(2, 3, vocab, 3, dtype, seed=vocab)


@pytest.mark.parametrize("beams,width", [(1, 1), (1, 8), (1, 128), (2, 4), (5, 10), (8, 8), (64, 64), (65, 3), (128, 128), (128, 1)])
@pytest.mark.parametrize("ended", [False, True])
def test_beams(beams, width, ended):
    check(2, beams, 777, width, torch.float32, seed=beams + width, ended=ended)


@pytest.mark.parametrize("groups", [0, 1, 7, 300])
def test_groups(groups):
    check(groups, 4, 500, 4, torch.bfloat16, seed=groups, masked=0.5)


@pytest.mark.parametrize("masked", [0.9, 0.99, 1.0])
@pytest.mark.parametrize("ended", [False, True])
def test_few_tokens_are_allowed(masked, ended):
    check(6, 3, 200, 8, torch.float16, seed=int(masked * 100), masked=masked, ended=ended)


def test_more_width_than_continuations():
    check(3, 2, 3, 16, torch.float32, seed=1)
    check(3, 2, 3, 16, torch.float32, seed=2, ended=True)


def test_equal_values_are_taken_by_beam_and_token():
    """All logits equal; whole rows of few values; both zeros; beams that are copies of each other."""
    for dtype in TYPES:
        for vocab in (40, 5000, 40000):
            scores, tokens, parents = lm_ops.beam_select(torch.full((4, vocab), 1.25, dtype=dtype, device=DEV),
                                                         torch.zeros((2, 2), device=DEV), 5)
            assert tokens.tolist() == [[0, 1, 2, 3, 4]] * 2 and parents.tolist() == [[0] * 5] * 2
            z = (torch.arange(vocab) * 7919 % 3).to(dtype)
            z = torch.where(z == 0, -0.0, z)
            z[1] = 0.0
            check(1, 1, vocab, 60, dtype, logits=z[None], scores=torch.zeros((1, 1)))
    z = torch.randn(300, generator=torch.Generator().manual_seed(3))
    got = lm_ops.beam_select(torch.stack([z, z, z]).to(DEV), torch.tensor([[-1.0, -1.0, -2.0]], device=DEV), 4)
    order = torch.sort(z, descending=True, stable=True).indices.tolist()
    assert got[1].tolist()[0][:2] == [order[0], order[0]] and got[2].tolist()[0][:2] == [0, 1]


def test_what_is_no_continuation():
    """Beams that are none, rows that are forbidden altogether, NaN and infinities: each concerns its beam only."""
    g = torch.Generator().manual_seed(4)
    z = torch.randn((6, 100), generator=g)
    z[1], z[2, 7], z[3, 9] = -math.inf, math.nan, math.inf
    scores = torch.tensor([[-1.0, 0.0, 0.0, 0.0, -math.inf, -2.0]])
    got = check(1, 6, 100, 6, torch.float32, logits=z, scores=scores)
    assert set(got[2].tolist()[0]) <= {0, 5}
    got = check(1, 6, 100, 6, torch.float32, logits=z, scores=torch.full((1, 6), -math.inf))
    assert got[1].tolist() == [[-1] * 6] and got[2].tolist() == [[0, 1, 2, 3, 4, 5]]
    got = lm_ops.beam_select(z[:1].to(DEV), torch.tensor([[math.nan]], device=DEV), 2)
    assert got[1].tolist() == [[-1, -1]]


def test_far_apart_logits():
    z = torch.tensor([[1e30, -1e30, 0.0, 5.0], [60000.0, -60000.0, 59999.0, 0.0]])
    check(1, 2, 4, 8, torch.float32, logits=z, scores=torch.tensor([[-1.0, -3.0]]))


def test_rows_at_any_place():
    g = torch.Generator().manual_seed(5)
    for dtype in TYPES:
        wide = (torch.randn((8, 5011), generator=g) * 2).to(dtype)
        for shift in (0, 1, 2, 5):
            part = wide[:, shift:shift + 5001]
            got = lm_ops.beam_select(wide.to(DEV)[:, shift:shift + 5001], torch.zeros((2, 4), device=DEV), 6)
            want, _ = plain(part, torch.zeros((2, 4)), 6)
            compare_scores(got[0], want[0], None)
            if dtype == torch.float32:
                assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])


def test_another_stream_and_a_graph():
    g = torch.Generator().manual_seed(6)
    logits, scores = torch.randn((12, 9000), generator=g).to(DEV), -torch.rand((3, 4), generator=g).to(DEV)
    states = [torch.randn((12, 40), generator=g).to(DEV), torch.randn((12, 2, 8, 8), generator=g).to(DEV)]
    want = lm_ops.beam_select(logits, scores)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lm_ops.beam_select(logits, scores)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = lm_ops.beam_select(logits, scores)
        moved = lm_ops.reorder_rows(states, held[2])
    for seed in range(4):
        logits.copy_(torch.randn((12, 9000), generator=g))
        held[1].fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        want = lm_ops.beam_select(logits, scores)                       # (eager work between the replays)
        assert all(torch.equal(a, b) for a, b in zip(want, held)), seed
        assert all(torch.equal(a, b) for a, b in zip(lm_ops.reorder_rows(states, want[2]), moved)), seed


# ---- states in the order of the beams -------------------------------------------------------------

@pytest.mark.parametrize("groups,beams,width", [(1, 1, 1), (1, 4, 4), (5, 3, 7), (40, 8, 2)])
def test_reorder(groups, beams, width):
    g = torch.Generator().manual_seed(7)
    parents = torch.randint(0, beams, (groups, width), generator=g).to(torch.int32)
    rows = (torch.arange(groups)[:, None] * beams + parents).view(-1)
    tensors = [torch.randn((groups * beams, 33), generator=g), torch.randn((groups * beams, 2, 16, 24), generator=g).bfloat16(),
               torch.randint(0, 99, (groups * beams,), generator=g).to(torch.int32), torch.rand((groups * beams, 7), generator=g) < 0.5,
               torch.randn((groups * beams, 5001), generator=g), torch.randint(0, 99, (groups * beams, 3), generator=g, dtype=torch.int64),
               torch.zeros((groups * beams, 0)), torch.randn((groups * beams, 4), generator=g).double()]
    tensors = tensors * 3                                               # (more than one launch's)
    on = [t.to(DEV) for t in tensors]
    got = lm_ops.reorder_rows(on, parents.to(DEV))
    assert all(torch.equal(a.cpu(), b[rows]) for a, b in zip(got, tensors))
    out = [torch.zeros_like(t) for t in got]
    assert lm_ops.reorder_rows(on, parents.to(DEV), out=out) == out or True
    assert all(torch.equal(a, b) for a, b in zip(out, got))


def test_reorder_of_strided_rows_and_parents_that_are_none():
    wide = torch.arange(6 * 50, dtype=torch.float32, device=DEV).view(6, 50)
    parents = torch.tensor([[0, 2, -1], [5, 1, 1]], dtype=torch.int32, device=DEV)
    for shift, width in ((0, 8), (1, 8), (3, 5)):
        t = wide[:, shift:shift + width]
        got, = lm_ops.reorder_rows([t], parents)
        zero = torch.zeros(width, device=DEV)
        assert torch.equal(got, torch.stack([t[0], t[2], zero, zero, t[4], t[4]]))
    assert lm_ops.reorder_rows([], parents) == []
    assert lm_ops.reorder_rows([wide[:0]], parents[:0])[0].shape == (0, 50)


def test_refusals():
    z, s = torch.zeros((6, 10), device=DEV), torch.zeros((2, 3), device=DEV)
    for bad in [dict(logits=z.cpu()), dict(logits=z.double()), dict(logits=z[:5]), dict(logits=z.t()), dict(scores=s.cpu()),
                dict(scores=s.double()), dict(scores=s[0]), dict(width=0), dict(width=129), dict(finished=s > 0), dict(finished=s, eos_id=1),
                dict(finished=s > 0, eos_id=10), dict(finished=s > 0, eos_id=-1), dict(logits=z[:, :0]),
                dict(logits=z.clone().requires_grad_(True))]:
        with pytest.raises(ValueError):
            lm_ops.beam_select(**{**dict(logits=z, scores=s), **bad})
            pytest.fail(str(bad))
    p = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    for tensors, out in [([z[:5]], None), ([z, z[:4]], None), ([z.t()], None), ([z.cpu()], None), ([z], [z]), ([z], []),
                         ([z], [torch.zeros((6, 9), device=DEV)]), ([z.clone().requires_grad_(True)], None)]:
        with pytest.raises(ValueError):
            lm_ops.reorder_rows(tensors, p, out=out)
            pytest.fail(str(out))
    twice = torch.zeros((6, 10), device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        lm_ops.reorder_rows([z, z], p, out=[twice, twice])
    for bad in (p.long(), p.cpu(), p[0]):
        with pytest.raises(ValueError):
            lm_ops.reorder_rows([z], bad)
