"""Rows of an embedding and the gradient of its weights against sums in 64 bits.

Tolerances.  A row is one product, rounded at most twice: u of itself and half a unit of its type.  A gradient's cell is a sum of n
values: sums of a part of the tokens, and sums of those, at most n roundings each of at most the sum of the sizes, and a
product: (n + 2) u sum|dy| scale, and half a unit of its type."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support.attention_reference import HALF, TINY, U

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(n, vocab, dim, dtype, seed=0, skew=2.0, idtype=torch.int32, outside=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(n, generator=g, dtype=torch.float64) ** skew * vocab).long().clamp(max=max(vocab - 1, 0))
    if outside:
        wrong = torch.tensor([-1, vocab, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (n,), generator=g)]
        ids = torch.where(torch.rand(n, generator=g) < outside, wrong, ids)
    weight = torch.randn((vocab, dim), generator=g).to(dtype).to(DEV)
    return ids.to(idtype).to(DEV), weight, torch.randn((n, dim), generator=g).to(dtype).to(DEV)


def check(n, vocab, dim, dtype, scale=1.0, train=True, **kw):
    print(f"embedding n={n} vocab={vocab} dim={dim} {dtype} scale={scale} {kw}", flush=True)
    ids, weight, dy = inputs(n, vocab, dim, dtype, **kw)
    weight.requires_grad_(train)
    y = lm_ops.embedding(ids, weight, scale=scale)
    compare(y, ids, weight, scale)
    if train:
        grad, = torch.autograd.grad(y, weight, dy)
        compare_grad(grad, ids, dy, scale)
        return grad


def compare(y, ids, weight, scale):
    hi, hw = ids.cpu().long(), weight.detach().cpu().double()
    known = (hi >= 0) & (hi < hw.shape[0])
    want = torch.zeros((*hi.shape, hw.shape[1]), dtype=torch.float64)
    want[known] = np.float64(np.float32(scale)) * hw[hi[known]]
    assert y.shape == want.shape and y.dtype == weight.dtype
    off = (y.detach().cpu().double() - want).abs() - want.abs() * (U + HALF[y.dtype] * (1 + 2 * U)) - TINY[y.dtype]
    assert off.numel() == 0 or off.max().item() <= 0


def compare_grad(grad, ids, dy, scale):
    hi, hd = ids.cpu().reshape(-1).long(), dy.cpu().double().reshape(-1, grad.shape[1])
    known = (hi >= 0) & (hi < grad.shape[0])
    want, size = (torch.zeros(grad.shape, dtype=torch.float64).index_add_(0, hi[known], t[known]) * np.float64(np.float32(scale))
                  for t in (hd, hd.abs()))
    count = torch.bincount(hi[known], minlength=grad.shape[0]).double()[:, None]
    slack = (count + 2) * U * size.abs() + HALF[grad.dtype] * want.abs() * (1 + 2 * HALF[grad.dtype]) + TINY[grad.dtype]
    off = (grad.cpu().double() - want).abs() - slack
    assert torch.isfinite(grad).all() and (off.numel() == 0 or off.max().item() <= 0), off.max().item()
    assert (grad.cpu()[count[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 255, 256, 257, 1000, 4095, 4096, 4097, 9000])
def test_tokens_and_types(n, dtype):
    check(n, 300, 72, dtype, 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 64, 65, 127, 128, 129, 130])
@pytest.mark.parametrize("vocab,dim", [(1, 40), (3, 5), (11, 203), (5000, 64), (270001, 8)])
def test_few_tokens(vocab, dim, n, dtype):
    check(n, vocab, dim, dtype, -0.25, outside=0.2, seed=n, idtype=torch.int64 if n % 2 else torch.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 2, 3, 7, 8, 9, 63, 64, 65, 100, 203, 255, 256, 257, 512, 513, 1000, 1024, 2048, 2049])
def test_dims(dim, dtype):
    check(700, 50, dim, dtype, 3.0)


@pytest.mark.parametrize("vocab", [1, 2, 5, 12, 255, 256, 257, 4096, 32000, 65535, 65536, 65537, 200000])
@pytest.mark.parametrize("n", [50, 6000])
def test_vocabularies(vocab, n):
    check(n, vocab, 24, torch.bfloat16)
    check(n, vocab, 20, torch.float32, skew=6.0)


@pytest.mark.parametrize("vocab", [1, 4, 12, 5000])
def test_many_tokens(vocab):
    """Few ids, each of them very often; all ids equal; ascending and falling ids."""
    check(60013, vocab, 40, torch.float32)
    for order in (lambda i: i % vocab, lambda i: vocab - 1 - i * vocab // 60013, lambda i: i * 0 + vocab // 2):
        ids = order(torch.arange(60013)).to(torch.int32).to(DEV)
        _, weight, dy = inputs(60013, vocab, 40, torch.bfloat16, 3)
        leaf = weight.requires_grad_(True)
        grad, = torch.autograd.grad(lm_ops.embedding(ids, leaf, scale=0.25), leaf, dy)
        compare_grad(grad, ids, dy, 0.25)


@pytest.mark.parametrize("idtype", [torch.int32, torch.int64])
def test_ids_outside_the_table(idtype):
    check(5000, 100, 33, torch.float16, idtype=idtype, outside=0.3)
    check(300, 100, 16, torch.float32, idtype=idtype, outside=1.0)
    ids = torch.tensor([2 ** 32 + 1, -2 ** 32, 1, -2 ** 63, 2 ** 63 - 1], device=DEV)
    weight = torch.ones((4, 8), device=DEV)
    assert lm_ops.embedding(ids, weight).sum(1).tolist() == [0, 0, 8, 0, 0]
    assert (lm_ops.embedding(ids, weight[:0]) == 0).all()               # no table at all


def test_shapes_and_strides():
    ids, weight, dy = inputs(24 * 7, 60, 40, torch.bfloat16, 4)
    wide = torch.zeros((60, 91), dtype=torch.bfloat16, device=DEV)
    for shift in (0, 1, 8):
        wide[:, shift:shift + 40] = weight
        table = wide[:, shift:shift + 40].detach().requires_grad_(True)  # rows at any place
        y = lm_ops.embedding(ids.view(24, 7), table, scale=2.0)
        compare(y, ids.view(24, 7), weight, 2.0)
        out = torch.zeros((24, 7, 91), dtype=torch.bfloat16, device=DEV)
        out[:, :, shift:shift + 40] = dy.view(24, 7, 40)
        grad, = torch.autograd.grad(y, table, out[:, :, shift:shift + 40])
        compare_grad(grad, ids, dy, 2.0)
    y = lm_ops.embedding(ids.view(24, 7).t(), table)                     # (ids in another order are copied)
    assert torch.equal(y, lm_ops.embedding(ids.view(24, 7).t().contiguous(), table))
    grad, = torch.autograd.grad(lm_ops.embedding(ids, table).float().sum(), table)       # a broadcast gradient
    compare_grad(grad, ids, torch.ones_like(dy), 1.0)


def test_infinities_and_nan_stay_in_their_row():
    ids, weight, dy = inputs(3000, 20, 24, torch.bfloat16, 5)
    dy[ids == 3] = float("inf")
    dy[7] = float("nan")
    leaf = weight.requires_grad_(True)
    y = lm_ops.embedding(ids, leaf)
    grad, = torch.autograd.grad(y, leaf, dy)
    odd = {3, int(ids[7])}
    for v in range(20):
        assert bool(torch.isfinite(grad[v]).all()) == (v not in odd), v
    assert torch.isinf(grad[3]).all() or int(ids[7]) == 3


def test_the_same_every_time_and_with_other_tokens_between():
    ids, weight, dy = inputs(50000, 700, 96, torch.float32, 6)
    leaf = weight.requires_grad_(True)
    first, = torch.autograd.grad(lm_ops.embedding(ids, leaf), leaf, dy)
    for _ in range(4):
        again, = torch.autograd.grad(lm_ops.embedding(ids, leaf), leaf, dy)
        assert torch.equal(first, again)


def test_another_stream_and_a_graph():
    ids, weight, dy = inputs(7000, 900, 64, torch.bfloat16, 7)
    leaf = weight.requires_grad_(True)
    want = lm_ops.embedding(ids, leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lm_ops.embedding(ids, leaf)
        grad, = torch.autograd.grad(got, leaf, dy)
    side.synchronize()
    assert torch.equal(got, want)
    compare_grad(grad, ids, dy, 1.0)
    del want, got, grad
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lm_ops.embedding(ids, leaf, scale=1.5)
        grad, = torch.autograd.grad(y, leaf, dy)
    for seed in range(4):
        new = inputs(7000, 900, 64, torch.bfloat16, 20 + seed, skew=1.0 + seed)
        ids.copy_(new[0])
        dy.copy_(new[2])
        grad.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        compare_grad(grad, new[0], new[2], 1.5)
        assert torch.equal(y, lm_ops.embedding(new[0], leaf, scale=1.5))  # (eager work between the replays)


def test_refusals():
    ids, weight, dy = inputs(10, 5, 8, torch.float32)
    for bad in [(ids.cpu(), weight), (ids.float(), weight), (ids.short(), weight), (ids, weight.double()), (ids, weight[0]),
                (ids, weight.t()), (ids, weight.cpu())]:
        with pytest.raises(ValueError):
            lm_ops.embedding(*bad)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            lm_ops.embedding(ids, weight, scale=scale)


def test_narrow_rows_of_many_tokens():
    """Rows of a few bytes lie next to each other in a wave, two rounds of them where there are very many."""
    n, vocab = 17_000_003, 50
    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(-1, vocab + 1, (n,), generator=g, device=DEV, dtype=torch.int32)
    weight = torch.randn((vocab, 3), generator=g, device=DEV).bfloat16()
    y = lm_ops.embedding(ids, weight)
    known = (ids >= 0) & (ids < vocab)
    for lo in range(0, n, 4_000_000):
        i, k = ids[lo:lo + 4_000_000].long().clamp(0, vocab - 1), known[lo:lo + 4_000_000]
        assert torch.equal(y[lo:lo + 4_000_000], torch.where(k[:, None], weight[i], 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 3, 40, 2000])
@pytest.mark.parametrize("dim", [1, 4, 9, 16, 33, 64, 100, 128, 129, 200, 256])
def test_gradients_of_narrow_rows(dim, vocab, dtype):
    check(20011, vocab, dim, dtype, 0.125, outside=0.05, seed=dim)


@pytest.mark.parametrize("vocab", [1, 2, 5])
@pytest.mark.parametrize("run", [255, 256, 257, 271, 272, 273, 300])
def test_runs_that_end_at_tiles(run, vocab):
    """Ids of so many tokens each (tiles have sixteen): runs that begin and end at tiles, that one wave joins and that several do."""
    ids = torch.arange(vocab * run, device=DEV, dtype=torch.int32) // run
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(run)).to(DEV)]
    g = torch.Generator().manual_seed(vocab)
    weight = torch.randn((vocab + 1, 24), generator=g).to(DEV).requires_grad_(True)
    dy = torch.randn((ids.numel(), 24), generator=g).to(DEV)
    grad, = torch.autograd.grad(lm_ops.embedding(ids, weight), weight, dy)
    compare_grad(grad, ids, dy, 1.0)
