"""Linear attention with a decay for each head against the recurrence in 64 bits (tolerances: attention_reference)."""
import itertools

import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import attention_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(lengths, heads, kv, dim_k, dim_v, dtype, seed=0, room=0, decay=None):
    """Parts of one projection's output, half-lives from one token to hundreds, states, outgoing gradients."""
    g = torch.Generator().manual_seed(seed)
    off = [0] + list(itertools.accumulate(lengths))
    total = off[-1] + room
    both = torch.randn((total, heads * dim_k + kv * (dim_k + dim_v)), generator=g).to(dtype).to(DEV)
    q, k, v = both.split([heads * dim_k, kv * dim_k, kv * dim_v], 1)
    q, k, v = q.view(total, heads, dim_k), k.view(total, kv, dim_k), v.view(total, kv, dim_v)
    if decay is None:
        decay = torch.log1p(-torch.exp2(-1.0 - 9.0 * torch.rand(heads, generator=g)))
    state = (len(lengths), heads, dim_k, dim_v)
    h0, dlast = (torch.randn(state, generator=g).to(DEV) for _ in range(2))
    dy = torch.randn((total, heads, dim_v), generator=g).to(dtype).to(DEV)
    return q, k, v, decay.to(DEV), off, h0, dy, dlast


def run(q, k, v, decay, off, h0, dy, dlast, scale=None, reverse=False, train=True):
    """All results, as the reference names them."""
    offsets = torch.tensor(off, device=DEV)
    leaves = [t.detach().requires_grad_(train) for t in (q, k, v)] + ([] if h0 is None else [h0.detach().requires_grad_(train)])
    y, last = lm_ops.linear_attention(*leaves[:3], decay, offsets, h0=None if h0 is None else leaves[3], scale=scale, reverse=reverse)
    got = {"y": y, "last": last}
    if train:
        got.update(zip(("dq", "dk", "dv", "dh0"), torch.autograd.grad((y, last), leaves, (dy, dlast))))
    return got


def check(lengths, heads, kv, dim_k, dim_v, dtype, reverse=False, start=True, train=True, seed=0, scale=None, room=0, decay=None):
    print(f"linear_attention rows={len(lengths)} total={sum(lengths)} heads={heads}/{kv} dims={dim_k}x{dim_v} {dtype} reverse={reverse} "
          f"start={start} train={train}", flush=True)
    q, k, v, ld, off, h0, dy, dlast = inputs(lengths, heads, kv, dim_k, dim_v, dtype, seed, room, decay)
    h0 = h0 if start else None
    got = run(q, k, v, ld, off, h0, dy, dlast, scale, reverse, train)
    compare(got, (q, k, v, ld, off, h0, dy, dlast), dtype, scale, reverse, max(lengths, default=0))


def compare(got, data, dtype, scale, reverse, longest):
    q, k, v, ld, off, h0, dy, dlast = data
    train = "dq" in got
    args = (q, k, v, ld, off, h0, scale, reverse) + ((dy, dlast) if train else ())
    want, size = ref.attention(*args), ref.attention(*args, sizes=True)
    count = ref.roundings(dtype, q.shape[2], v.shape[2], longest) + q.shape[1] // k.shape[1]
    for name, value in got.items():
        ref.check(value, want[name], size[name], torch.float32 if name in ("last", "dh0") else dtype, count, name)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("reverse", [False, True])
def test_one_row(length, reverse):
    check([length], 2, 2, 32, 48, torch.bfloat16, reverse)


@pytest.mark.parametrize("length", [511, 512, 513, 1100])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_one_row_in_pieces(length, reverse, dtype):
    check([length], 2, 1, 40, 24, dtype, reverse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(1, 1), (1, 128), (128, 1), (3, 5), (16, 16), (33, 31), (63, 65), (64, 64), (64, 128), (128, 64), (127, 120),
                                  (128, 128)])
def test_dims_and_types(dims, dtype):
    check([70, 1, 130], 2, 2, *dims, dtype, reverse=dims[0] % 2 == 0)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (6, 2), (4, 1), (9, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_heads(heads, kv, dtype):
    check([90, 3, 600], heads, kv, 20, 36, dtype)


RAGGED = {"empty_rows": [0, 0, 5, 0, 300, 0, 0, 1, 16, 0, 240, 0],
          "only_empty": [0, 0, 0],
          "single_tokens": [1] * 700,
          "rows_at_cuts": [512, 512, 0, 1024, 0, 0, 511, 1],
          "one_before_cuts": [511, 512, 1, 513, 700],
          "many_empty": [0] * 500 + [3] + [0] * 500 + [40] + [0] * 300,
          "mixed": [100, 1, 1700, 3, 0, 517, 64, 63, 65, 1]}


@pytest.mark.parametrize("name", sorted(RAGGED))
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("start", [False, True])
def test_ragged_rows(name, reverse, start):
    check(RAGGED[name], 2, 1, 16, 24, torch.float32, reverse, start)


@pytest.mark.parametrize("reverse", [False, True])
def test_tokens_in_no_row(reverse):
    """In front of the first row and behind the last one: zeros, whatever is there."""
    lengths, room = [30, 0, 600], 90
    q, k, v, ld, off, h0, dy, dlast = inputs(lengths, 2, 1, 24, 40, torch.bfloat16, 1, room)
    off = [o + 25 for o in off]
    for t in (q, k, v, dy):
        t[:25], t[off[-1]:] = float("nan"), float("inf")
    got = run(q, k, v, ld, off, h0, dy, dlast, reverse=reverse)
    for name in ("y", "dq", "dk", "dv"):
        assert (got[name][:25] == 0).all() and (got[name][off[-1]:] == 0).all(), name
    cut = slice(25, off[-1])
    inner = tuple(t[cut] for t in (q, k, v)) + (ld, [o - 25 for o in off], h0, dy[cut], dlast)
    compare({n: t[cut] if n in ("y", "dq", "dk", "dv") else t for n, t in got.items()}, inner, torch.bfloat16, None, reverse, 600)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decay", [0.0, -1e-6, -3.0, -60.0, -3e38, float("-inf")])
def test_decays(decay, dtype):
    check([200, 700], 2, 2, 32, 32, dtype, reverse=decay < -1, decay=torch.full((2,), decay))


@pytest.mark.parametrize("scale", [1.0, -0.01, 300.0])
def test_scales(scale):
    for dtype in TYPES:
        check([150, 20], 2, 1, 24, 40, dtype, scale=scale)


def test_a_long_row_with_slow_decays():
    """A factor rounded once and multiplied thousands of times would be seen here."""
    check([20011, 7], 2, 2, 8, 8, torch.bfloat16, decay=torch.tensor([-1e-5, -3e-4]), seed=3)
    check([20011, 7], 2, 2, 8, 8, torch.float32, reverse=True, decay=torch.tensor([-1e-5, -3e-4]), seed=4)


@pytest.mark.parametrize("sizes", [(300.0, 300.0, 1e-4), (1e-3, 1e-3, 1e-3), (1.0, 200.0, 200.0)])
def test_float16_scores_and_states_beyond_its_range(sizes):
    q, k, v, ld, off, h0, dy, dlast = inputs([200, 70], 2, 2, 64, 32, torch.float16, 5)
    q, k, v = ((t * s).contiguous() for t, s in zip((q, k, v), sizes))
    h0 = h0 * sizes[1] * sizes[2]
    scale = 1.0 / (64 * max(1.0, sizes[0] * sizes[1] * sizes[2]))
    got = run(q, k, v, ld, off, h0, dy, dlast, scale, train=False)
    compare(got, (q, k, v, ld, off, h0, dy, dlast), torch.float16, scale, False, 200)


def test_rows_keep_apart_and_nothing_reaches_earlier_steps():
    for dtype, reverse in itertools.product(TYPES, (False, True)):
        q, k, v, ld, off, h0, dy, dlast = inputs([40, 700, 90], 2, 2, 48, 64, dtype, 6)
        offsets = torch.tensor(off, device=DEV)
        clean, _ = lm_ops.linear_attention(q, k, v, ld, offsets, h0=h0, reverse=reverse)
        for value, which in itertools.product((float("nan"), float("inf"), float("-inf")), range(3)):
            bad = [t.clone() for t in (q, k, v)]
            at = 40 + 333
            bad[which][at, 1, 5] = value
            y, last = lm_ops.linear_attention(*bad, ld, offsets, h0=h0, reverse=reverse)
            before = slice(at + 1, 740) if reverse else slice(40, at)
            for part in (slice(0, 40), slice(740, 830), before):
                assert torch.equal(y[part], clean[part]), (dtype, reverse, value, which)
            assert torch.equal(y[:, 0], clean[:, 0])                    # the other head
            if which == 2:                                              # a value reaches its own column only
                others = [c for c in range(64) if c != 5]
                assert torch.equal(y[:, 1, others], clean[:, 1, others])
            assert not torch.isfinite(y[at, 1]).all()


def test_gradients_keep_rows_apart():
    q, k, v, ld, off, h0, dy, dlast = inputs([40, 200, 90], 2, 1, 48, 64, torch.bfloat16, 7)
    clean = run(q, k, v, ld, off, h0, dy, dlast)
    bad = v.clone()
    bad[100] = float("nan")
    got = run(q, k, bad, ld, off, h0, dy, dlast)
    for part in (slice(0, 40), slice(240, 330)):
        for name in ("dq", "dk", "dv"):
            assert torch.equal(got[name][part], clean[name][part]), name
    assert torch.equal(got["dh0"], clean["dh0"])                        # (a state's gradient does not depend on values)


@pytest.mark.parametrize("dtype", TYPES)
def test_any_place_and_distance(dtype):
    """Heads that begin on no multiple of a wide load, tokens at odd distances, heads apart, one token for all."""
    g = torch.Generator().manual_seed(8)
    wide = torch.randn((150, 401), generator=g).to(dtype).to(DEV)
    off, ld = [0, 61, 150], torch.tensor([-0.1, -0.01], device=DEV)
    for shift in (0, 1, 3):
        q, k, v = (torch.as_strided(wide, (150, 2, d), (401, 70, 1), shift + at) for at, d in ((0, 40), (140, 40), (260, 24)))
        got = run(q, k, v, ld, off, None, torch.ones((150, 2, 24), dtype=dtype, device=DEV).expand(150, 2, 24),
                  torch.zeros((2, 2, 40, 24), device=DEV))
        compare(got, (q, k, v, ld, off, None, torch.ones((150, 2, 24), dtype=dtype), torch.zeros((2, 2, 40, 24))), dtype, None, False, 89)
    one = wide[:1, :40].view(1, 1, 40).expand(150, 2, 40)
    y, last = lm_ops.linear_attention(one, one, one, ld, torch.tensor(off, device=DEV))
    compare({"y": y, "last": last}, (one, one, one, ld, off, None, None, None), dtype, None, False, 89)


def test_dense_rows_are_packed_ones():
    q, k, v, ld, off, h0, dy, dlast = inputs([129] * 6, 4, 2, 32, 48, torch.bfloat16, 9)
    want = lm_ops.linear_attention(q, k, v, ld, torch.tensor(off, device=DEV), h0=h0)
    dense = [t.reshape(6, 129, t.shape[1], t.shape[2]) for t in (q, k, v)]
    got = lm_ops.linear_attention(*dense, ld, h0=h0)
    compare({"y": got[0].view(-1, 4, 48), "last": got[1]}, (q, k, v, ld, off, h0, None, None), torch.bfloat16, None, False, 129)
    assert got[0].shape == (6, 129, 4, 48) and want[0].shape == (774, 4, 48)
    leaves = [t.detach().clone().requires_grad_(True) for t in dense]
    y, _ = lm_ops.linear_attention(*leaves, ld)
    y.float().sum().backward()                                          # (a broadcast gradient; none for the last states)
    ones = torch.ones((774, 4, 48), dtype=torch.bfloat16)
    grads = {n: t.grad.view(774, *t.shape[2:]) for n, t in zip(("dq", "dk", "dv"), leaves)}
    compare(grads, (q, k, v, ld, off, None, ones, None), torch.bfloat16, None, False, 129)


def test_only_the_last_states_have_gradients():
    q, k, v, ld, off, h0, dy, dlast = inputs([70, 0, 600], 2, 2, 24, 40, torch.float32, 10)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, h0)]
    _, last = lm_ops.linear_attention(*leaves[:3], ld, torch.tensor(off, device=DEV), h0=leaves[3])
    got = dict(zip(("dq", "dk", "dv", "dh0"), torch.autograd.grad(last, leaves, dlast)))
    compare(got, (q, k, v, ld, off, h0, torch.zeros_like(dy), dlast), torch.float32, None, False, 600)
    assert not lm_ops.linear_attention(q.detach(), k.detach(), v.detach(), ld, torch.tensor(off, device=DEV))[0].requires_grad


def test_no_rows_and_no_tokens():
    ld = torch.zeros(2, device=DEV)
    q, k, v, h0 = (torch.zeros(s, device=DEV) for s in ((0, 2, 8), (0, 1, 8), (0, 1, 4), (3, 2, 8, 4)))
    h0 += 2.5
    y, last = lm_ops.linear_attention(q, k, v, ld, torch.zeros(1, dtype=torch.int64, device=DEV))
    assert y.shape == (0, 2, 4) and last.shape == (0, 2, 8, 4)
    y, last = lm_ops.linear_attention(q, k, v, ld, torch.zeros(4, dtype=torch.int64, device=DEV), h0=h0)
    assert y.shape == (0, 2, 4) and torch.equal(last, h0)
    y, last = lm_ops.linear_attention(*(t.view(3, 0, *t.shape[1:]) for t in (q, k, v)), ld, h0=h0)
    assert y.shape == (3, 0, 2, 4) and torch.equal(last, h0)


def test_gradient_against_differences():
    """The kernel's own values, a little to either side along a random direction."""
    q, k, v, ld, off, h0, dy, dlast = inputs([150, 0, 37, 1], 2, 1, 24, 16, torch.float32, 11)
    offsets = torch.tensor(off, device=DEV)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, h0)]

    def value(ts):
        y, last = lm_ops.linear_attention(*ts[:3], ld, offsets, h0=ts[3])
        return (y.double() * dy.double()).sum() + (last.double() * dlast.double()).sum()

    grads = torch.autograd.grad(value(leaves), leaves)
    sizes = ref.attention(q, k, v, ld, off, h0, sizes=True)
    weight = float((sizes["y"] * dy.cpu().double().abs()).sum() + (sizes["last"] * dlast.cpu().double().abs()).sum())
    g = torch.Generator().manual_seed(1)
    for i in range(4):
        way = torch.randn(leaves[i].shape, generator=g).to(DEV)
        eps = 0.5                                  # (linear in each argument: the difference is exact up to rounding)
        with torch.no_grad():
            up = value([t + eps * way if j == i else t for j, t in enumerate(leaves)])
            down = value([t - eps * way if j == i else t for j, t in enumerate(leaves)])
        slope = float((grads[i].double() * way.double()).sum())
        diff = float((up - down) / (2 * eps))
        # roundings of values whose terms weigh at most some four times `weight` (the argument is moved by half of a normal number)
        assert abs(slope - diff) <= 4 * weight * 64 * ref.U * 2 / eps, i


def test_the_same_every_time():
    for dtype in TYPES:
        q, k, v, ld, off, h0, dy, dlast = inputs([2000, 3, 900], 4, 2, 64, 64, dtype, 12)
        first = None
        for _ in range(4):
            out = list(run(q, k, v, ld, off, h0, dy, dlast).values())
            first = [t.detach().clone() for t in out] if first is None else first
            assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_on_another_stream_and_in_a_graph():
    q, k, v, ld, off, h0, dy, dlast = inputs([1500, 0, 500], 4, 2, 64, 48, torch.bfloat16, 13)
    offsets = torch.tensor(off, device=DEV)
    want = lm_ops.linear_attention(q, k, v, ld, offsets, h0=h0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lm_ops.linear_attention(q, k, v, ld, offsets, h0=h0)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    held = [t.clone().requires_grad_(True) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, last = lm_ops.linear_attention(*held, ld, offsets, h0=h0)
        grads = torch.autograd.grad((y, last), held, (dy, dlast))
    for seed in range(4):
        new = inputs([1500, 0, 500], 4, 2, 64, 48, torch.bfloat16, 20 + seed)
        with torch.no_grad():
            for t, n in zip(held, new):
                t.copy_(n)
        y.detach().fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(*new[:3], ld, off, h0, dy, dlast)                   # (eager work between the replays)
        for name, t in zip(("y", "last", "dq", "dk", "dv"), (y, last, *grads)):
            assert torch.equal(t, eager[name]), (seed, name)


# ---- one token of each row ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 8, 8, 64, 64), (7, 6, 2, 33, 20), (3, 2, 1, 128, 128), (60, 4, 4, 16, 125), (2, 2, 2, 128, 3)])
def test_step(shape, dtype):
    rows, heads, kv, dk, dv = shape
    q, k, v, ld, off, h0, _, _ = inputs([1] * rows, heads, kv, dk, dv, dtype, 14)
    data = (q, k, v, ld, off, h0, None, None)
    y, new = lm_ops.linear_attention_step(q, k, v, ld, h0)
    compare({"y": y, "last": new}, data, dtype, None, False, 1)
    y2, same = lm_ops.linear_attention_step(q, k, v, ld, h0, out_state=h0)          # in place
    assert same is h0 and torch.equal(h0, new) and torch.equal(y2, y)
    y0, n0 = lm_ops.linear_attention_step(q, k, v, ld, scale=2.0)
    compare({"y": y0, "last": n0}, (q, k, v, ld, off, None, None, None), dtype, 2.0, False, 1)


def test_steps_are_the_rows():
    q, k, v, ld, off, h0, _, _ = inputs([50] * 3, 4, 2, 32, 40, torch.bfloat16, 15)
    want, size = (ref.attention(q, k, v, ld, off, h0, sizes=s) for s in (False, True))
    state = h0.clone()
    count = ref.roundings(torch.float32, 32, 40, 50) + 50
    for t in range(50):
        y, _ = lm_ops.linear_attention_step(q[t::50], k[t::50], v[t::50], ld, state, out_state=state)
        ref.check(y, want["y"][t::50], size["y"][t::50], torch.bfloat16, count, t)
    ref.check(state, want["last"], size["last"], torch.float32, count, "state")
    y, last = lm_ops.linear_attention(q, k, v, ld, torch.tensor(off, device=DEV), h0=h0)
    ref.check(last, want["last"], size["last"], torch.float32, count, "last")


def test_step_with_a_decay_of_everything():
    q, k, v, _, off, h0, _, _ = inputs([1] * 4, 2, 2, 16, 16, torch.float32, 16)
    ld = torch.tensor([float("-inf"), 0.0], device=DEV)
    _, new = lm_ops.linear_attention_step(q, k, v, ld, h0)
    compare({"last": new}, (q, k, v, ld, off, h0, None, None), torch.float32, None, False, 1)


def test_refusals():
    q, k, v, ld, off, h0, dy, dlast = inputs([5, 6], 4, 2, 8, 12, torch.float32)
    offsets = torch.tensor(off, device=DEV)
    ok = dict(q=q, k=k, v=v, log_decay=ld, offsets=offsets, h0=h0)
    lm_ops.linear_attention(**ok)
    bad = [dict(q=q.cpu()), dict(q=q.double()), dict(k=k.bfloat16()), dict(k=k[:, :, :7]), dict(v=v[:10]), dict(v=v[:, :1]),
           dict(q=q[:, :3]), dict(log_decay=ld[:3]), dict(log_decay=ld.double()), dict(offsets=None), dict(offsets=offsets.int()),
           dict(h0=h0[:1]), dict(h0=h0.bfloat16()), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(q=q.transpose(1, 2)), dict(v=v.repeat(1, 1, 11)), dict(q=q.repeat(1, 1, 17), k=k.repeat(1, 1, 17)),
           dict(log_decay=ld.clone().requires_grad_(True)), dict(offsets=offsets[:0]), dict(offsets=offsets[:1])]
    for change in bad:
        with pytest.raises(ValueError):
            lm_ops.linear_attention(**{**ok, **change})
            pytest.fail(str(list(change)))
    step = dict(q=q[:2], k=k[:2], v=v[:2], log_decay=ld, state=h0)
    lm_ops.linear_attention_step(**step)
    for change in [dict(state=h0[:1]), dict(out_state=h0.double()), dict(q=q[:1]), dict(q=q[:2].clone().requires_grad_(True)),
                   dict(state=h0.clone().requires_grad_(True)), dict(scale=0.0), dict(out_state=h0.view(-1)[:-1])]:
        with pytest.raises(ValueError):
            lm_ops.linear_attention_step(**{**step, **change})
            pytest.fail(str(list(change)))
    twice = torch.zeros((3, 4, 8, 12), device=DEV)
    with pytest.raises(ValueError, match="overlaps"):                    # a state that is part of the result's
        lm_ops.linear_attention_step(q[:2], k[:2], v[:2], ld, twice[:2], out_state=twice[1:])
    with pytest.raises(ValueError, match="overlaps"):
        part = h0.view(-1)[:2 * 4 * 8].view(2, 4, 8)
        lm_ops.linear_attention_step(part, k[:2], v[:2], ld, h0, out_state=h0)


def test_a_scale_that_is_changed_in_place():
    """The scale is taken as the number that it is when it is given."""
    q, k, v, ld, off, h0, _, _ = inputs([9, 3], 2, 2, 8, 8, torch.float32)
    scale, offsets = torch.tensor(1.0), torch.tensor(off, device=DEV)
    one, _ = lm_ops.linear_attention(q, k, v, ld, offsets, h0=h0, scale=scale)
    scale.fill_(2.0)                               # (twice each result, exactly)
    two, _ = lm_ops.linear_attention(q, k, v, ld, offsets, h0=h0, scale=scale)
    assert torch.equal(two, one * 2)
    with pytest.raises(ValueError):
        lm_ops.linear_attention(q, k, v, ld, offsets, scale=2.0 ** -50)
