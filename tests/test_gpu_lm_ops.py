"""The model operators against plain restatements in 64 bits.

Tolerances.  u is 2^-24, half a unit of float32.  Recurrence: a step's factors are good to a few u (exp, a
reciprocal, products), a convex combination does not enlarge an error, so after L steps a state of values up
to M is off by at most (L + 16) 2u M, and twice that where pieces of a row are joined by products of
factors; gradients the same with the largest |dh| in M's place (and M times it for the gates').  16-bit
outputs add half of their own unit.  Products: a sum over a group rounds once a column, at most at
144 scale sum|x|, errors of either sign: 4 sqrt(group) u 144 scale sum|x|.  Logits: a handful of
operations, 4 u of the largest value in each."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import lm_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a unit of the last place: eps / 2
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def host(t):
    return None if t is None else t.detach().cpu().double().numpy()


def close(got, want, tol, dtype, what):
    got = host(got)
    assert got.shape == want.shape, what
    off = np.abs(got - want) - (tol + HALF[dtype] * np.abs(want) * (1 + 2 * HALF[dtype]) + TINY[dtype])
    worst = float(np.max(off, initial=-1.0))
    assert worst <= 0 and np.isfinite(got).all(), f"{what}: {worst} beyond the tolerance"


def rows_of(lengths):
    off = np.zeros(len(lengths) + 1, dtype=np.int64)
    np.cumsum(lengths, out=off[1:])
    return off


def scan_inputs(lengths, dim, dtype, seed=0, spread=4.0, shift=1.0):
    """Values and gates as the two halves of one tensor, states, outgoing gradients."""
    g = torch.Generator().manual_seed(seed)
    off = rows_of(lengths)
    total = int(off[-1])
    both = torch.randn((total, 2 * dim), generator=g)
    both[:, dim:] = both[:, dim:] * spread + shift
    both = both.to(dtype).to(DEV)
    h0 = torch.randn((len(lengths), dim), generator=g).to(DEV)
    dy = torch.randn((total, dim), generator=g).to(dtype).to(DEV)
    dlast = torch.randn((len(lengths), dim), generator=g).to(DEV)
    return both[:, :dim], both[:, dim:], torch.from_numpy(off).to(DEV), off, h0, dy, dlast


def check_scan(lengths, dim, dtype, reverse=False, start=True, train=True, seed=0):
    x, gate, off_d, off, h0, dy, dlast = scan_inputs(lengths, dim, dtype, seed)
    print(f"gated_scan rows={len(lengths)} total={off[-1]} dim={dim} {dtype} reverse={reverse} start={start} "
          f"train={train}", flush=True)
    h0 = h0 if start else None
    if train:
        for t in (x, gate, h0):
            if t is not None:
                t.requires_grad_(True)
    y, last = lm_ops.gated_scan(x, gate, off_d, h0=h0, reverse=reverse)
    hx, hg, hh = host(x), host(gate), host(h0)
    wy, wlast = ref.scan(hx, hg, off, hh, reverse)
    longest = max(lengths, default=0)
    most = max(np.abs(hx).max(initial=0.0), 0.0 if hh is None else np.abs(hh).max(initial=0.0))
    tol = (longest + 16) * 4 * U * most
    close(y, wy, tol, dtype, "y")
    close(last, wlast, tol, torch.float32, "last")
    if not train:
        return
    wrt = [x, gate] + ([h0] if start else [])
    got = torch.autograd.grad((y, last), wrt, (dy, dlast))
    wdx, wdg, wdh0, top = ref.scan_grad(hx, hg, off, host(dy), host(dlast), hh, reverse)
    tol = (longest + 16) * 8 * U * top
    close(got[0], wdx, tol, dtype, "dx")
    close(got[1], wdg, tol * (1 + most), dtype, "dgate")
    if start:
        close(got[2], wdh0, tol, torch.float32, "dh0")


# every length about the sizes of a thread's, a wave's and a workgroup's piece of the axis
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 255, 256, 257, 511, 512, 513, 1031, 4099])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_one_row(length, reverse):
    check_scan([length], 130, torch.bfloat16, reverse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 2, 3, 31, 64, 65, 127, 128, 129, 512])
def test_scan_channels_and_types(dim, dtype):
    check_scan([70, 1, 333], dim, dtype, reverse=dim % 2 == 0)


RAGGED = {"empty_rows": [0, 0, 5, 0, 300, 0, 0, 1, 16, 0, 240, 0],
          "only_empty": [0, 0, 0],
          "single_tokens": [1] * 700,
          "ends_with_tiles": [16, 16, 32, 64, 128, 256, 512, 256],
          "many_empty": [0] * 500 + [3] + [0] * 500 + [40] + [0] * 300,
          "mixed": [100, 1, 2000, 3, 0, 517, 64, 63, 65, 1]}


@pytest.mark.parametrize("name", sorted(RAGGED))
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("start", [False, True])
def test_scan_of_ragged_rows(name, reverse, start):
    check_scan(RAGGED[name], 96, torch.float32, reverse, start)


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_many_reads(reverse):
    rng = np.random.default_rng(5)
    check_scan(list(rng.integers(0, 60, 3000)), 34, torch.bfloat16, reverse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_a_long_row(dtype, reverse):
    check_scan([60011, 7], 5, dtype, reverse, train=True)


def test_scan_keeps_what_it_should_over_a_long_row():
    """A channel that forgets a millionth a token, and one that forgets everything at once: the share of a state
    that is left must be right, not one rounded factor to the power of the length."""
    length = 200000
    gate = torch.empty((length, 3), device=DEV)
    gate[:, 0], gate[:, 1], gate[:, 2] = 13.815510, -30.0, 30.0
    x = torch.zeros((length, 3), device=DEV)
    x[:, 1] = 3.0
    h0 = torch.full((1, 3), 1e6, device=DEV)
    off = torch.tensor([0, length], device=DEV)
    y, last = lm_ops.gated_scan(x, gate, off, h0=h0)
    k = float(ref.sigmoid(-np.float64(np.float32(13.815510))))
    left = 1e6 * np.exp(length * np.log1p(-k))
    got = last.cpu().double().numpy()[0]
    # the factor's own error: a few u of k a token (k known to 8u), and a rounding of the state a token (of either sign)
    assert abs(got[0] - left) <= left * (8 * U * k * length + 6 * U * length ** 0.5 + 16 * U)
    assert abs(got[1] - 3.0) <= 3.0 * 4 * U
    assert abs(got[2] - 1e6) <= 1e6 * (1e-13 * length + 4 * U)
    assert abs(float(y[0, 1]) - 3.0) <= 3.0 * 4 * U + 1e6 * 1e-13


def test_scan_keeps_rows_apart():
    """Infinities and NaN stay in their row."""
    x, gate, off_d, off, h0, dy, dlast = scan_inputs([40, 300, 0, 90], 70, torch.bfloat16, 3)
    clean = lm_ops.gated_scan(x, gate, off_d, h0=h0)
    bad = x.clone()
    bad[45] = float("nan")
    bad[200] = float("inf")
    for reverse in (False, True):
        want = lm_ops.gated_scan(x, gate, off_d, h0=h0, reverse=reverse)
        leaf = bad.clone().requires_grad_(True)
        y, last = lm_ops.gated_scan(leaf, gate, off_d, h0=h0, reverse=reverse)
        dx, = torch.autograd.grad((y, last), leaf, (dy, dlast))
        for lo, hi, b in ((0, 40, 0), (340, 430, 3)):
            assert torch.equal(y[lo:hi], want[0][lo:hi]) and torch.equal(last[b], want[1][b])
            assert torch.isfinite(dx[lo:hi]).all()
        assert torch.isnan(y[45]).all() and torch.isnan(last[1]).all()
    assert torch.isfinite(clean[0]).all()


def test_scan_is_the_same_every_time():
    for dtype in TYPES:
        x, gate, off_d, off, h0, dy, dlast = scan_inputs([5000, 3, 900], 256, dtype, 4)
        x, gate = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
        first = None
        for _ in range(5):
            y, last = lm_ops.gated_scan(x, gate, off_d, h0=h0)
            out = (y, last) + torch.autograd.grad((y, last), (x, gate), (dy, dlast))
            if first is None:
                first = [t.detach().clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_scan_of_dense_rows_is_that_of_packed_ones():
    x, gate, off_d, off, h0, dy, dlast = scan_inputs([129] * 6, 48, torch.bfloat16, 6)
    want = lm_ops.gated_scan(x, gate, off_d, h0=h0)
    got = lm_ops.gated_scan(x.reshape(6, 129, 48), gate.reshape(6, 129, 48), h0=h0)
    assert torch.equal(got[0].reshape(-1, 48), want[0]) and torch.equal(got[1], want[1])
    leaf = x.reshape(6, 129, 48).clone().requires_grad_(True)
    y, _ = lm_ops.gated_scan(leaf, gate.reshape(6, 129, 48))
    y.float().sum().backward()                                          # (a broadcast gradient; none for the last states)
    _, wgrad = leaf, ref.scan_grad(host(x), host(gate), off, np.ones((774, 48)), np.zeros((6, 48)))[0]
    close(leaf.grad.reshape(-1, 48), wgrad, (129 + 16) * 8 * U * 130, torch.bfloat16, "dx")


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_scan_takes_rows_at_any_place(shift):
    """First channels that lie on no multiple of a wide load, odd distances between tokens."""
    total, dim = 77, 20
    g = torch.Generator().manual_seed(shift)
    for width in (64, 63):
        wide = torch.randn((total, width), generator=g).bfloat16().to(DEV)
        x, gate = wide[:, shift:shift + dim], wide[:, shift + 30:shift + 30 + dim]
        off = np.array([0, 30, 77])
        y, last = lm_ops.gated_scan(x, gate, torch.from_numpy(off).to(DEV))
        wy, wlast = ref.scan(host(x), host(gate), off)
        tol = (47 + 16) * 4 * U * np.abs(host(x)).max()
        close(y, wy, tol, torch.bfloat16, "y")
        close(last, wlast, tol, torch.float32, "last")


def test_scan_gradient_against_differences():
    """The kernel's own values, a little to either side along a random direction."""
    x, gate, off_d, off, h0, dy, dlast = scan_inputs([150, 0, 37, 1], 24, torch.float32, 8, spread=2.0)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, gate, h0)]

    def value(ts):
        y, last = lm_ops.gated_scan(ts[0], ts[1], off_d, h0=ts[2])
        return (y.double() * dy.double()).sum() + (last.double() * dlast.double()).sum()

    grads = torch.autograd.grad(value(leaves), leaves)
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        way = torch.randn(leaves[i].shape, generator=g).to(DEV)
        eps = 1e-2
        with torch.no_grad():
            up = value([t + eps * way if j == i else t for j, t in enumerate(leaves)])
            down = value([t - eps * way if j == i else t for j, t in enumerate(leaves)])
        slope = float((grads[i].double() * way.double()).sum())
        diff = float((up - down) / (2 * eps))
        # rounding of the values (16u of each, of either sign) over 2 eps, and eps^2 times a third derivative of about
        # the sum's own size
        size = float((dy.double() ** 2).sum().sqrt()) * 4
        assert abs(slope - diff) <= size * (64 * U / eps + 20 * eps * eps), i


def test_scan_is_differentiable_once_and_only_where_asked():
    x, gate, off_d, off, h0, dy, dlast = scan_inputs([20, 9], 8, torch.float32)
    gate = gate.detach().clone().requires_grad_(True)
    y, last = lm_ops.gated_scan(x, gate, off_d)
    (dg,) = torch.autograd.grad(last, gate, dlast)                      # nothing flows into y
    close(dg, ref.scan_grad(host(x), host(gate), off, 0 * host(dy), host(dlast))[1], 40 * 16 * U * 8, torch.float32, "dg")
    assert not lm_ops.gated_scan(x, gate.detach(), off_d)[0].requires_grad


def test_scan_on_another_stream_and_in_a_graph():
    x, gate, off_d, off, h0, dy, dlast = scan_inputs([3000, 0, 500], 130, torch.bfloat16, 9)
    want = lm_ops.gated_scan(x, gate, off_d, h0=h0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lm_ops.gated_scan(x, gate, off_d, h0=h0)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    bx, bg = x.clone(), gate.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, last = lm_ops.gated_scan(bx, bg, off_d, h0=h0)
    for seed in range(4):
        nx, ng, *_ = scan_inputs([3000, 0, 500], 130, torch.bfloat16, 20 + seed)
        bx.copy_(nx)
        bg.copy_(ng)
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want = lm_ops.gated_scan(nx, ng, off_d, h0=h0)                  # (eager work between the replays)
        assert torch.equal(y, want[0]) and torch.equal(last, want[1]), seed


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 512), (7, 33), (300, 128), (5, 1030)])
def test_step(shape, dtype):
    b, d = shape
    x, gate, _, off, h0, _, _ = scan_inputs([1] * b, d, dtype, 11)
    wy, wh = ref.scan(host(x), host(gate), off, host(h0))
    tol = 17 * 4 * U * max(np.abs(host(x)).max(), np.abs(host(h0)).max())
    y, h = lm_ops.gated_step(x, gate, h0)
    close(y, wy, tol, dtype, "y")
    close(h, wh, tol, torch.float32, "state")
    y2, h2 = lm_ops.gated_step(x, gate, h0, out_state=h0)               # in place
    assert h2 is h0 and torch.equal(h0, h) and torch.equal(y2, y)
    y0, _ = lm_ops.gated_step(x, gate)
    close(y0, ref.scan(host(x), host(gate), off)[0], tol, dtype, "y from nothing")


def test_steps_are_the_scan():
    x, gate, off_d, off, h0, _, _ = scan_inputs([50, 50, 50], 66, torch.bfloat16, 12)
    y, last = lm_ops.gated_scan(x, gate, off_d, h0=h0)
    h = h0.clone()
    tol = (50 + 16) * 4 * U * max(np.abs(host(x)).max(), np.abs(host(h0)).max())
    for t in range(50):
        yt, _ = lm_ops.gated_step(x[t::50], gate[t::50], h, out_state=h)
        close(yt, host(y[t::50]), tol + 2 * HALF[torch.bfloat16] * 4, torch.bfloat16, t)
    close(h, host(last), tol, torch.float32, "state")


# ---- products with 4-bit weights ----------------------------------------------------------------

def w4_inputs(m, n, k, group, dtype, zeros, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    words, groups = -(-k // 8), -(-k // group)
    q = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g).to(torch.int32).to(DEV)
    scales = (0.002 + 0.004 * torch.rand((n, groups), generator=g)).to(dtype).to(DEV)
    z = torch.randint(0, 16, (n, groups), generator=g).to(torch.uint8).to(DEV) if zeros else None
    x = (torch.randn((m, k), generator=g) + shift).to(dtype).to(DEV)
    return q, scales, z, x, torch.randn(n, generator=g).to(DEV)


def check_w4(m, n, k, group, dtype, zeros, out_dtype=None, bias=True, seed=0, shift=0.0):
    print(f"w4 m={m} n={n} k={k} group={group} {dtype} zeros={zeros} out={out_dtype}", flush=True)
    q, scales, z, x, b = w4_inputs(m, n, k, group, dtype, zeros, seed, shift)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=k, group=group)
    y = matrix.matvec(x, bias=b if bias else None, out_dtype=out_dtype)
    hx, hs = host(x), host(scales)
    want = ref.w4(hx, q.cpu().numpy(), hs, None if z is None else z.cpu().numpy(), k, group, host(b) if bias else None)
    tol = 4 * min(group, k) ** 0.5 * U * 144 * hs.max() * np.abs(hx).sum(1, keepdims=True) + 8 * U * np.abs(want)
    close(y, want, tol, y.dtype, "y")
    return matrix, x, y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 512])
@pytest.mark.parametrize("m", [1, 3, 17])
def test_w4_groups_and_types(m, group, zeros, dtype):
    check_w4(m, 80, 1024, group, dtype, zeros)


@pytest.mark.parametrize("k", [1, 2, 7, 8, 9, 31, 32, 33, 64, 100, 127, 128, 129, 255, 257, 500, 1000, 2041, 4096, 5001])
@pytest.mark.parametrize("m", [1, 5])
def test_w4_depths(k, m):
    check_w4(m, 37, k, 64, torch.bfloat16, True, torch.float32)
    check_w4(m, 37, k, 128, torch.float16, False)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 65, 127, 1000, 4097])
@pytest.mark.parametrize("m", [1, 2, 4, 8, 15, 16, 32, 33, 61, 64, 130])
def test_w4_rows(m, n):
    check_w4(m, n, 416, 32, torch.bfloat16, m % 2 == 0, torch.float32 if n % 2 else None)


def test_w4_with_values_of_one_sign():
    """Sums that grow: values about 3."""
    for dtype in (torch.bfloat16, torch.float16):
        check_w4(2, 50, 2048, 128, dtype, True, torch.float32, shift=3.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_w4_takes_strided_rows_and_vectors(dtype):
    q, scales, z, x, b = w4_inputs(6, 70, 320, 64, dtype, True)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=320, group=64)
    want = matrix.matvec(x, bias=b)
    wide = torch.full((6, 901), float("nan"), dtype=dtype, device=DEV)
    wide[:, 3:323] = x
    out = torch.full((6, 99), 7.0, dtype=dtype, device=DEV)
    got = matrix.matvec(wide[:, 3:323], bias=b, out=out[:, 5:75])
    assert torch.equal(got, want) and (out[:, :5] == 7).all() and (out[:, 75:] == 7).all()
    spaced = torch.full((70, 57), -1, dtype=torch.int32, device=DEV)
    spaced[:, :40] = q
    assert torch.equal(lm_ops.W4Matrix(spaced[:, :40], scales, z, in_features=320, group=64).matvec(x, bias=b), want)
    vec = matrix.matvec(x[2], bias=b)
    assert vec.shape == (70,)
    close(vec, host(want[2]), np.abs(host(want[2])) * 2 * HALF[dtype] + 1e-3, dtype, "a vector")


def test_w4_rows_do_not_touch_each_other():
    """A row of x with infinities or NaN leaves the others alone."""
    for dtype in (torch.bfloat16, torch.float16):
        matrix, x, want = check_w4(19, 40, 256, 64, dtype, True)
        bad = x.clone()
        bad[4, 17], bad[9, 0] = float("inf"), float("nan")
        got = matrix.matvec(bad, bias=w4_inputs(19, 40, 256, 64, dtype, True)[4])
        keep = [i for i in range(19) if i not in (4, 9)]
        assert torch.equal(got[keep], want[keep])
        assert not torch.isfinite(got[[4, 9]]).any()


def test_w4_unused_values_behind_the_last_column():
    """What lies in the last word behind the k-th value does not count, whatever it is."""
    q, scales, z, x, b = w4_inputs(3, 20, 61, 64, torch.bfloat16, False)
    a = lm_ops.W4Matrix(q, scales, z, in_features=61, group=64).matvec(x)
    q2 = q.clone()
    q2[:, -1] ^= -(1 << 20)                                             # (bits 20 .. 31: values 61, 62 and 63)
    assert torch.equal(lm_ops.W4Matrix(q2, scales, z, in_features=61, group=64).matvec(x), a)


def test_w4_quantize_and_back():
    g = torch.Generator().manual_seed(2)
    w = torch.randn((50, 200), generator=g).to(DEV)
    w[3] = 0.0
    for symmetric in (True, False):
        matrix = lm_ops.W4Matrix.quantize(w, 64, symmetric=symmetric)
        back = matrix.dequantize()
        step = matrix.scales.float().repeat_interleave(64, 1)[:, :200]
        # half a step, and where the step is itself rounded to 8 bits (2^-9), as much of the largest whole number
        assert ((back - w).abs() <= step * (0.5 + 16 * 2.0 ** -8)).all()
        x = torch.randn((2, 200), generator=g).bfloat16().to(DEV)
        want = host(x) @ host(back).T
        close(matrix.matvec(x, out_dtype=torch.float32), want,
              4 * 8 * U * 144 * float(step.max()) * np.abs(host(x)).sum(1, keepdims=True), torch.float32, "y")


# ---- logits -------------------------------------------------------------------------------------

def logits_inputs(rows, vocab, lengths, dtype, seed=0, states=7):
    g = torch.Generator().manual_seed(seed)
    off = rows_of(lengths)
    total = int(off[-1])
    r = {"logits": (torch.randn((rows, vocab), generator=g) * 4).to(dtype),
         "history": (torch.rand(total, generator=g) ** 2 * vocab).to(torch.int32).clamp(max=vocab - 1),
         "history_offsets": torch.from_numpy(off), "prompt_lengths": torch.from_numpy(np.asarray(lengths) // 3).to(torch.int32),
         "repetition": 0.8 + torch.rand(rows, generator=g), "presence": torch.rand(rows, generator=g),
         "frequency": torch.randn(rows, generator=g) * 0.3, "bias": torch.randn(vocab, generator=g),
         "allowed": torch.randint(-2 ** 31, 2 ** 31, (states, -(-vocab // 32)), generator=g).to(torch.int32),
         "state": torch.randint(-1, states, (rows,), generator=g, dtype=torch.int32)}
    return {k: v.to(DEV) for k, v in r.items()}


def check_logits(a, **kw):
    z = a["logits"]
    rest = {k: v for k, v in a.items() if k != "logits"}
    print("logits", tuple(z.shape), z.dtype, sorted(rest), kw, flush=True)
    got = lm_ops.process_logits(z, **rest, **kw)
    names = {"history_offsets": "offsets", "prompt_lengths": "prompt"}
    want = ref.logits(host(z), **{names.get(k, k): v.cpu().numpy() if v.dtype in (torch.int32, torch.int64) else host(v)
                                  for k, v in rest.items()})
    masked = np.isneginf(want)
    assert np.array_equal(np.isneginf(host(got)), masked)
    out = torch.where(torch.from_numpy(masked).to(DEV), torch.zeros_like(got), got)
    want = np.where(masked, 0.0, want)
    size = np.abs(want).max(initial=0.0) + 2 * np.abs(np.nan_to_num(host(z), neginf=0.0)).max(initial=0.0)
    if "frequency" in rest:
        size += float(rest["frequency"].abs().max()) * float(np.diff(rest["history_offsets"].cpu().numpy()).max())
    close(out, want, 4 * U * size, got.dtype, "logits")
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 5, 31, 32, 33, 1000, 4096, 8191, 8192, 8193, 32000, 70001])
def test_logits_vocabularies(vocab, dtype):
    check_logits(logits_inputs(3, vocab, [0, 50, 700], dtype))
    check_logits(logits_inputs(3, vocab, [0, 50, 700], dtype), out_dtype=torch.float32)


@pytest.mark.parametrize("rows", [1, 2, 9, 200])
def test_logits_rows(rows):
    rng = np.random.default_rng(rows)
    check_logits(logits_inputs(rows, 4096, list(rng.integers(0, 900, rows)), torch.float32, rows))


@pytest.mark.parametrize("length", [1, 3, 4, 1023, 1024, 1025, 4096, 100001])
def test_logits_history_lengths(length):
    check_logits(logits_inputs(2, 3000, [length, 1], torch.float32, 1))


def test_logits_one_token_over_and_over():
    """A count that passes 16 bits, on one address."""
    a = logits_inputs(1, 100, [200000], torch.float32)
    a["history"].fill_(17)
    a["prompt_lengths"].fill_(3)
    check_logits(a)


@pytest.mark.parametrize("keys", [("bias",), ("allowed", "state"), ("history", "history_offsets", "repetition"),
                                  ("history", "history_offsets", "presence", "prompt_lengths"),
                                  ("history", "history_offsets", "frequency"), ()])
def test_logits_each_on_its_own(keys):
    a = logits_inputs(4, 1500, [10, 0, 90, 400], torch.bfloat16)
    check_logits({k: a[k] for k in ("logits",) + keys})


def test_logits_numbers_for_all_rows_and_biases_of_each_row():
    a = logits_inputs(4, 1500, [10, 0, 90, 400], torch.float32)
    want = lm_ops.process_logits(**{**a, "repetition": torch.full((4,), 1.5, device=DEV)})
    assert torch.equal(lm_ops.process_logits(**{**a, "repetition": 1.5}), want)
    wide = torch.randn((4, 1503), device=DEV)
    check_logits({**a, "bias": wide[:, 2:1502]})


def test_logits_ids_outside_the_vocabulary_and_prompts_longer_than_the_history():
    a = logits_inputs(3, 777, [300, 300, 300], torch.float32)
    a["history"][::7] = -1
    a["history"][1::7] = 777
    a["history"][2::7] = 2 ** 31 - 1
    a["history"][3::7] = -2 ** 31
    a["prompt_lengths"][:] = torch.tensor([0, 300, 5000], dtype=torch.int32)
    check_logits(a)


def test_logits_masks():
    a = logits_inputs(5, 100, [9, 9, 9, 9, 9], torch.float32)
    a["allowed"][0] = 0                                                 # nothing may follow
    a["allowed"][1] = -1
    a["state"][:] = torch.tensor([0, 1, -1, 7, 2 ** 31 - 1], dtype=torch.int32)     # (7 and more: no such mask)
    a["logits"][:, 3] = float("-inf")
    a["logits"][0, 5], a["logits"][3, 6] = float("nan"), float("inf")   # forbidden there
    got = lm_ops.process_logits(**a)
    assert torch.isneginf(got[0]).all() and torch.isneginf(got[3]).all() and torch.isneginf(got[4]).all()
    assert torch.isneginf(got[:, 3]).all() and torch.isfinite(got[1, :3]).all() and torch.isfinite(got[2, 4:]).all()
    free = {k: v for k, v in a.items() if k != "state"}
    free["logits"] = torch.randn_like(a["logits"])
    check_logits({**free, "allowed": a["allowed"][2:3]})                # one mask for all rows
    check_logits({**free, "allowed": a["allowed"][1:6]})                # one of each row
    low = torch.finfo(torch.float32).min                                # the type's lowest value is a number like any other
    free["logits"][1:, ::2] = low
    check_logits({k: free[k] for k in ("logits", "allowed")} | {"state": a["state"].clamp(max=1)})


def test_logits_in_place_and_strided():
    a = logits_inputs(4, 1003, [40, 3, 0, 800], torch.bfloat16)
    want = lm_ops.process_logits(**a)
    z = a["logits"].clone()
    got = lm_ops.process_logits(**{**a, "logits": z}, out=z)
    assert got is z and torch.equal(z, want)
    wide = torch.full((4, 1100), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 11:1014] = a["logits"]
    masks = torch.zeros((7, 50), dtype=torch.int32, device=DEV)
    masks[:, 3:35] = a["allowed"]
    got = lm_ops.process_logits(**{**a, "logits": wide[:, 11:1014], "allowed": masks[:, 3:35]}, out=wide[:, 11:1014])
    assert torch.equal(got, want) and (wide[:, :11] == 7).all() and (wide[:, 1014:] == 7).all()


def test_logits_in_a_graph():
    a = logits_inputs(2, 5000, [3000, 40], torch.float32)
    lm_ops.process_logits(**a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lm_ops.process_logits(**a)
    for seed in range(4):
        b = logits_inputs(2, 5000, [3000, 40], torch.float32, 30 + seed)
        for k in a:
            a[k].copy_(b[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lm_ops.process_logits(**b)), seed


# ---- refusals -----------------------------------------------------------------------------------

def test_refusals():
    x = torch.randn((10, 8), device=DEV)
    off = torch.tensor([0, 4, 10], device=DEV)
    ok = lm_ops.gated_scan(x, x, off)
    assert ok[0].shape == (10, 8) and ok[1].shape == (2, 8)
    for bad in (lambda: lm_ops.gated_scan(x.cpu(), x, off), lambda: lm_ops.gated_scan(x, x.half(), off),
                lambda: lm_ops.gated_scan(x, x[:9], off), lambda: lm_ops.gated_scan(x, x, off.int()),
                lambda: lm_ops.gated_scan(x, x), lambda: lm_ops.gated_scan(x.double(), x.double(), off),
                lambda: lm_ops.gated_scan(x.t(), x.t(), off), lambda: lm_ops.gated_scan(x, x, off[:1]),
                lambda: lm_ops.gated_scan(x, x, off, h0=torch.zeros((3, 8), device=DEV)),
                lambda: lm_ops.gated_scan(x, x, off, h0=torch.zeros((2, 8), device=DEV).half()),
                lambda: lm_ops.gated_scan(x[:, :0], x[:, :0], off),
                lambda: lm_ops.gated_step(x, x, x[:9]), lambda: lm_ops.gated_step(x[0], x[0]),
                lambda: lm_ops.gated_step(x, x, out_state=x.half()),
                lambda: lm_ops.gated_step(x.clone().requires_grad_(True), x)):
        with pytest.raises(ValueError):
            bad()
    q, scales, z, xh, b = w4_inputs(2, 16, 64, 32, torch.bfloat16, True)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=64, group=32)
    for bad in (lambda: lm_ops.W4Matrix(q, scales.float(), z, in_features=64, group=32),
                lambda: lm_ops.W4Matrix(q, scales, z, in_features=64, group=48),
                lambda: lm_ops.W4Matrix(q, scales, z, in_features=72, group=32),
                lambda: lm_ops.W4Matrix(q, scales, z.int(), in_features=64, group=32),
                lambda: lm_ops.W4Matrix(q.long(), scales, z, in_features=64, group=32),
                lambda: matrix.matvec(xh.half()), lambda: matrix.matvec(xh[:, :63]), lambda: matrix.matvec(xh.cpu()),
                lambda: matrix.matvec(xh, bias=b.half()), lambda: matrix.matvec(xh, out_dtype=torch.float16),
                lambda: matrix.matvec(xh, out=torch.empty((2, 15), device=DEV)),
                lambda: matrix.matvec(xh.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            bad()
    a = logits_inputs(2, 40, [3, 3], torch.float32)
    for change in ({"history_offsets": None}, {"history": None, "history_offsets": None},
                   {"history": a["history"].long()}, {"prompt_lengths": a["prompt_lengths"][:1]},
                   {"repetition": a["repetition"].double()}, {"bias": a["bias"][:39]}, {"bias": a["bias"].half()},
                   {"allowed": None}, {"allowed": a["allowed"][:, :1]}, {"allowed": a["allowed"][:0]},
                   {"state": a["state"].long()}, {"state": None}, {"logits": a["logits"][0]},
                   {"logits": a["logits"].double()}, {"out": torch.empty((2, 41), device=DEV)},
                   {"out_dtype": torch.float16}, {"logits": a["logits"].t().contiguous().t()}):
        with pytest.raises(ValueError):
            lm_ops.process_logits(**{**a, **change})


def test_nothing_to_do():
    x = torch.empty((0, 8), device=DEV)
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    y, last = lm_ops.gated_scan(x, x, off)
    assert y.shape == (0, 8) and last.shape == (0, 8)
    assert lm_ops.gated_step(x, x)[0].shape == (0, 8)
    q, scales, z, xh, b = w4_inputs(0, 16, 64, 32, torch.bfloat16, True)
    assert lm_ops.W4Matrix(q, scales, z, in_features=64, group=32).matvec(xh).shape == (0, 16)
    assert lm_ops.process_logits(torch.empty((0, 9), device=DEV)).shape == (0, 9)


# ---- all of them together -----------------------------------------------------------------------

def test_example_trains_and_generates_what_the_motif_allows(capsys):
    import importlib.util
    import os
    import re
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "generate_dna.py")
    spec = importlib.util.spec_from_file_location("generate_dna", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    print("example: 12 training steps, a motif", flush=True)
    losses, sequences = example.main(["--motif", "ATGNNNRYNNTAA", "--rows", "3", "--train", "12"])
    assert len(losses) == 12 and losses[-1] < losses[0]
    assert len(sequences) == 3
    for s in sequences:
        assert re.fullmatch("ATG[ACGT]{3}[AG][CT][ACGT]{2}TAA", s), s
