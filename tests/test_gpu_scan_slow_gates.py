"""The recurrence where channels keep what they hold over many tiles and groups of tiles: mean gates of 6 to 10, rows of more
than seventeen groups (of 16 x 168 tokens forwards, 16 x 264 backwards), every result against 64 bits."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import lm_bounds
from tests.test_gpu_lm_ops import DEV, HALF, TINY, TYPES, host, rows_of

pytestmark = pytest.mark.gpu


def slow_inputs(lengths, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    off = rows_of(lengths)
    total = int(off[-1])
    both = torch.randn((total, 2 * dim), generator=g)
    both[:, dim:] += torch.linspace(6.0, 10.0, dim)
    both = both.to(dtype).to(DEV)
    h0, dlast = (torch.randn((len(lengths), dim), generator=g).to(DEV) for _ in range(2))
    dy = torch.randn((total, dim), generator=g).to(dtype).to(DEV)
    return both[:, :dim].requires_grad_(True), both[:, dim:].requires_grad_(True), off, h0.requires_grad_(True), dy, dlast


def within(got, want, bound, dtype, what):
    off = np.abs(host(got) - want) - (bound + HALF[dtype] * (1 + 2 * HALF[dtype]) * (np.abs(want) + bound) + TINY[dtype])
    worst = float(np.max(off, initial=-1.0))
    assert worst <= 0 and torch.isfinite(got).all(), f"{what}: {worst} beyond the bound"


@pytest.mark.parametrize("dim", [5, 70])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_carries_over_groups(dtype, dim, reverse):
    lengths = [9000, 80000, 300]                                       # (a row that starts inside a group among them)
    print(f"gated_scan slow gates dim={dim} {dtype} reverse={reverse}", flush=True)
    x, gate, off, h0, dy, dlast = slow_inputs(lengths, dim, dtype, dim)
    y, last = lm_ops.gated_scan(x, gate, torch.from_numpy(off).to(DEV), h0=h0, reverse=reverse)
    dx, dg, dh0 = torch.autograd.grad((y, last), (x, gate, h0), (dy, dlast))
    want, bound = lm_bounds.scan(host(x), host(gate), off, host(dy), host(dlast), host(h0), reverse)
    # what is carried over groups is far more than the bound: the test sees it
    assert np.median(bound["y"]) < 0.1 * np.median(np.abs(want["y"]))
    within(y, want["y"], bound["y"], dtype, "y")
    within(last, want["last"], bound["last"], torch.float32, "last")
    within(dx, want["dx"], bound["dx"], dtype, "dx")
    within(dg, want["dgate"], bound["dgate"], dtype, "dgate")
    within(dh0, want["dh0"], bound["dh0"], torch.float32, "dh0")


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_of_a_row_past_two_billion_elements(reverse):
    """All of a row whose elements pass 2^31, against the same call on the row's two ends: the last piece continued from
    the first one's state.  A channel's state is a sum of what it met on the way, so a wrong offset or a lost carry would show in
    every token behind it; the slowest channels keep 1e-4 of it over 100,000 tokens."""
    dim, dtype = 512, torch.bfloat16
    length = 2 ** 31 // dim + 5000
    print(f"gated_scan one row of {length} dim={dim} reverse={reverse}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(15)
    x, gate, dy = (torch.randn((length, dim), generator=g, device=DEV, dtype=dtype) for _ in range(3))
    gate += torch.linspace(2.0, 9.3, dim, device=DEV).to(dtype)
    h0, dlast = (torch.randn((1, dim), generator=g, device=DEV) for _ in range(2))
    for t in (x, gate, h0):
        t.requires_grad_(True)
    y, last = lm_ops.gated_scan(x, gate, torch.tensor([0, length], device=DEV), h0=h0, reverse=reverse)
    grads = torch.autograd.grad((y, last), (x, gate, h0), (dy, dlast))
    # in four pieces, states and gradients handed on by the caller
    cuts = [0, length // 4 + 1, length // 2 + 3, length - 700, length]
    pieces = [slice(a, b) for a, b in zip(cuts, cuts[1:])]
    if reverse:
        pieces.reverse()
    state, kept = h0.detach(), []
    for p in pieces:
        own = torch.tensor([0, p.stop - p.start], device=DEV)
        leaves = [t.detach()[p].requires_grad_(True) for t in (x, gate)] + [state.clone().requires_grad_(True)]
        yp, lp = lm_ops.gated_scan(*leaves[:2], own, h0=leaves[2], reverse=reverse)
        kept.append((leaves, yp, lp))
        state = lp.detach()

    def near(a, b, scale):
        # both are within 32-bit rounding errors of each other: e_t of the bound is at most 16 u H / k + 8 (|g| + 8) u 3 max|x|
        # with k >= e^-14 of the slowest token; typical tokens' k is 100 times as large.  16-bit results may round apart by a unit.
        limit = 2.0 ** -7 * b.float().abs() + 2e-3 * scale
        return bool(((a.float() - b.float()).abs() <= limit).all())

    assert torch.equal(state.isfinite(), torch.ones_like(state, dtype=torch.bool))
    assert near(last, state, 1.0)
    flow = dlast
    for p, (leaves, yp, lp) in zip(reversed(pieces), reversed(kept)):
        assert near(y[p], yp, 1.0), f"y of {p}"
        dxp, dgp, flow = torch.autograd.grad((yp, lp), leaves, (dy[p], flow))
        assert near(grads[0][p], dxp, 1.0) and near(grads[1][p], dgp, 1.0), f"gradients of {p}"
    assert near(grads[2], flow, 1.0 + float(flow.abs().max()))
