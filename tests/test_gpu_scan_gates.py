"""The recurrence where gates are closed: f = sigmoid(gate) next to nothing.  What is left of a state, and every gradient, is
right to a few units of the result itself, however small.  Bounds from tests/support/lm_bounds.py."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import lm_bounds
from tests.test_gpu_lm_ops import DEV, host, rows_of

pytestmark = pytest.mark.gpu
GATES = [-4.0, -8.0, -10.0, -12.0, -14.0, -16.0, -17.5, -20.0, -25.0, -40.0, -80.0]


def test_step_with_closed_gates_and_large_states():
    g = torch.Generator().manual_seed(1)
    gate = torch.tensor(GATES + [-v for v in GATES] + [0.0, 0.3]).repeat(50, 1)
    x = torch.rand(gate.shape, generator=g) * 0.9 + 0.1
    for size in (1.0, 1e6, 1e-6):
        state = torch.randn(gate.shape, generator=g) * size
        y, h = lm_ops.gated_step(x.to(DEV), gate.to(DEV), state.to(DEV))
        want, bound = lm_bounds.step(host(x), host(gate), host(state))
        assert (np.abs(host(h) - want) <= bound).all(), size
        assert torch.equal(y, h)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lengths", [[1] * 60, [2, 1, 3, 2] * 40, [5] * 61])
def test_scan_with_closed_gates_and_large_states(lengths, reverse):
    """Short rows, so that a result holds few errors: each a few units of what the token adds."""
    g = torch.Generator().manual_seed(2)
    off = rows_of(lengths)
    total, rows, dim = int(off[-1]), len(lengths), len(GATES)
    gate = torch.tensor(GATES).repeat(total, 1) + torch.rand((total, dim), generator=g)
    x = torch.rand((total, dim), generator=g) * 0.9 + 0.1
    h0 = torch.randn((rows, dim), generator=g) * 1e6
    y, last = lm_ops.gated_scan(x.to(DEV), gate.to(DEV), torch.from_numpy(off).to(DEV), h0=h0.to(DEV), reverse=reverse)
    hx, hg, hh = host(x), host(gate), host(h0)
    for b in range(rows):
        h, tol = hh[b], np.zeros(dim)
        tokens = range(off[b], off[b + 1])
        for t in reversed(tokens) if reverse else tokens:
            f = 1.0 / (1.0 + np.exp(-hg[t]))
            h, own = lm_bounds.step(hx[t], hg[t], h)
            # twice for the piece of a row in front of a join and once for what comes in; the piece's factor
            tol = f * tol + 4 * own + 40 * lm_bounds.U * f * np.abs(h)
            assert (np.abs(host(y[t]) - h) <= tol).all(), (b, t)
        assert (np.abs(host(last[b]) - h) <= tol).all(), b


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lengths", [[1] * 60, [30, 1, 3, 200, 2], [700]])
def test_gradients_with_closed_gates(lengths, reverse):
    g = torch.Generator().manual_seed(3)
    off = rows_of(lengths)
    total, rows, dim = int(off[-1]), len(lengths), len(GATES)
    gate = (torch.tensor(GATES).repeat(total, 1) + torch.rand((total, dim), generator=g)).to(DEV).requires_grad_(True)
    x, dy = (torch.randn((total, dim), generator=g).to(DEV) for _ in range(2))
    h0, dlast = (torch.randn((rows, dim), generator=g).to(DEV) for _ in range(2))
    x.requires_grad_(True), h0.requires_grad_(True)
    y, last = lm_ops.gated_scan(x, gate, torch.from_numpy(off).to(DEV), h0=h0, reverse=reverse)
    got = torch.autograd.grad((y, last), (x, gate, h0), (dy, dlast))
    want, bound = lm_bounds.scan(host(x), host(gate), off, host(dy), host(dlast), host(h0), reverse)
    for t, name in zip((y, last) + got, ("y", "last", "dx", "dgate", "dh0")):
        assert (np.abs(host(t) - want[name]) <= bound[name]).all(), name
    # dgate to a part in a hundred thousand wherever the formula's does not cancel (1e-30: below is next to what 32 bits hold)
    big = (np.abs(want["dgate"]) > 1e-30) & (bound["dgate"] < 1e-4 * np.abs(want["dgate"]))
    assert big.mean() > 0.5
    ratio = host(got[1])[big] / want["dgate"][big]
    assert np.abs(ratio - 1.0).max() < 1e-4
