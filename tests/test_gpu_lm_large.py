"""The model operators where offsets pass 2^31 elements, and gradients of inputs that are one row broadcast.
Tolerances are those of the small cases."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import lm_reference as ref
from tests.test_gpu_lm_ops import DEV, U, close, host, rows_of, w4_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_past_two_billion_elements(reverse):
    dim, dtype = 512, torch.bfloat16
    lengths = [300, 2 ** 31 // dim + 5000, 700]
    off = rows_of(lengths)
    total = int(off[-1])
    print(f"gated_scan total={total} dim={dim} reverse={reverse}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    x, gate, dy = (torch.randn((total, dim), generator=g, device=DEV, dtype=dtype) for _ in range(3))
    h0, dlast = (torch.randn((3, dim), generator=g, device=DEV) for _ in range(2))
    x.requires_grad_(True), gate.requires_grad_(True), h0.requires_grad_(True)
    y, last = lm_ops.gated_scan(x, gate, torch.from_numpy(off).to(DEV), h0=h0, reverse=reverse)
    dx, dg, dh0 = torch.autograd.grad((y, last), (x, gate, h0), (dy, dlast))
    for r in (0, 2):
        part, n = slice(int(off[r]), int(off[r + 1])), lengths[r]
        hx, hg, hd, own = host(x[part]), host(gate[part]), host(dy[part]), rows_of([n])
        hh, hl = host(h0[r:r + 1]), host(dlast[r:r + 1])
        wy, wlast = ref.scan(hx, hg, own, hh, reverse)
        most = max(np.abs(hx).max(), np.abs(hh).max())
        tol = (n + 16) * 4 * U * most
        close(y[part], wy, tol, dtype, f"y of row {r}")
        close(last[r:r + 1], wlast, tol, torch.float32, f"last of row {r}")
        wdx, wdg, wdh0, top = ref.scan_grad(hx, hg, own, hd, hl, hh, reverse)
        tol = (n + 16) * 8 * U * top
        close(dx[part], wdx, tol, dtype, f"dx of row {r}")
        close(dg[part], wdg, tol * (1 + most), dtype, f"dgate of row {r}")
        close(dh0[r:r + 1], wdh0, tol, torch.float32, f"dh0 of row {r}")


@pytest.mark.parametrize("m,n,stride", [(1, 300, 2 ** 22 - 1), (17, 300, 2 ** 22 - 4), (40, 10300, 2 ** 16)])
def test_w4_with_rows_of_weights_far_apart(m, n, stride):
    k, group = 1000, 64
    print(f"w4 m={m} n={n} k={k} stride={stride}", flush=True)
    q, scales, z, x, b = w4_inputs(m, n, k, group, torch.bfloat16, True)
    wide = torch.zeros(n * stride, dtype=torch.int32, device=DEV)
    far = wide.as_strided(q.shape, (stride, 1))
    far.copy_(q)
    got = lm_ops.W4Matrix(far, scales, z, in_features=k, group=group).matvec(x, bias=b)
    assert torch.equal(got, lm_ops.W4Matrix(q, scales, z, in_features=k, group=group).matvec(x, bias=b))


def test_logits_past_two_billion_elements():
    rows, vocab = 54000, 40000
    print(f"logits {rows} x {vocab}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(6)
    z = torch.randn((rows, vocab), generator=g, device=DEV, dtype=torch.bfloat16)
    history = torch.randint(0, vocab, (rows * 10,), generator=g, device=DEV, dtype=torch.int32)
    offsets = torch.arange(rows + 1, device=DEV) * 10
    allowed = torch.randint(-2 ** 31, 2 ** 31, (5, -(-vocab // 32)), generator=g, device=DEV).to(torch.int32)
    state = (torch.arange(rows, device=DEV) % 5).to(torch.int32)
    rest = dict(repetition=1.5, presence=0.5, frequency=0.25)
    got = lm_ops.process_logits(z, history=history, history_offsets=offsets, allowed=allowed, state=state, **rest)
    for part in (slice(0, 2), slice(rows - 2, rows)):
        own = offsets[part.start:part.stop + 1].clone()
        want = lm_ops.process_logits(z[part], history=history, history_offsets=own, allowed=allowed, state=state[part], **rest)
        assert torch.equal(got[part], want)


def test_logits_with_a_history_past_two_billion_ids():
    first, lengths, vocab = 2 ** 31 + 3, [700, 197], 1000
    print(f"logits history at {first}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(7)
    history = torch.zeros(first + sum(lengths), dtype=torch.int32, device=DEV)
    tail = torch.randint(0, vocab, (sum(lengths),), generator=g, device=DEV, dtype=torch.int32)
    history[first:] = tail
    offsets = torch.from_numpy(rows_of(lengths)).to(DEV)
    z = torch.randn((2, vocab), generator=g, device=DEV)
    rest = dict(repetition=1.5, presence=0.5, frequency=0.25)
    got = lm_ops.process_logits(z, history=history, history_offsets=offsets + first, **rest)
    assert torch.equal(got, lm_ops.process_logits(z, history=tail, history_offsets=offsets, **rest))


@pytest.mark.parametrize("which", ["x", "gate"])
def test_scan_of_one_broadcast_row_and_its_gradient(which):
    n, dim = 200, 70
    off = rows_of([n])
    g = torch.Generator().manual_seed(8)
    one = torch.randn((1, dim), generator=g).to(DEV).requires_grad_(True)
    other = torch.randn((n, dim), generator=g).to(DEV)
    dy = torch.randn((n, dim), generator=g).to(DEV)
    wide = one.expand(n, dim)
    x, gate = (wide, other) if which == "x" else (other, wide)
    y, _ = lm_ops.gated_scan(x, gate, torch.from_numpy(off).to(DEV))
    (got,) = torch.autograd.grad(y, one, dy)
    hx, hg = np.ascontiguousarray(host(x)), np.ascontiguousarray(host(gate))
    wdx, wdg, _, top = ref.scan_grad(hx, hg, off, host(dy), np.zeros((1, dim)))
    most = np.abs(hx).max()
    each = (n + 16) * 8 * U * top * (1.0 if which == "x" else 1 + most)
    want = (wdx if which == "x" else wdg).sum(0, keepdims=True)
    # the sum of n gradients: n times the error of one, and n roundings of sums of magnitudes
    rounded = n * U * np.abs(wdx if which == "x" else wdg).sum(0).max()
    close(got, want, n * each + rounded, torch.float32, which)
