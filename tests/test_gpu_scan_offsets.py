"""Buffers that are longer than the rows in them, as a packer leaves them: tokens in no row give zeros and take no gradient,
whatever they hold, and rows are as they are without them."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import DEV, rows_of

pytestmark = pytest.mark.gpu

# tokens in front of the first row, the rows, tokens behind the last one; a tile is 168 tokens (264 backwards), a group 16 tiles
SHAPES = {"tail": (0, [100, 0, 57], 13), "long_tail": (0, [300, 20], 9000), "tail_from_a_tile": (0, [168, 168 * 3], 700),
          "tail_from_a_backward_tile": (0, [264 * 5], 264 * 40), "front": (77, [1000, 5], 0), "both": (6000, [40, 0, 900], 6000),
          "nothing_but_room": (0, [0, 0, 0], 5000), "rows_in_the_middle_of_nothing": (3000, [0, 1, 0], 3000),
          "little": (3, [2], 4)}


@pytest.mark.parametrize("name", sorted(SHAPES))
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 130), (torch.float16, 5), (torch.float32, 70)])
def test_tokens_in_no_row(name, reverse, dtype, dim):
    front, lengths, behind = SHAPES[name]
    print(f"gated_scan {name} dim={dim} {dtype} reverse={reverse}", flush=True)
    off = rows_of(lengths)
    total = int(off[-1])
    g = torch.Generator().manual_seed(7)
    inner = [torch.randn((total, dim), generator=g).to(dtype).to(DEV) for _ in range(3)]
    inner[1] += 3.0
    h0, dlast = (torch.randn((len(lengths), dim), generator=g).to(DEV) for _ in range(2))

    def run(x, gate, dy, offsets):
        leaves = [x.clone().requires_grad_(True), gate.clone().requires_grad_(True), h0.clone().requires_grad_(True)]
        y, last = lm_ops.gated_scan(leaves[0], leaves[1], torch.from_numpy(offsets).to(DEV), h0=leaves[2], reverse=reverse)
        return (y, last) + torch.autograd.grad((y, last), leaves, (dy, dlast))

    want = run(*inner, off)
    wide = []
    for t, value in zip(inner, (float("nan"), float("inf"), 5.0)):     # (what is not initialised may be anything)
        w = torch.full((front + total + behind, dim), value, dtype=dtype, device=DEV)
        w[front:front + total] = t
        wide.append(w)
    got = run(*wide, off + front)
    rows = slice(front, front + total)
    tol = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[dtype]
    for i in (0, 2, 3):                                                # y, dx, dgate: cut into tiles elsewhere, so not the same bits
        assert (got[i][:front] == 0).all() and (got[i][front + total:] == 0).all()
        assert torch.allclose(got[i][rows].float(), want[i].float(), rtol=tol, atol=1e-4)
    for i in (1, 4):                                                   # last, dh0
        assert torch.allclose(got[i], want[i], rtol=1e-5, atol=1e-4)


def test_scan_of_what_the_packer_leaves():
    """Ids packed into a buffer of the batch's capacity, embedded and scanned without a look at how many there are."""
    from dnatok_amd import encoders
    lens = torch.tensor([7, 0, 300, 41], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, 20, 20, 520, 600], device=DEV)
    tok = torch.arange(600, dtype=torch.int32, device=DEV) % 90
    ids, offsets, _ = encoders.pack_ragged(tok, off, lens)
    total = int(lens.sum())
    assert ids.numel() > total
    g = torch.Generator().manual_seed(8)
    table = torch.randn((90, 2 * 64), generator=g).to(DEV)
    both = table[ids.clamp(0, 89).long()]
    y, last = lm_ops.gated_scan(both[:, :64], both[:, 64:], offsets)
    want_y, want_last = lm_ops.gated_scan(both[:total, :64], both[:total, 64:], offsets)
    assert torch.equal(y[:total], want_y) and torch.equal(last, want_last) and (y[total:] == 0).all()
