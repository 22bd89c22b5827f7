"""Tensors past 2^31 elements: the places behind that border are computed as those in front of it."""
import pytest
import torch

from dnatok_amd import lm_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BORDER = 2 ** 31


def test_attention_behind_2_to_the_31():
    total, heads, dim = 1100000, 16, 128
    assert total * heads * dim > BORDER
    rows = [0, 600000, 1099000, total]
    print("linear_attention of", total, "tokens", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(0)
    q, k, v, dy = (torch.empty((total, heads, dim), dtype=torch.bfloat16, device=DEV).normal_(generator=gen) for _ in range(4))
    ld = torch.linspace(-3.0, -0.001, heads, device=DEV)
    off = torch.tensor(rows, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    y, last = lm_ops.linear_attention(*leaves, ld, off)
    grads = torch.autograd.grad(y, leaves, dy)
    tail = slice(rows[2], total)
    own = [t.detach()[tail].clone().requires_grad_(True) for t in (q, k, v)]
    # (a row of its own may be cut elsewhere: results to within what the two sums round differently, 2^-16 of a type's unit of 2^-8)
    y1, last1 = lm_ops.linear_attention(*own, ld, torch.tensor([0, total - rows[2]], device=DEV))
    grads1 = torch.autograd.grad(y1, own, dy[tail])
    for got, want in ((y[tail], y1), *zip([t[tail] for t in grads], grads1)):
        got, want = got.detach().float(), want.detach().float()
        assert (got - want).abs().max() <= 2 ** -7 * want.abs().max() and (got - want).norm() <= 2 ** -9 * want.norm()
    assert (last[2] - last1[0]).norm() <= 1e-5 * last1.norm()


def test_embedding_behind_2_to_the_31():
    n, dim, vocab = 4300000, 512, 50
    assert n * dim > BORDER
    print("embedding of", n, "tokens", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(0, vocab - 1, (n,), generator=gen, device=DEV, dtype=torch.int32)
    ids[-700:] = vocab - 1                                                # an id that only the last tokens have
    weight = torch.randn((vocab, dim), generator=gen, device=DEV).bfloat16().requires_grad_(True)
    y = lm_ops.embedding(ids, weight, scale=0.5)
    assert torch.equal(y[-1000:].detach(), (weight.detach()[ids[-1000:].long()].float() * 0.5).bfloat16())
    dy = torch.empty_like(y).normal_(generator=gen)
    grad, = torch.autograd.grad(y, weight, dy)
    want = dy[-700:].double().sum(0) * 0.5
    size = dy[-700:].double().abs().sum(0) * 0.5
    assert ((grad[-1].double() - want).abs() <= 702 * 2 ** -24 * size + 2 ** -8 * want.abs() * 1.01).all()


def test_beams_and_states_behind_2_to_the_31():
    groups, beams, vocab = 17000, 4, 32000
    assert groups * beams * vocab > BORDER
    print("beam_select of", groups, "groups", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(2)
    logits = torch.empty((groups * beams, vocab), dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    scores = -torch.rand((groups, beams), generator=gen, device=DEV)
    got = lm_ops.beam_select(logits, scores)
    want = lm_ops.beam_select(logits[-8 * beams:], scores[-8:])
    # (few rows are taken in slices: the sums of exponentials in another order, 64 bits)
    assert torch.equal(got[1][-8:], want[1]) and torch.equal(got[2][-8:], want[2])
    assert (got[0][-8:] - want[0]).abs().max() <= 2 ** -20
    moved, = lm_ops.reorder_rows([logits], got[2])
    at = (torch.arange(groups, device=DEV)[:, None] * beams + got[2]).view(-1)
    assert torch.equal(moved[-64:], logits[at[-64:]]) and torch.equal(moved[:64], logits[at[:64]])
