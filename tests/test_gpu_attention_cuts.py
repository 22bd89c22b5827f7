"""Rows of linear attention that are really cut, against 64 bits: dense ones, and heads of 128 x 128 (tolerances: attention_reference)."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support.attention_reference import U
from tests.test_gpu_linear_attention import DEV, TYPES, compare, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("rows,length,dims", [(1, 1100, (24, 40)), (2, 1500, (16, 16)), (3, 1025, (13, 7)), (2, 1200, (40, 72))])
def test_dense_rows(rows, length, dims, reverse, dtype):
    """Without offsets rows of one length are cut into equal pieces of 512 tokens and more: states, outputs and gradients."""
    print(f"dense {rows} x {length} {dims} {dtype} reverse={reverse}", flush=True)
    data = inputs([length] * rows, 4, 2, *dims, dtype, 31)
    q, k, v, ld, off, h0, dy, dlast = data
    leaves = [t.reshape(rows, length, *t.shape[1:]).detach().requires_grad_(True) for t in (q, k, v)] + [h0.detach().requires_grad_(True)]
    y, last = lm_ops.linear_attention(*leaves[:3], ld, h0=leaves[3], reverse=reverse)
    grads = torch.autograd.grad((y, last), leaves, (dy.view_as(y), dlast))
    got = {"y": y.flatten(0, 1), "last": last, **{n: g.flatten(0, 1) for n, g in zip(("dq", "dk", "dv"), grads)}, "dh0": grads[3]}
    compare(got, data, dtype, None, reverse, length)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dims", [(128, 128), (128, 64), (96, 128)])
def test_wide_heads(dims, reverse, dtype):
    print(f"cut rows, heads of {dims} {dtype} reverse={reverse}", flush=True)
    data = inputs([1100, 3, 600], 2, 1, *dims, dtype, 32)
    compare(run(*data, reverse=reverse), data, dtype, None, reverse, 1100)


def test_a_gradient_at_any_place():
    """What comes in for y lies where autograd has put it: tokens far apart, heads first, one number for all."""
    data = inputs([2, 0, 1], 2, 1, 16, 24, torch.bfloat16, 33)
    q, k, v, ld, off, h0, dy, dlast = data
    far = torch.as_strided(torch.empty(2 * 2 ** 23 + 48, dtype=torch.bfloat16, device=DEV), (3, 2, 24), (2 ** 23, 24, 1)).copy_(dy)
    want = run(*data)
    for other in (far, dy.transpose(0, 1).contiguous().transpose(0, 1), dy.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        got = run(q, k, v, ld, off, h0, other, dlast)
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_a_state_that_lasts_is_rounded_twice_a_chunk():
    """32 bits: what a chunk adds is summed by itself, so of 64 steps a state has two roundings, its decay's and the sum's.  With
    log_decay = -2.5e-4 the chunks' weights, squared, add up to 31: 62 roundings of at most u of a cell, each to its own side, are some
    sqrt(62) u = 7.9 u of the state's norm; one more for what each chunk's sum is off by."""
    q, k, v, _, off, _, _, _ = inputs([20000], 2, 2, 16, 16, torch.float32, 34)
    ld = torch.full((2,), -2.5e-4, device=DEV)
    for reverse in (False, True):
        _, last = lm_ops.linear_attention(q, k, v, ld, torch.tensor(off, device=DEV), reverse=reverse)
        age = torch.arange(20000, device=DEV, dtype=torch.float64)
        weight = torch.exp((age if reverse else age.flip(0)) * ld[0].double())
        want = (k.double() * weight[:, None, None]).permute(1, 2, 0).contiguous() @ v.double().transpose(0, 1).contiguous()
        assert (last[0].double() - want).norm() <= 9 * U * want.norm(), reverse
