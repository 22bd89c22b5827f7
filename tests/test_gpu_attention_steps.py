"""Single tokens of linear attention: many of them in a row, and what is infinite."""
import math

import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import attention_reference as ref
from tests.test_gpu_attention_infinities import DECAYS, KINDS, compare, plant
from tests.test_gpu_linear_attention import TYPES, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_many_steps_keep_the_rate():
    """20,000 steps that only decay.  A step rounds a cell once, by up to u = 2^-24 of it to either side: after n steps that is some
    sqrt(n) u (8.4e-6), and six times that is asked for of the mean over 4,096 cells, which is nearer.  exp(log_decay) rounded to 32 bits
    is off by 2.4e-8 to 3e-8 for these rates, which over n steps is 4.8e-4 and more."""
    n, rates = 20000, []
    for i in range(1000):
        ld = torch.tensor(-1e-5 * 1.01 ** i, dtype=torch.float32)
        off = (torch.exp(ld.double()).float().double() - torch.exp(ld.double())).abs().item()
        if off > 2.4e-8 and -ld.item() * n < 8:
            rates.append(ld.item())
    heads = min(len(rates), 8)
    assert heads == 8
    ld = torch.tensor(rates[:heads], device=DEV)
    g = torch.Generator().manual_seed(0)
    start = (1.0 + torch.rand((1, heads, 64, 64), generator=g)).to(DEV)
    state = start.clone()
    zero = torch.zeros((1, heads, 64), device=DEV)
    for _ in range(n):
        lm_ops.linear_attention_step(zero, zero, zero, ld, state, out_state=state)
    rate = (state.double() / start.double()).log().mean((0, 2, 3))
    assert (rate - n * ld.double()).abs().max().item() <= 6 * math.sqrt(n) * ref.U


@pytest.mark.parametrize("kind", [k for k in KINDS if not k.startswith("d")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(24, 40), (13, 7)])
def test_infinities(dims, dtype, kind):
    print(f"step {dims} {dtype} {kind}", flush=True)
    data = plant(inputs([1] * 9, 6, 3, *dims, dtype, 1, decay=DECAYS), kind, 3)
    q, k, v, ld, off, h0, _, _ = data
    y, new = lm_ops.linear_attention_step(q, k, v, ld, h0)
    odd = compare({"y": y, "last": new}, data, dtype, 1)
    assert odd
    first, _ = lm_ops.linear_attention_step(q, k, v, ld)                 # no state: the decays do not matter
    compare({"y": first}, (q, k, v, ld, off, None, None, None), dtype, 1)


@pytest.mark.parametrize("kind", ["v", "v of both signs", "k", "h0"])
def test_steps_are_the_rows(kind):
    """The prompt's way and the steps' give the same infinities."""
    q, k, v, ld, off, h0, dy, dlast = plant(inputs([40], 6, 3, 16, 24, torch.bfloat16, 2, decay=DECAYS), kind, 20)
    y, last = lm_ops.linear_attention(q, k, v, ld, torch.tensor(off, device=DEV), h0=h0)
    state = h0.clone()
    for t in range(40):
        out, _ = lm_ops.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], ld, state, out_state=state)
        assert torch.equal(torch.isnan(out), torch.isnan(y[t:t + 1])), t
        assert torch.equal(out == math.inf, y[t:t + 1] == math.inf) and torch.equal(out == -math.inf, y[t:t + 1] == -math.inf), t
    assert torch.equal(torch.isnan(state), torch.isnan(last)) and torch.equal(torch.isinf(state), torch.isinf(last))


def test_a_token_out_of_a_long_prompt():
    """One token of one row, whose stride to the next is that of no address: in a step, in a row, and in its backward pass."""
    g = torch.Generator().manual_seed(3)
    part = torch.randn((1, 12, 16), generator=g).to(DEV)
    long = torch.empty((1, 2 ** 17, 12, 16), device=DEV)
    long[:, -1] = part
    ld = torch.tensor([-0.1, -0.2, -0.3, 0.0], device=DEV)
    q, k, v = long[:, -1].split(4, 1)
    assert q.stride(0) > 2 ** 23
    want = lm_ops.linear_attention_step(*part.split(4, 1), ld)
    got = lm_ops.linear_attention_step(q, k, v, ld)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    off, leaves = torch.tensor([0, 1], device=DEV), [t.detach().requires_grad_(True) for t in (q, k, v)]
    y, last = lm_ops.linear_attention(*leaves, ld, off)
    data = (q, k, v, ld, off.tolist(), None, torch.ones((1, 4, 16)), None)
    got = {"y": y, "last": last, **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y.sum(), leaves)))}
    assert compare(got, data, torch.float32, 1) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_out_of_long_prompts(dtype):
    """The last tokens of dense prompts, 2^23 elements and more apart."""
    q, k, v, ld, off, h0, _, _ = inputs([1] * 3, 4, 2, 16, 24, dtype, 4)
    far = []
    for t, apart in ((q, 2 ** 23), (k, 2 ** 23 + 7), (v, 2 ** 24)):
        wide = torch.empty(2 * apart + t.shape[1] * t.shape[2], dtype=dtype, device=DEV)
        far.append(torch.as_strided(wide, t.shape, (apart, t.shape[2], 1)).copy_(t))
    want = lm_ops.linear_attention_step(q, k, v, ld, h0)
    for mix in (far, [far[0], k, v], [q, k, far[2]]):
        got = lm_ops.linear_attention_step(*mix, ld, h0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError, match="overlaps"):                    # where the tokens are, not where they are copied to
        wide = torch.zeros((2, 2 ** 23), device=DEV)
        part = wide[:, :4 * 16].view(2, 4, 16)
        lm_ops.linear_attention_step(part, part, part, ld, out_state=wide.view(-1)[:2 * 4 * 16 * 16].view(2, 4, 16, 16))


@pytest.mark.parametrize("rows", [65535, 65536, 140000])
def test_many_rows(rows):
    """As many rows as a search over many beams has: y = scale q (g h0 + k v^T) of each."""
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k = (torch.randn((rows, 2, 8), generator=g, device=DEV) for _ in range(2))
    v = torch.randn((rows, 1, 2, 4), generator=g, device=DEV)[:, 0, :, :]
    h0 = torch.randn((rows, 2, 8, 4), generator=g, device=DEV)
    ld = torch.tensor([-0.25, -2.0], device=DEV)
    print("step of", rows, "rows", flush=True)
    y, new = lm_ops.linear_attention_step(q, k, v, ld, h0)
    kv = k.double()[..., None] * v.double()[:, :, None]
    old = torch.exp(ld.double())[:, None, None] * h0.double()
    # a cell: two products, a sum, and the decay's own roundings; y: eight of those and eight sums
    assert ((new.double() - old - kv).abs() <= 6 * ref.U * (old.abs() + kv.abs())).all()
    size = 8 ** -0.5 * (q.double().abs()[..., None] * (old.abs() + kv.abs())).sum(2)
    assert ((y.double() - 8 ** -0.5 * (q.double()[..., None] * (old + kv)).sum(2)).abs() <= 20 * ref.U * size).all()
    again, _ = lm_ops.linear_attention_step(q, k, v, ld)
    assert ((again.double() - 8 ** -0.5 * (q.double()[..., None] * kv).sum(2)).abs() <= 20 * ref.U * size).all()
    same = h0.clone()
    y2, out = lm_ops.linear_attention_step(q, k, v, ld, same, out_state=same)
    assert out is same and torch.equal(out, new) and torch.equal(y2, y)
