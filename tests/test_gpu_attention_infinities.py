"""Infinities and NaN in linear attention go on as the recurrence has them (attention_reference, in 64 bits): the same outputs, states and
gradients are infinite, of the same sign, or NaN, and all others are as near as ever.  A state that is infinite stays so
as long as anything is left of it; a decay of -inf leaves nothing, whatever it was."""
import math

import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import attention_reference as ref
from tests.test_gpu_linear_attention import TYPES, inputs, run

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = math.inf, math.nan
DECAYS = torch.tensor([0.0, -1e-6, -1e-3, -0.5, -200.0, -INF])


def compare(got, data, dtype, longest, scale=None, reverse=False):
    q, k, v, ld, off, h0, dy, dlast = data
    args = (q, k, v, ld, off, h0, scale, reverse) + ((dy, dlast) if "dq" in got else ())
    want, size = ref.attention(*args), ref.attention(*args, sizes=True)
    count = ref.roundings(dtype, q.shape[2], v.shape[2], longest) + q.shape[1] // k.shape[1]
    odd = 0
    for name, value in got.items():
        value, w = value.detach().cpu().double(), want[name]
        # (e^-200 is 1.4e-87; the smallest number of 32 bits is 2^-149, so whatever is below half of that is 0 when it is rounded)
        w = torch.where(w.abs() < 2.0 ** -150, 0.0, w)
        finite = torch.isfinite(w)
        odd += int((~finite).sum())
        assert torch.equal(torch.isnan(value), torch.isnan(w)), name
        assert torch.equal(value[torch.isinf(w)], w[torch.isinf(w)]), name
        ref.check(torch.where(finite, value, 0.0), torch.where(finite, w, 0.0), torch.where(finite, size[name], 0.0),
                  torch.float32 if name in ("last", "dh0") else dtype, count, name)
    return odd


def plant(data, kind, at):
    """Numbers that are none at token ``at`` and some behind it; all of keys and queries are positive, as after a feature map."""
    q, k, v, ld, off, h0, dy, dlast = data
    q, k, v, h0, dy, dlast = (t.clone() for t in (q, k, v, h0, dy, dlast))
    q, k = q.abs(), k.abs()
    if kind == "v":
        v[at, 1, 3] = INF
        v[at + 5, 0, 0] = -INF
        k[at + 5, 0, 2] = 0.0                      # (one row of the state becomes NaN, the others infinite)
    elif kind == "v of both signs":
        v[at, 0, 4], v[at + 3, 0, 4], v[at + 3, 2, 1] = INF, -INF, NAN
    elif kind == "k":
        k[at, 1, 3] = INF
        v[at, 1, 2] = 0.0
    elif kind == "q":
        q[at, 2, 5], q[at + 1, 4, 0] = INF, -INF
    elif kind == "h0":
        h0[0, :, 2, 3] = INF
        h0[-1, :, 1, 1] = -INF
        h0[-1, 0, 0, 0] = NAN
    elif kind == "dy":
        dy[at, 0, 3], dy[at, 3, 1], dy[at + 2, 5, 0] = INF, -INF, NAN
    elif kind == "dlast":
        dlast[0, :, 2, 3] = -INF
        dlast[-1, 1, 0, 0] = NAN
    return q, k, v, ld, off, h0, dy, dlast


KINDS = ["v", "v of both signs", "k", "q", "h0", "dy", "dlast"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_in_chunks(dtype, reverse, kind):
    print(f"rows in chunks {dtype} reverse={reverse} {kind}", flush=True)
    data = plant(inputs([40, 0, 200], 6, 3, 24, 40, dtype, 1, decay=DECAYS), kind, 40 + 97)
    assert compare(run(*data, reverse=reverse), data, dtype, 200, reverse=reverse)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_in_pieces(dtype, reverse, kind):
    """Three pieces of some 530 tokens: what the cuts pass on."""
    print(f"a row in pieces {dtype} reverse={reverse} {kind}", flush=True)
    data = plant(inputs([1600], 6, 3, 13, 7, dtype, 2, decay=DECAYS), kind, 700)
    assert compare(run(*data, reverse=reverse), data, dtype, 1600, reverse=reverse)


@pytest.mark.parametrize("kind", ["v", "k", "h0"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(128, 128), (128, 64), (64, 64), (48, 33)])
def test_wide_heads(dims, dtype, kind):
    print(f"wide heads {dims} {dtype} {kind}", flush=True)
    data = plant(inputs([150], 6, 6, *dims, dtype, 3, decay=DECAYS), kind, 70)
    assert compare(run(*data), data, dtype, 150)


def test_numbers_of_any_sign():
    for dtype in TYPES:
        q, k, v, ld, off, h0, dy, dlast = inputs([300], 6, 6, 16, 16, dtype, 4, decay=DECAYS)
        v[100, :, 3], k[150, :, 2], q[200, :, 1] = INF, -INF, INF
        data = (q, k, v, ld, off, h0, dy, dlast)
        assert compare(run(*data), data, dtype, 300)


def test_what_is_finite_keeps_its_bits():
    """An infinite value reaches its own column of the state only, and no earlier step."""
    for dtype in TYPES:
        q, k, v, ld, off, h0, dy, dlast = inputs([1600], 2, 2, 32, 48, dtype, 5)
        clean = run(q, k, v, ld, off, h0, dy, dlast)
        bad = v.clone()
        bad[600, 1, 7] = INF
        got = run(q, k, bad, ld, off, h0, dy, dlast)
        others = [c for c in range(48) if c != 7]
        assert torch.equal(got["y"][:, 0], clean["y"][:, 0]) and torch.equal(got["y"][:, 1, others], clean["y"][:, 1, others])
        assert torch.equal(got["y"][:600], clean["y"][:600])
        assert torch.equal(got["last"][..., others], clean["last"][..., others])
        assert torch.equal(got["dv"], clean["dv"]) and torch.equal(got["dh0"], clean["dh0"])
        assert torch.equal(got["dq"][:600], clean["dq"][:600]) and not torch.isfinite(got["dq"][600:, 1]).any()


def test_a_decay_that_is_nan():
    q, k, v, ld, off, h0, dy, dlast = inputs([70, 700], 2, 2, 16, 16, torch.bfloat16, 6)
    ld[0] = NAN
    y, last = lm_ops.linear_attention(q, k, v, ld, torch.tensor(off, device=DEV), h0=h0)
    assert torch.isnan(y[:, 0]).all() and torch.isnan(last[:, 0]).all()
    assert torch.isfinite(y[:, 1]).all() and torch.isfinite(last[:, 1]).all()
