"""Linear attention with decays token by token in 64 bits (torch, CPU), and how far results in 32 bits may be from it.

Every result is a walk: T_t = D_(t-1) + b_t c_t^T, D_t = g T_t, out_t = a_t T_t.  The same walk over the operands' sizes gives, for each
cell, the sum of what its terms weigh; the tolerance is a number of roundings of u = 2^-24 times that sum.  The roundings that a term
of age n can meet: sums over Dk (or Dv) and twice over the 64 steps of a chunk, the state's decay once a chunk
(T / 64, and its factor's own), a decay exp(n ld), which is off by 2 n |ld| u of itself (n |ld| is at most 88 before it
vanishes), a handful of factors and joins; for bfloat16 also scores and states in two parts of 8 bits, off by 2^-18 of
themselves (64 u each, and 2^-26 for what is added to a state), for float16 by 2^-22 (4 u each)."""
import torch

U = 2.0 ** -24
SPLIT = {torch.float32: 0, torch.bfloat16: 160, torch.float16: 16}
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a unit of the last place: eps / 2
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def walk(a, b, c, log_decay, offsets, start, reverse, late):
    """a, b, c [total, H, .] in 64 bits; start and the returned end [rows, H, ., .]; ``late``: a step's decay comes behind it."""
    g = torch.exp(log_decay)[:, None, None]
    out = torch.zeros((a.shape[0], a.shape[1], c.shape[2]), dtype=torch.float64)
    end = start.clone()
    for r in range(len(offsets) - 1):
        tokens = range(offsets[r], offsets[r + 1])
        state = end[r].clone()
        for t in reversed(tokens) if reverse else tokens:
            if not late:
                state = torch.where(g == 0, 0.0, g * state)
            state = state + b[t][:, :, None] * c[t][:, None, :]
            out[t] = (a[t][:, :, None] * state).sum(1)
            if late:
                state = torch.where(g == 0, 0.0, g * state)
        end[r] = state
    return out, end


def attention(q, k, v, log_decay, offsets, h0=None, scale=None, reverse=False, dy=None, dlast=None, sizes=False):
    """y, last and, where dy is given, dq, dk, dv, dh0.  ``sizes``: of the operands' magnitudes, for the tolerances."""
    q, k, v, log_decay, h0, dy, dlast = (None if t is None else t.detach().cpu().double() for t in
                                         (q, k, v, log_decay, h0, dy, dlast))
    heads, kv = q.shape[1], k.shape[1]
    shared, scale = heads // kv, q.shape[2] ** -0.5 if scale is None else scale
    rows = len(offsets) - 1
    if h0 is None:
        h0 = torch.zeros((rows, heads, q.shape[2], v.shape[2]), dtype=torch.float64)
    if dlast is None:
        dlast = torch.zeros_like(h0)
    if sizes:
        q, k, v, h0, dlast, scale = q.abs(), k.abs(), v.abs(), h0.abs(), dlast.abs(), abs(scale)
        dy = None if dy is None else dy.abs()
    k, v = k.repeat_interleave(shared, 1), v.repeat_interleave(shared, 1)
    y, last = walk(q, k, v, log_decay, offsets, h0, reverse, False)
    result = {"y": scale * y, "last": last}
    if dy is not None:
        dy = scale * dy
        result["dq"] = walk(dy, v, k, log_decay, offsets, h0.transpose(2, 3), reverse, False)[0]
        dv, result["dh0"] = walk(k, q, dy, log_decay, offsets, dlast, not reverse, True)
        dk, _ = walk(v, dy, q, log_decay, offsets, dlast.transpose(2, 3), not reverse, True)
        result["dk"] = dk.view(dk.shape[0], kv, shared, dk.shape[2]).sum(2)
        result["dv"] = dv.view(dv.shape[0], kv, shared, dv.shape[2]).sum(2)
    return result


def roundings(dtype, dim_k, dim_v, longest):
    return dim_k + dim_v + 3 * 64 + 180 + 40 + longest / 32 + SPLIT[dtype]


def check(got, want, size, dtype, count, what):
    """``got`` is ``want`` up to ``count`` roundings of ``size`` and one to its own type."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    slack = count * U * size + HALF[dtype] * want.abs() * (1 + 2 * HALF[dtype]) + TINY[dtype]
    off = (got - want).abs() - slack
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = off.max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: {worst} beyond the tolerance"
