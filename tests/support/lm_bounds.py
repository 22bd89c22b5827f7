"""How far the recurrence's results in 32 bits may be from those in 64 bits, cell by cell (numpy, CPU).

A token's f and k = 1 - f: the smaller of them, s, has a relative error of at most (|g| + 8) u (the rounding of g log2(e), an
exponential and a reciprocal of an ulp or two each, a product), the other an absolute one of as much.  A step rounds
products and sums, of magnitudes f |h|, k |x| and |h|, at most twice each.  Tokens in one row of a piece are met twice, once from
zero (the piece's own state, at most twice the largest |h| of the channel in the row) and once with what comes
in, and the factor of a piece rounds once a token and once a join.  An error made at a token goes on as the state does.
So, with H the largest |h| of a row's channel,

    e_t = f_t e_(t-1) + u (12 H + 4 (|g_t| + 8) s_t (|x_t| + 2 H))

bounds the state's error; the gradients' has the same form with dh in the place of h and dy in that of x.  u is 2^-24."""
import numpy as np

from tests.support.lm_reference import sigmoid

U = 2.0 ** -24


def _order(lo, hi, reverse):
    return range(hi - 1, lo - 1, -1) if reverse else range(lo, hi)


def scan(x, gate, offsets, dy=None, dlast=None, h0=None, reverse=False):
    """The results in 64 bits and their bounds, two dicts: y, last, and dx, dgate, dh0 where dy and dlast are given."""
    rows, dim = len(offsets) - 1, x.shape[1]
    f, k = sigmoid(gate), sigmoid(-gate)
    s, eps = np.minimum(f, k), U * (np.abs(gate) + 8.0)
    y, e = np.zeros_like(x), np.zeros_like(x)
    last = np.zeros((rows, dim)) if h0 is None else h0.copy()
    elast = np.zeros((rows, dim))
    train = dy is not None
    if train:
        dx, dg, edx, edg = (np.zeros_like(x) for _ in range(4))
        dh0, edh0 = dlast.copy(), np.zeros((rows, dim))
    for b in range(rows):
        tokens = list(_order(offsets[b], offsets[b + 1], reverse))
        if not tokens:
            continue
        h = last[b].copy()
        most = np.abs(h)
        for t in tokens:
            h = f[t] * h + k[t] * x[t]
            y[t] = h
            np.maximum(most, np.abs(h), out=most)
        last[b] = h
        err = np.zeros(dim)
        for t in tokens:
            err = f[t] * err + U * 12.0 * most + 4.0 * eps[t] * s[t] * (np.abs(x[t]) + 2.0 * most)
            e[t] = err
        elast[b] = err
        if not train:
            continue
        carry, dh = dlast[b].copy(), np.zeros((len(tokens), dim))
        for i in range(len(tokens) - 1, -1, -1):
            t = tokens[i]
            dh[i] = dy[t] + carry
            carry = f[t] * dh[i]
        dh0[b] = carry
        most = np.abs(dh).max(0)
        err = np.zeros(dim)
        first = np.zeros(dim) if h0 is None else h0[b]
        for i in range(len(tokens) - 1, -1, -1):
            t = tokens[i]
            before, ebefore = (y[tokens[i - 1]], e[tokens[i - 1]]) if i else (first, 0.0)
            step = err + U * 4.0 * most                                # (of dh; f times it goes on)
            dx[t] = k[t] * dh[i]
            edx[t] = k[t] * step + 4.0 * (eps[t] * s[t] + U * k[t]) * np.abs(dh[i])
            away = before - x[t]
            dg[t] = dh[i] * away * f[t] * k[t]
            edg[t] = f[t] * k[t] * (step * (np.abs(away) + ebefore) + np.abs(dh[i]) * (ebefore + U * np.abs(away))) + \
                (4.0 * eps[t] + 8.0 * U) * np.abs(dg[t])
            err = f[t] * step + U * 8.0 * f[t] * most + 4.0 * eps[t] * s[t] * 2.0 * most
        edh0[b] = err
    want, bound = {"y": y, "last": last}, {"y": e, "last": elast}
    if train:
        want.update(dx=dx, dgate=dg, dh0=dh0)
        bound.update(dx=edx, dgate=edg, dh0=edh0)
    return want, bound


def step(x, gate, h):
    """One token of each row: the state in 64 bits and its bound, without joins."""
    f, k = sigmoid(gate), sigmoid(-gate)
    eps = U * (np.abs(gate) + 8.0)
    s = np.minimum(f, k)
    return f * h + k * x, U * 4.0 * (f * np.abs(h) + k * np.abs(x)) + 2.0 * eps * s * (np.abs(h) + np.abs(x))
