"""Plain 64-bit restatements of the model operators, token by token and cell by cell (numpy, CPU)."""
import numpy as np


def sigmoid(v):
    e = np.exp(-np.abs(v))
    return np.where(v >= 0, 1.0 / (1.0 + e), e / (1.0 + e))


def scan(x, gate, offsets, h0=None, reverse=False):
    """(y, last) of the recurrence over packed rows, float64."""
    n, dim = len(offsets) - 1, x.shape[1]
    y = np.zeros_like(x)
    last = np.zeros((n, dim)) if h0 is None else h0.copy()
    f, keep = sigmoid(gate), sigmoid(-gate)
    for b in range(n):
        tokens = range(offsets[b], offsets[b + 1])
        h = last[b]
        for t in reversed(tokens) if reverse else tokens:
            h = f[t] * h + keep[t] * x[t]
            y[t] = h
        last[b] = h
    return y, last


def scan_grad(x, gate, offsets, dy, dlast, h0=None, reverse=False):
    """(dx, dgate, dh0) of sum(y dy) + sum(last dlast), from the formulas; and the largest |dh|."""
    n = len(offsets) - 1
    y, _ = scan(x, gate, offsets, h0, reverse)
    f, keep = sigmoid(gate), sigmoid(-gate)
    dx, dgate, dh0 = np.zeros_like(x), np.zeros_like(x), dlast.copy()
    most = np.abs(dlast).max(initial=0.0)
    for b in range(n):
        tokens = list(range(offsets[b], offsets[b + 1]))
        if reverse:
            tokens.reverse()
        carry = dlast[b]
        for i in range(len(tokens) - 1, -1, -1):
            t = tokens[i]
            before = y[tokens[i - 1]] if i else (np.zeros(x.shape[1]) if h0 is None else h0[b])
            dh = dy[t] + carry
            dx[t] = keep[t] * dh
            dgate[t] = dh * (before - x[t]) * f[t] * keep[t]
            carry = f[t] * dh
            most = max(most, np.abs(dh).max(initial=0.0))
        dh0[b] = carry
    return dx, dgate, dh0, most


def unpack4(q, k):
    """int32 [N, words] -> whole numbers [N, k]."""
    q = np.asarray(q).astype(np.int64) & 0xFFFFFFFF
    return ((q[:, :, None] >> (4 * np.arange(8))) & 15).reshape(q.shape[0], -1)[:, :k]


def w4(x, q, scales, zeros, k, group, bias=None):
    g = np.arange(k) // group
    w = unpack4(q, k) - (8.0 if zeros is None else zeros.astype(np.float64)[:, g])
    y = x @ (w * scales[:, g]).T
    return y if bias is None else y + bias


def logits(z, history=None, offsets=None, prompt=None, repetition=None, presence=None, frequency=None, bias=None,
           allowed=None, state=None):
    z = z.copy()
    rows, vocab = z.shape
    for r in range(rows):
        if history is not None:
            ids = history[offsets[r]:offsets[r + 1]]
            first = 0 if prompt is None else prompt[r]
            made = ids[first:]
            made = made[(made >= 0) & (made < vocab)]
            ids = ids[(ids >= 0) & (ids < vocab)]
            seen = np.bincount(ids, minlength=vocab) > 0
            c = np.bincount(made, minlength=vocab).astype(np.float64)
            if repetition is not None:
                z[r] = np.where(seen, np.where(z[r] > 0, z[r] / repetition[r], z[r] * repetition[r]), z[r])
            if presence is not None:
                z[r] -= presence[r] * (c > 0)
            if frequency is not None:
                z[r] -= frequency[r] * c
        if bias is not None:
            z[r] += bias if bias.ndim == 1 else bias[r]
        if allowed is not None:
            s = state[r] if state is not None else (0 if len(allowed) == 1 else r)
            if s >= len(allowed):
                z[r] = -np.inf
            elif s >= 0:
                words = allowed[s].astype(np.int64) & 0xFFFFFFFF
                ok = (words[np.arange(vocab) >> 5] >> (np.arange(vocab) & 31)) & 1
                z[r] = np.where(ok == 1, z[r], -np.inf)
    return z
