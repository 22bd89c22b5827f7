"""What the operators around a recurrent model are timed on: the calls that a program makes through ``lm_ops`` to
embed tokens, to mix them with linear attention, and to search over several continuations.

Kinds of case, and what each stands for:

attend  linear attention with a decay for each head over packed rows: windows, one contig, reads of mixed
        lengths; forward, or forward and backward in a training step.  Queries, keys and values come as
        the parts of one projection's output, as a layer has them
step    the same for one new token of each row
embed   rows of an embedding for packed ids; forward, or forward and the weights' gradient
beam    one step of a beam search: the choice over beams and vocabulary, and the layers' states in their new order

``run`` computes them in elementary torch operations in 32 bits (in 64 where long sums or the order of neighbouring
scores need them), or, with ``own`` set, with the framework's operators.
"""
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # generation for one sequence: one token through one layer, a call that is all latency
        {"name": "step_1_h8_d64", "kind": "step", "rows": 1, "heads": 8, "kv_heads": 8, "dk": 64, "dv": 64,
         "dtype": "bfloat16"},
        # generation for many sequences at once
        {"name": "step_250_h8_d128", "kind": "step", "rows": 250, "heads": 8, "kv_heads": 2, "dk": 128, "dv": 128,
         "dtype": "float16"},
        # a batch of windows, forward only (scoring, or the prompts of a batch)
        {"name": "attend_64x8192_h8_d64", "kind": "attend", "layout": "even", "rows": 64, "length": 8192, "heads": 8,
         "kv_heads": 8, "dk": 64, "dv": 64, "dtype": "bfloat16", "reverse": False, "start": False, "train": False},
        # one contig, read from its end, continued from a state
        {"name": "attend_1x262147_h4_d128", "kind": "attend", "layout": "even", "rows": 1, "length": 262147, "heads": 4,
         "kv_heads": 4, "dk": 128, "dv": 128, "dtype": "float16", "reverse": True, "start": True, "train": False},
        # a training step on windows of tokens
        {"name": "train_256x1024_h4_d128", "kind": "attend", "layout": "even", "rows": 256, "length": 1024, "heads": 4,
         "kv_heads": 4, "dk": 128, "dv": 128, "dtype": "bfloat16", "reverse": False, "start": False, "train": True},
        # a training step in 32 bits on long reads of mixed lengths, shared keys and values, sizes that fit no tile
        {"name": "train_300_reads_h6_d48", "kind": "attend", "layout": "long_reads", "rows": 300, "length": 2000, "heads": 6,
         "kv_heads": 2, "dk": 48, "dv": 40, "dtype": "float32", "reverse": True, "start": True, "train": True},
        # one new token of each of a few sequences
        {"name": "embed_64x512_v4096", "kind": "embed", "tokens": 64, "vocab": 4096, "dim": 512, "dtype": "bfloat16",
         "train": False},
        # a batch of windows, forward only
        {"name": "embed_524288x512_v4096", "kind": "embed", "tokens": 524288, "vocab": 4096, "dim": 512, "dtype": "bfloat16",
         "train": False},
        # a training step over the larger vocabulary
        {"name": "embed_train_262144x512_v32000", "kind": "embed", "tokens": 262144, "vocab": 32000, "dim": 512,
         "dtype": "bfloat16", "train": True},
        # a training step on single nucleotides: few ids, each of them very often; an odd number of channels
        {"name": "embed_train_1000003x203_v12", "kind": "embed", "tokens": 1000003, "vocab": 12, "dim": 203,
         "dtype": "float32", "train": True},
        # one sequence, a few beams, the smaller vocabulary: latency
        {"name": "beam_1x4_v4096", "kind": "beam", "groups": 1, "beams": 4, "width": 4, "vocab": 4096, "dtype": "float32",
         "dim": 512, "heads": 8, "masked": False, "ended": False},
        # a batch of searches over the larger vocabulary, some tokens forbidden, some beams at their end
        {"name": "beam_64x8_v32000", "kind": "beam", "groups": 64, "beams": 8, "width": 8, "vocab": 32000,
         "dtype": "bfloat16", "dim": 1024, "heads": 8, "masked": True, "ended": True},
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng):
    kv = rng.choice([1, 1, 2, 4, 8])
    size = (lambda: rng.choice([32, 64, 64, 128, 128, 16 + rng.randrange(113)]))
    return {"heads": kv * rng.choice([1, 1, 1, 2, 3]), "kv_heads": kv, "dk": size(), "dv": size()}


def draw(rng):
    kind = rng.choice(["step", "attend", "attend", "attend", "embed", "embed", "beam"])
    case = {"kind": kind}
    if kind == "step":
        case.update(rows=_between(rng, 1, 250), dtype=rng.choice(sorted(TYPES)), **_heads(rng))
        while case["rows"] * case["heads"] * case["dk"] * case["dv"] > 32000000:
            case["rows"] //= 2
    elif kind == "attend":
        layout = rng.choice(["even", "reads", "long_reads"])
        case.update(_heads(rng))
        dtype, train = rng.choice(sorted(TYPES)), rng.random() < 0.5
        cells = case["heads"] * max(case["dk"], case["dv"], 48)
        most = (60000000 if train else 130000000) // (2 if dtype == "float32" else 1) // cells
        if layout == "even":
            length = _between(rng, 1, most)
            rows = _between(rng, 1, max(1, min(4000, most // length)))
        elif layout == "reads":
            length, rows = 200, _between(rng, 1, max(1, min(10000, most // 400)))
        else:
            length, rows = 2000, _between(rng, 1, max(1, most // 5000))
        case.update(layout=layout, rows=rows, length=length, dtype=dtype, reverse=rng.random() < 0.5,
                    start=rng.random() < 0.5, train=train)
    elif kind == "embed":
        dim, train = _between(rng, 16, 2048), rng.random() < 0.6
        if rng.random() < 0.6:
            dim = max(64, dim - dim % 64)
        case.update(tokens=_between(rng, 1, min(1000003, 200000000 // dim)),
                    vocab=rng.choice([12, 4096, 32000, _between(rng, 5, 32000)]), dim=dim,
                    dtype=rng.choice(sorted(TYPES)), train=train)
    else:
        beams, vocab = _between(rng, 1, 16), rng.choice([4096, 32000, _between(rng, 50, 32000)])
        case.update(groups=_between(rng, 1, max(1, min(64, 16000000 // (beams * vocab)))), beams=beams,
                    width=rng.choice([beams, beams, 2 * beams]), vocab=vocab, dtype=rng.choice(sorted(TYPES)),
                    dim=_between(rng, 16, 1024), heads=rng.choice([0, 2, 8]), masked=rng.random() < 0.5,
                    ended=rng.random() < 0.5)
    return case


# ---- inputs ---------------------------------------------------------------------------------

def _in_any_order(lengths, gen):
    """The batch's lengths are those of its size; which row has which comes from the seed."""
    return lengths[torch.randperm(lengths.numel(), generator=gen, device="cuda")]


def _lengths(case, gen):
    rows = case["rows"]
    if case["layout"] == "even":
        return torch.full((rows,), case["length"], dtype=torch.int64, device="cuda")
    if case["layout"] == "reads":                                # 100 - 300, evenly
        return _in_any_order(100 + torch.arange(rows, device="cuda") * 201 // rows, gen)
    q = (torch.arange(rows, device="cuda", dtype=torch.float64) + 0.5) / rows
    z = torch.special.ndtri(q)                                   # lognormal, median 2,000
    return _in_any_order(torch.exp(z * 0.87 + 7.6009).round().long().clamp(100, 131072), gen)


def _offsets(lengths):
    off = torch.zeros(lengths.numel() + 1, dtype=torch.int64, device="cuda")
    torch.cumsum(lengths, 0, out=off[1:])
    return off


def _parts(total, case, dtype, gen):
    """Queries, keys and values as a projection leaves them next to each other, and the heads' decays: half-lives from
    one token to a few thousand."""
    h, g, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    both = torch.empty((total, h * dk + g * (dk + dv)), dtype=dtype, device="cuda").normal_(generator=gen)
    q, k, v = both.split([h * dk, g * dk, g * dv], 1)
    forget = torch.exp2(-1.0 - 11.0 * torch.rand(h, generator=gen, device="cuda", dtype=torch.float64))
    return q.view(total, h, dk), k.view(total, g, dk), v.view(total, g, dv), torch.log1p(-forget).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}

    def normal(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)

    if case["kind"] == "step":
        q, k, v, decay = _parts(case["rows"], case, TYPES[case["dtype"]], gen)
        s.update(q=q, k=k, v=v, decay=decay, state=normal(case["rows"], case["heads"], case["dk"], case["dv"]))
    elif case["kind"] == "attend":
        dtype, rows, h = TYPES[case["dtype"]], case["rows"], case["heads"]
        off = _offsets(_lengths(case, gen))
        total = int(off[-1])
        q, k, v, decay = _parts(total, case, dtype, gen)
        h0 = normal(rows, h, case["dk"], case["dv"]) if case["start"] else None
        s.update(q=q, k=k, v=v, decay=decay, off=off, h0=h0)
        if case["train"]:
            s.update(dy=normal(total, h, case["dv"], dtype=dtype), dlast=normal(rows, h, case["dk"], case["dv"]))
            for t in (q, k, v) if h0 is None else (q, k, v, h0):
                t.requires_grad_(True)
    elif case["kind"] == "embed":
        n, vocab, dim, dtype = case["tokens"], case["vocab"], case["dim"], TYPES[case["dtype"]]
        u = torch.rand(n, generator=gen, device="cuda")
        s.update(ids=(u * u * vocab).to(torch.int32).clamp(max=vocab - 1),           # some tokens come often
                 weight=normal(vocab, dim, dtype=dtype), scale=math.sqrt(dim))
        if case["train"]:
            s["dy"] = normal(n, dim, dtype=dtype)
            s["weight"].requires_grad_(True)
    else:
        groups, beams, vocab, dtype = case["groups"], case["beams"], case["vocab"], TYPES[case["dtype"]]
        logits = (3.0 * normal(groups * beams, vocab)).to(dtype)
        if case["masked"]:                                       # a grammar leaves a quarter of the tokens
            logits.masked_fill_(torch.rand((groups * beams, vocab), generator=gen, device="cuda") >= 0.25, float("-inf"))
        s.update(logits=logits, scores=-10.0 * torch.rand((groups, beams), generator=gen, device="cuda"),
                 ended=torch.rand((groups, beams), generator=gen, device="cuda") < 0.2 if case["ended"] else None,
                 # a layer of each kind of recurrence
                 states=[normal(groups * beams, case["dim"])])
        if case["heads"]:
            s["states"].append(normal(groups * beams, case["heads"], 64, 64))
    return s


# ---- the operators --------------------------------------------------------------------------

CHUNK = 128


def _chunks(lens):
    """The rows cut into chunks: each token's place [chunks, CHUNK], which of them are there, the chunks' row and number in
    their row, and the number of chunks of each row."""
    dev = lens.device
    n = (lens + CHUNK - 1) // CHUNK
    first = torch.cumsum(n, 0) - n
    row = torch.repeat_interleave(torch.arange(lens.numel(), device=dev), n)
    number = torch.arange(row.numel(), device=dev) - first[row]
    start = (torch.cumsum(lens, 0) - lens)[row] + number * CHUNK
    at = torch.arange(CHUNK, device=dev)
    there = number[:, None] * CHUNK + at < lens[row][:, None]
    return (start[:, None] + at) * there, there, row, number, n, first


def _walk(a, b, c, log_decay, lens, start, reverse, decayed):
    """T_t = D_(t-1) + b_t c_t^T and D_t = g T_t in every row: a_t T_t for every token, and what is left behind the
    rows' last one.  ``start`` [rows, H, ., .] is in front of a row's first token, and what is returned behind its last:
    T if not ``decayed`` (so that it decays on its way in), D otherwise.  a, b, c: float32 [total, H, .]."""
    if reverse:
        y, last = _walk(a.flip(0), b.flip(0), c.flip(0), log_decay, lens.flip(0), start.flip(0), False, decayed)
        return y.flip(0), last.flip(0)
    total, heads, _ = a.shape
    y, last = c.new_empty((total, heads, c.shape[2])), start.clone()
    if total == 0:
        return y, last
    index, there, row, number, n, first = _chunks(lens)

    def cut(x):                                                   # [chunks, H, CHUNK, .]
        return (x[index] * there[:, :, None, None]).transpose(1, 2).contiguous()

    a, b, c = cut(a), cut(b), cut(c)
    ld = log_decay.double()
    t = torch.arange(CHUNK, device=a.device)
    apart = (t[:, None] - t).clamp(min=0)
    within = (torch.exp(apart * ld[:, None, None]) * (t[:, None] >= t)).float()
    out = torch.matmul(torch.matmul(a, b.transpose(2, 3).contiguous()) * within, c)
    count = there.sum(1)
    left = (count[:, None] - 1 - t).clamp(min=0) + int(decayed)  # decays behind each token in its chunk
    b *= torch.exp(left[:, None] * ld[:, None]).float()[..., None]
    own_part = torch.matmul(b.transpose(2, 3).contiguous(), c)
    before = torch.empty_like(own_part)                           # what is in front of each chunk
    decay = torch.exp(count[:, None] * ld).float()[..., None, None]
    order = torch.argsort(n, descending=True, stable=True)
    state, first = start[order], first[order]
    many = torch.bincount(number)                                 # rows that have a chunk of this number
    for i, m in enumerate(many.tolist()):
        at = first[:m] + i
        before[at] = state[:m]
        state[:m] = state[:m] * decay[at] + own_part[at]
    last[order] = state
    out += torch.matmul(a, before) * torch.exp((t + 1 - int(decayed)) * ld[:, None]).float()[..., None]
    y[index[there]] = out.transpose(1, 2)[there]
    return y, last


def _plain_attend(s):
    case, off = s["case"], s["off"]
    heads, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    lens, rev = off[1:] - off[:-1], case["reverse"]
    shared, scale, dtype = heads // kv, dk ** -0.5, s["q"].dtype
    q = s["q"].detach().float()
    k, v = (s[n].detach().float().repeat_interleave(shared, 1) for n in ("k", "v"))
    h0 = q.new_zeros((lens.numel(), heads, dk, dv)) if s["h0"] is None else s["h0"].detach()
    y, last = _walk(q, k, v, s["decay"], lens, h0, rev, False)
    out = {"y": (y * scale).to(dtype), "last": last}
    if case["train"]:
        del y
        dy, dlast = s["dy"].float() * scale, s["dlast"]
        out["dq"] = _walk(dy, v, k, s["decay"], lens, h0.transpose(2, 3), rev, False)[0].to(dtype)
        # the states' gradients come from the other end; what reaches a row's first token goes on, decayed, to h0
        dv_, dh0 = _walk(k, q, dy, s["decay"], lens, dlast, not rev, True)
        dk_, _ = _walk(v, dy, q, s["decay"], lens, dlast.transpose(2, 3), not rev, True)
        out["dk"] = dk_.view(-1, kv, shared, dk).sum(2).to(dtype)
        out["dv"] = dv_.view(-1, kv, shared, dv).sum(2).to(dtype)
        if s["h0"] is not None:
            out["dh0"] = dh0
    return out


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    shared = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(shared, 1), v.repeat_interleave(shared, 1)
    state = s["state"] * torch.exp(s["decay"])[:, None, None] + k[..., None] * v[:, :, None]
    y = (q[..., None] * state).sum(2) * q.shape[2] ** -0.5
    return y.to(s["q"].dtype), state


def _plain_embed(s):
    w = s["weight"].detach()
    y = (w.float()[s["ids"].long()] * s["scale"]).to(w.dtype)
    if not s["case"]["train"]:
        return y
    grad = torch.zeros(w.shape, dtype=torch.float64, device=w.device)      # (a nucleotide has 100,000 tokens)
    step, few = 1 << 17, w.shape[0] <= 256                        # (few rows: additions to one place would queue)
    for i in range(0, s["ids"].numel(), step):
        ids, dy = s["ids"][i:i + step].long(), s["dy"][i:i + step].double()
        if few:
            grad += (ids == torch.arange(w.shape[0], device=w.device)[:, None]).double() @ dy
        else:
            grad.index_add_(0, ids, dy)
    return y, (grad * s["scale"]).to(w.dtype)


def _plain_beam(s):
    groups, beams = s["scores"].shape
    vocab, width = s["logits"].shape[1], s["case"]["width"]
    z = s["logits"].double()                                      # (neighbours are a millionth apart)
    top = z.amax(1, keepdim=True).clamp(min=-1e300)
    z = z - (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))
    z = z.view(groups, beams, vocab) + s["scores"].double()[:, :, None]
    if s["ended"] is not None:                                    # only their end again, which costs nothing
        z = torch.where(s["ended"][:, :, None], float("-inf"), z)
        z[:, :, 0] = torch.where(s["ended"], s["scores"].double(), z[:, :, 0])
    best, at = torch.sort(z.view(groups, -1), dim=1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    none = torch.isneginf(best)
    token = torch.where(none, -1, at % vocab).to(torch.int32)
    parent = torch.where(none, torch.arange(width, device=at.device) % beams, at // vocab).to(torch.int32)
    from_row = (torch.arange(groups, device=at.device)[:, None] * beams + parent).view(-1)
    return (best.float(), token, parent) + tuple(t[from_row] for t in s["states"])


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from dnatok_amd import lm_ops
        if kind == "step":
            return lm_ops.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"])
        if kind == "attend":
            y, last = lm_ops.linear_attention(s["q"], s["k"], s["v"], s["decay"], s["off"], h0=s["h0"],
                                              reverse=case["reverse"])
            out = {"y": y.detach(), "last": last.detach()}
            if case["train"]:
                wrt = [s["q"], s["k"], s["v"]] + ([] if s["h0"] is None else [s["h0"]])
                out.update(zip(("dq", "dk", "dv", "dh0"), torch.autograd.grad((y, last), wrt, (s["dy"], s["dlast"]))))
            return out
        if kind == "embed":
            y = lm_ops.embedding(s["ids"], s["weight"], scale=s["scale"])
            if not case["train"]:
                return y
            return y.detach(), torch.autograd.grad(y, s["weight"], s["dy"])[0]
        scores, tokens, parents = lm_ops.beam_select(s["logits"], s["scores"], case["width"], finished=s["ended"],
                                                     eos_id=None if s["ended"] is None else 0)
        return (scores, tokens, parents) + tuple(lm_ops.reorder_rows(s["states"], parents))
    with torch.no_grad():
        return {"step": _plain_step, "attend": _plain_attend, "embed": _plain_embed, "beam": _plain_beam}[kind](s)


# ---- the same from the definitions in 64 bits -----------------------------------------------

def _tokens64(a, b, c, decay, off, start, backwards, decayed):
    """The recurrence token by token in 64 bits: pieces of the rows side by side from zero, which gives what each piece adds;
    then all pieces again from the states in front of them."""
    heads, rows, dev = a.shape[1], off.numel() - 1, a.device
    longest = int((off[1:] - off[:-1]).max())
    piece = max(16, int(longest ** 0.5))
    lo, hi, of = [], [], []
    bounds = off.tolist()
    for r in range(rows):
        cuts = list(range(bounds[r], bounds[r + 1], piece))
        cuts = cuts[::-1] if backwards else cuts
        for p in cuts:
            lo.append(p)
            hi.append(min(p + piece, bounds[r + 1]))
            of.append(r)
    lo, hi = torch.tensor(lo, device=dev), torch.tensor(hi, device=dev)
    g = torch.exp(decay.double())[:, None, None]
    y = torch.zeros((a.shape[0], heads, c.shape[2]), dtype=torch.float64, device=dev)

    def through(state, write):
        for i in range(piece):
            here = lo + i < hi
            at = torch.where(here, hi - 1 - i if backwards else lo + i, 0)
            m = here[:, None].double()
            if not decayed:
                state.mul_(torch.where(here[:, None, None, None], g, 1.0))
            state.addcmul_((b[at].double() * m[:, :, None])[..., None], c[at].double()[:, :, None])
            if write:
                seen = torch.matmul(a[at].double()[:, :, None], state)[:, :, 0]
                y[at[here]] = seen[here]
            if decayed:
                state.mul_(torch.where(here[:, None, None, None], g, 1.0))
        return state

    shape = (lo.numel(), heads, b.shape[2], c.shape[2])
    added = through(torch.zeros(shape, dtype=torch.float64, device=dev), False)
    whole = torch.exp(decay.double() * (hi - lo)[:, None])[..., None, None]
    last, front = start.double().clone(), torch.empty_like(added)
    for p, r in enumerate(of):
        front[p] = last[r]
        last[r] = last[r] * whole[p] + added[p]
    del added
    through(front, True)
    return y, last


def _exact_attend(s):
    case, off, rev = s["case"], s["off"], s["case"]["reverse"]
    heads, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    owner = torch.arange(heads, device=off.device) // (heads // kv)
    scale = 1.0 / math.sqrt(dk)
    q, k, v = s["q"].detach(), s["k"].detach()[:, owner], s["v"].detach()[:, owner]
    rows = off.numel() - 1
    h0 = torch.zeros((rows, heads, dk, dv), device=q.device) if s["h0"] is None else s["h0"].detach()
    y, last = _tokens64(q, k, v, s["decay"], off, h0, rev, False)
    out = {"y": y * scale, "last": last}
    if case["train"]:
        dy = s["dy"].double() * scale
        out["dq"] = _tokens64(dy, v, k, s["decay"], off, h0.transpose(2, 3), rev, False)[0]
        each_dv, dh0 = _tokens64(k, q, dy, s["decay"], off, s["dlast"], not rev, True)
        each_dk, _ = _tokens64(v, dy, q, s["decay"], off, s["dlast"].transpose(2, 3), not rev, True)
        for name, each in (("dk", each_dk), ("dv", each_dv)):
            out[name] = torch.stack([each[:, owner == i].sum(1) for i in range(kv)], 1)
        if s["h0"] is not None:
            out["dh0"] = dh0
    return out


def _exact_embed(s):
    w = s["weight"].detach().double()
    y = torch.index_select(w, 0, s["ids"].long()) * s["scale"]
    if not s["case"]["train"]:
        return y
    ids, order = torch.sort(s["ids"].long(), stable=True)
    dim, step = w.shape[1], 64
    grad = torch.zeros_like(w)
    ends = torch.searchsorted(ids, torch.arange(w.shape[0] + 1, device=w.device))
    for c in range(0, dim, step):                                # differences of running sums: 2^-53 of 10^6 terms
        run_sum = torch.zeros((ids.numel() + 1, min(step, dim - c)), dtype=torch.float64, device=w.device)
        torch.cumsum(s["dy"][:, c:c + step][order].double(), 0, out=run_sum[1:])
        grad[:, c:c + step] = run_sum[ends[1:]] - run_sum[ends[:-1]]
    return y, grad * s["scale"]


def _exact_beam(s):
    groups, beams = s["scores"].shape
    vocab, width = s["logits"].shape[1], s["case"]["width"]
    scores, tokens, parents = [], [], []
    for g in range(groups):
        value = torch.log_softmax(s["logits"][g * beams:(g + 1) * beams].double(), 1).nan_to_num(nan=-math.inf)
        value += s["scores"][g].double()[:, None]
        if s["ended"] is not None:
            for b in torch.nonzero(s["ended"][g])[:, 0].tolist():
                value[b] = -math.inf
                value[b, 0] = s["scores"][g, b].double()
        value = value.view(-1)
        # the best ones with all that are equal to the last of them, the lowest places first
        border = torch.topk(value, min(width, value.numel())).values[-1]
        place = torch.nonzero(value >= border)[:, 0].tolist()
        found = sorted(((-v, i) for v, i in zip(value[place].tolist(), place) if v > -math.inf))[:width]
        found += [(math.inf, None)] * (width - len(found))
        scores.append([-v for v, _ in found])
        tokens.append([-1 if i is None else i % vocab for _, i in found])
        parents.append([j % beams if i is None else i // vocab for j, (_, i) in enumerate(found)])
    dev = s["logits"].device
    parent = torch.tensor(parents, device=dev)
    rows = (torch.arange(groups, device=dev)[:, None] * beams + parent).flatten()
    return (torch.tensor(scores, dtype=torch.float64, device=dev), torch.tensor(tokens, dtype=torch.int32, device=dev),
            parent.to(torch.int32)) + tuple(torch.index_select(t, 0, rows) for t in s["states"])


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "step":
            owner = torch.arange(case["heads"], device="cuda") // (case["heads"] // case["kv_heads"])
            q, k, v = s["q"].double(), s["k"].double()[:, owner], s["v"].double()[:, owner]
            state = torch.exp(s["decay"].double()).view(1, -1, 1, 1) * s["state"].double()
            state += k.unsqueeze(3) * v.unsqueeze(2)
            return (q.unsqueeze(2) @ state).squeeze(2) / math.sqrt(case["dk"]), state
        if case["kind"] == "attend":
            return _exact_attend(s)
        return _exact_embed(s) if case["kind"] == "embed" else _exact_beam(s)


def work(case):
    """Each input read once, each output written once."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] in ("step", "attend"):
        h, g, dk, dv = (float(case[n]) for n in ("heads", "kv_heads", "dk", "dv"))
        into, out, state = h * dk + g * (dk + dv), h * dv, 4.0 * h * dk * dv
        if case["kind"] == "step":
            return {"bytes": case["rows"] * (size * (into + out) + 2 * state), "flops": case["rows"] * h * dk * dv * 5}
        rows = float(case["rows"])
        tokens = rows * {"even": case["length"], "reads": 200, "long_reads": 2920}[case["layout"]]
        # (a training step reads y's gradients as well and writes those of the inputs)
        each = 2 * (into + out) if case["train"] else into + out
        ends = rows * state * ((2 if case["start"] else 1) * (2 if case["train"] else 1))
        return {"bytes": tokens * size * each + ends, "flops": tokens * h * dk * dv * (12 if case["train"] else 4)}
    if case["kind"] == "embed":
        n, rows, dim = float(case["tokens"]), float(min(case["tokens"], case["vocab"])), float(case["dim"])
        forward = n * 4 + (n + rows) * dim * size
        back = (n * (dim * size + 4) + case["vocab"] * dim * size) if case["train"] else 0.0
        return {"bytes": forward + back, "flops": n * dim * (2 if case["train"] else 1)}
    rows, out = float(case["groups"] * case["beams"]), float(case["groups"] * case["width"])
    state = 4.0 * (case["dim"] + case["heads"] * 64 * 64)
    moved = out + min(rows, out)
    return {"bytes": rows * case["vocab"] * size + moved * state + 12 * out, "flops": 4.0 * rows * case["vocab"]}
