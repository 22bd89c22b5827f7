"""What the model operators are timed on: the calls that a program makes through ``lm_ops`` once the
tokens are there, over the sizes that such programs bring.

Kinds of case, and what each stands for:

scan    the gated linear recurrence over packed rows of base embeddings: windows, one contig, reads of
        mixed lengths; forward, or forward and backward in a training step.  Values and gates come as
        the two halves of one projection's output, as a layer has them
step    the same recurrence for one new token of each row
w4      a projection or a vocabulary's head with 4-bit weights, for one token of each row
logits  penalties for repeated tokens, biases and a grammar's mask on the head's output

``run`` computes them in elementary torch operations in 32 bits, or, with ``own`` set, with the
framework's operators.
"""
import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # generation for one sequence: one token through one layer, a call that is all latency
        {"name": "step_1x512", "kind": "step", "rows": 1, "dim": 512, "dtype": "bfloat16"},
        # generation for many sequences at once
        {"name": "step_1000x1024", "kind": "step", "rows": 1000, "dim": 1024, "dtype": "float16"},
        # a batch of windows of single nucleotides, forward only (scoring)
        {"name": "scan_64x8192_d512", "kind": "scan", "layout": "even", "rows": 64, "length": 8192, "dim": 512,
         "dtype": "bfloat16", "reverse": False, "start": False, "train": False},
        # one contig, read from its end, continued from a state
        {"name": "scan_1x1000003_d256", "kind": "scan", "layout": "even", "rows": 1, "length": 1000003, "dim": 256,
         "dtype": "bfloat16", "reverse": True, "start": True, "train": False},
        # a training step on windows of tokens
        {"name": "train_256x1024_d512", "kind": "scan", "layout": "even", "rows": 256, "length": 1024, "dim": 512,
         "dtype": "bfloat16", "reverse": False, "start": False, "train": True},
        # a training step in 32 bits on long reads of mixed lengths, an odd number of channels
        {"name": "train_300_reads_d203", "kind": "scan", "layout": "long_reads", "rows": 300, "length": 2000, "dim": 203,
         "dtype": "float32", "reverse": True, "start": True, "train": True},
        # a small projection for one sequence: latency
        {"name": "w4_1x4096x1024", "kind": "w4", "m": 1, "n": 4096, "k": 1024, "group": 128, "dtype": "bfloat16",
         "zeros": False, "out": "float32"},
        # the head of a wide model over the larger vocabulary, one sequence: the rate at which weights arrive
        {"name": "w4_1x32000x4096", "kind": "w4", "m": 1, "n": 32000, "k": 4096, "group": 64, "dtype": "bfloat16",
         "zeros": False, "out": "float32"},
        # a projection for a batch of sequences, small groups with zero points
        {"name": "w4_16x8192x8192", "kind": "w4", "m": 16, "n": 8192, "k": 8192, "group": 32, "dtype": "float16",
         "zeros": True, "out": "same"},
        # the largest batch, sizes that fit no tile
        {"name": "w4_61x12301x2040", "kind": "w4", "m": 61, "n": 12301, "k": 2040, "group": 128, "dtype": "bfloat16",
         "zeros": True, "out": "same"},
        # one sequence of the smaller vocabulary
        {"name": "logits_1x4096", "kind": "logits", "rows": 1, "vocab": 4096, "history": 1000, "dtype": "float32",
         "bias": False, "states": 16},
        # a batch over the larger vocabulary with histories of mixed lengths, everything on
        {"name": "logits_256x32000", "kind": "logits", "rows": 256, "vocab": 32000, "history": 8000, "dtype": "bfloat16",
         "bias": True, "states": 300},
    ]


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "scan", "w4", "w4", "logits"])
    case = {"kind": kind}
    if kind == "step":
        case.update(rows=_between(rng, 1, 1000), dim=_between(rng, 16, 1024), dtype=rng.choice(sorted(TYPES)))
    elif kind == "scan":
        layout = rng.choice(["even", "reads", "long_reads"])
        dim = _between(rng, 16, 1024) if rng.random() < 0.4 else rng.choice([64, 128, 256, 512, 768, 1024])
        dtype, train = rng.choice(sorted(TYPES)), rng.random() < 0.5
        most = (100000000 if train else 250000000) // (2 if dtype == "float32" else 1) // dim
        if layout == "even":
            length = _between(rng, 1, most)
            rows = _between(rng, 1, max(1, most // length))
        elif layout == "reads":
            length, rows = 200, _between(rng, 1, min(100000, most // 300))
        else:
            length, rows = 2000, _between(rng, 1, max(1, most // 4000))
        case.update(layout=layout, rows=rows, length=length, dim=dim, dtype=dtype, reverse=rng.random() < 0.5,
                    start=rng.random() < 0.5, train=train)
    elif kind == "w4":
        m, k = _between(rng, 1, 64), _between(rng, 64, 8192)
        if rng.random() < 0.6:
            k = max(128, k - k % 128)
        case.update(m=m, n=_between(rng, 16, min(32000, 67000000 // k)), k=k, group=rng.choice([32, 64, 128]),
                    dtype=rng.choice(["bfloat16", "float16"]), zeros=rng.random() < 0.5,
                    out=rng.choice(["same", "float32"]))
    else:
        rows = _between(rng, 1, 256)
        case.update(rows=rows, vocab=rng.choice([4096, 32000, _between(rng, 16, 32000)]),
                    history=_between(rng, 1, min(100000, 2048000 // rows)), dtype=rng.choice(sorted(TYPES)),
                    bias=rng.random() < 0.5, states=rng.choice([0, 16, 300]))
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


def _projection(total, dim, dtype, gen):
    """Values around zero and gate logits whose channels forget within one to a few thousand tokens."""
    both = torch.empty((total, 2 * dim), dtype=dtype, device="cuda").normal_(generator=gen)
    both[:, dim:] += torch.linspace(-1.0, 8.0, dim, device="cuda").to(dtype)
    return both[:, :dim], both[:, dim:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}

    def normal(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)

    if case["kind"] == "step":
        x, gate = _projection(case["rows"], case["dim"], TYPES[case["dtype"]], gen)
        s.update(x=x, gate=gate, state=normal(case["rows"], case["dim"]))
    elif case["kind"] == "scan":
        dtype, rows, dim = TYPES[case["dtype"]], case["rows"], case["dim"]
        off = _offsets(_lengths(case, gen))
        total = int(off[-1])
        x, gate = _projection(total, dim, dtype, gen)
        h0 = normal(rows, dim) if case["start"] else None
        s.update(x=x, gate=gate, off=off, h0=h0)
        if case["train"]:
            s.update(dy=normal(total, dim, dtype=dtype), dlast=normal(rows, dim))
            for t in (x, gate) if h0 is None else (x, gate, h0):
                t.requires_grad_(True)
    elif case["kind"] == "w4":
        m, n, k, dtype = case["m"], case["n"], case["k"], TYPES[case["dtype"]]
        words, groups = -(-k // 8), -(-k // case["group"])
        q = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
        scales = (0.002 + 0.004 * torch.rand((n, groups), generator=gen, device="cuda")).to(dtype)
        zeros = None
        if case["zeros"]:
            zeros = torch.randint(5, 11, (n, groups), generator=gen, device="cuda", dtype=torch.uint8)
        s.update(q=q, scales=scales, zeros=zeros, x=normal(m, k, dtype=dtype), bias=normal(n))
        if own:
            from dnatok_amd import lm_ops
            s["matrix"] = lm_ops.W4Matrix(q, scales, zeros, in_features=k, group=case["group"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        mean = case["history"]                                   # from none to twice the mean
        lens = _in_any_order(torch.arange(rows, device="cuda") * 2 * mean // max(rows - 1, 1), gen) if rows > 1 else \
            torch.full((1,), mean, dtype=torch.int64, device="cuda")
        off = _offsets(lens)
        u = torch.rand(int(off[-1]), generator=gen, device="cuda")
        s.update(logits=(3.0 * normal(rows, vocab)).to(TYPES[case["dtype"]]), off=off,
                 history=(u * u * vocab).to(torch.int32).clamp(max=vocab - 1),        # some tokens come often
                 prompt=(lens // 2).to(torch.int32),
                 repetition=1.0 + 0.5 * torch.rand(rows, generator=gen, device="cuda"),
                 presence=torch.rand(rows, generator=gen, device="cuda"),
                 frequency=0.1 * torch.rand(rows, generator=gen, device="cuda"),
                 bias=normal(vocab) if case["bias"] else None, allowed=None, state=None)
        if case["states"]:
            bits = torch.randint(-2 ** 31, 2 ** 31, (2, case["states"], -(-vocab // 32)), generator=gen, device="cuda",
                                 dtype=torch.int64).to(torch.int32)
            s["allowed"] = bits[0] & bits[1]                     # a quarter of the tokens may come next
            s["state"] = torch.randint(-1, case["states"], (rows,), generator=gen, device="cuda", dtype=torch.int32)
    return s


# ---- the operators --------------------------------------------------------------------------

def _row_starts(off, total):
    """Of the rows that are not empty: first token, number, last token."""
    nonempty = off[1:] > off[:-1]
    at = off[:-1][nonempty]
    row = torch.arange(off.numel() - 1, device=off.device)[nonempty]
    return at, row, off[1:][nonempty] - 1


def _doubling(a, h, longest):
    """h_t += a_t h_(t-1) along the first axis, by steps of 1, 2, 4 ... tokens (a is zero where a row starts)."""
    s = 1
    while s < longest:
        nh = h.clone()
        nh[s:].addcmul_(a[s:], h[:-s])
        na = a.clone()
        na[s:] *= a[:-s]
        na[:s] = 0
        h, a, s = nh, na, 2 * s
    return h


def _plain_scan(s):
    case, off = s["case"], s["off"]
    x, gate = s["x"].detach().float(), s["gate"].detach().float()
    total, dim = x.shape
    rev, h0 = case["reverse"], s["h0"]
    first, row, end = _row_starts(off, total)
    if rev:
        first, end = end, first
    longest = int((off[1:] - off[:-1]).max()) if case["layout"] != "even" else case["length"]
    f = 1.0 / (1.0 + torch.exp(-gate))
    u = x / (1.0 + torch.exp(gate))                              # (1 - f) x
    if h0 is not None:
        u[first] += f[first] * h0.detach()[row]
    a = f.clone()
    a[first] = 0
    h = _doubling(a.flip(0), u.flip(0), longest).flip(0) if rev else _doubling(a, u, longest)
    del u, a
    last = torch.zeros((off.numel() - 1, dim), device=x.device) if h0 is None else h0.detach().clone()
    last[row] = h[end]
    out = {"y": h.to(s["x"].dtype), "last": last}
    if case["train"]:
        dh = s["dy"].to(torch.float32, copy=True)
        dh[end] += s["dlast"][row]
        nxt = torch.zeros_like(f)                                # the factor between a token and the one after it
        if rev:
            nxt[1:] = f[:-1]
        else:
            nxt[:-1] = f[1:]
        nxt[end] = 0
        dh = _doubling(nxt, dh, longest) if rev else _doubling(nxt.flip(0), dh.flip(0), longest).flip(0)
        del nxt
        before = torch.zeros_like(h)
        if rev:
            before[:-1] = h[1:]
        else:
            before[1:] = h[:-1]
        before[first] = 0 if h0 is None else h0.detach()[row]
        out["dx"] = ((1.0 - f) * dh).to(s["x"].dtype)
        out["dgate"] = (dh * (before - x) * f * (1.0 - f)).to(s["x"].dtype)
        if h0 is not None:
            dh0 = s["dlast"].clone()
            dh0[row] = f[first] * dh[first]
            out["dh0"] = dh0
    return out


def _unpacked(q, k):
    """[N, words] of eight 4-bit values -> [N, K], whole numbers in 32 bits."""
    shift = torch.arange(0, 32, 4, device=q.device, dtype=torch.int32)
    return ((q[:, :, None] >> shift) & 15).reshape(q.shape[0], -1)[:, :k]


def _plain_w4(s):
    case = s["case"]
    k, group = case["k"], case["group"]
    w = _unpacked(s["q"], k).float()
    z = torch.full_like(s["scales"], 8.0, dtype=torch.float32) if s["zeros"] is None else s["zeros"].float()
    w -= z.repeat_interleave(group, 1)[:, :k]
    w *= s["scales"].float().repeat_interleave(group, 1)[:, :k]
    y = s["x"].float() @ w.t() + s["bias"]
    return y if case["out"] == "float32" else y.to(s["x"].dtype)


def _plain_logits(s):
    rows, vocab = s["logits"].shape
    lens = s["off"][1:] - s["off"][:-1]
    row = torch.repeat_interleave(torch.arange(rows, device="cuda"), lens)
    cell = row * vocab + s["history"].long()
    generated = torch.arange(cell.numel(), device="cuda") - s["off"][row] >= s["prompt"][row]
    seen = torch.zeros(rows * vocab, device="cuda").index_fill_(0, cell, 1.0).view(rows, vocab) > 0
    count = torch.zeros(rows * vocab, device="cuda").scatter_add_(0, cell, generated.float()).view(rows, vocab)
    z = s["logits"].float()
    r = s["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - s["presence"][:, None] * (count > 0) - s["frequency"][:, None] * count
    if s["bias"] is not None:
        z = z + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(vocab, device="cuda")
        ok = (s["allowed"][s["state"].clamp(min=0).long()][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        z = torch.where((ok == 1) | (s["state"] < 0)[:, None], z, float("-inf"))
    return z.to(s["logits"].dtype)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from dnatok_amd import lm_ops
        if kind == "step":
            return lm_ops.gated_step(s["x"], s["gate"], s["state"])
        if kind == "scan":
            y, last = lm_ops.gated_scan(s["x"], s["gate"], s["off"], h0=s["h0"], reverse=case["reverse"])
            out = {"y": y.detach(), "last": last.detach()}
            if case["train"]:
                wrt = [s["x"], s["gate"]] + ([] if s["h0"] is None else [s["h0"]])
                out.update(zip(("dx", "dgate", "dh0"), torch.autograd.grad((y, last), wrt, (s["dy"], s["dlast"]))))
            return out
        if kind == "w4":
            return s["matrix"].matvec(s["x"], bias=s["bias"], out_dtype=torch.float32 if case["out"] == "float32" else None)
        return lm_ops.process_logits(s["logits"], history=s["history"], history_offsets=s["off"],
                                     prompt_lengths=s["prompt"], repetition=s["repetition"], presence=s["presence"],
                                     frequency=s["frequency"], bias=s["bias"], allowed=s["allowed"], state=s["state"])
    if kind == "step":
        gate = s["gate"].float()
        h = s["state"] / (1.0 + torch.exp(-gate)) + s["x"].float() / (1.0 + torch.exp(gate))
        return h.to(s["x"].dtype), h
    if kind == "scan":
        with torch.no_grad():
            return _plain_scan(s)
    return _plain_w4(s) if kind == "w4" else _plain_logits(s)


# ---- the same from the definitions in 64 bits -----------------------------------------------

def _recurrence64(a, u):
    """h_t = a_t h_(t-1) + u_t token by token: pieces of the axis side by side from zero, then from the state
    that the piece before them ends in."""
    total, dim = a.shape
    piece = max(1, int(total ** 0.5))
    n = -(-total // piece)
    pad = n * piece - total
    if pad:
        a = torch.cat([a, a.new_zeros((pad, dim))])
        u = torch.cat([u, u.new_zeros((pad, dim))])
    a, u = a.view(n, piece, dim), u.view(n, piece, dim)
    decay, state = a.new_ones((n, dim)), u.new_zeros((n, dim))
    for i in range(piece):
        state = a[:, i] * state + u[:, i]
        decay = decay * a[:, i]
    carry = torch.zeros_like(state)
    for j in range(1, n):
        carry[j] = decay[j - 1] * carry[j - 1] + state[j - 1]
    h = torch.empty_like(u)
    for i in range(piece):
        carry = a[:, i] * carry + u[:, i]
        h[:, i] = carry
    return h.view(n * piece, dim)[:total]


def _exact_scan(s):
    case = s["case"]
    turn = (lambda t: t.flip(0)) if case["reverse"] else (lambda t: t)
    x, g = turn(s["x"].detach().double()), turn(s["gate"].detach().double())
    total, dim = x.shape
    lens = turn(s["off"][1:] - s["off"][:-1])
    ends = torch.cumsum(lens, 0)
    starts = ends - lens
    has = lens > 0
    f, keep = torch.sigmoid(g), torch.sigmoid(-g)
    first, end = starts[has], ends[has] - 1
    h0 = x.new_zeros((lens.numel(), dim)) if s["h0"] is None else turn(s["h0"].detach().double())
    a, u = f.clone(), keep * x
    u[first] += f[first] * h0[has]
    a[first] = 0
    h = _recurrence64(a, u)
    last = h0.clone()
    last[has] = h[end]
    out = {"y": turn(h), "last": turn(last)}
    if case["train"]:
        del a, u
        dlast = turn(s["dlast"].double())
        dy = turn(s["dy"].double()).clone()
        dy[end] += dlast[has]
        nxt = torch.roll(f, -1, 0)
        nxt[end] = 0
        dh = _recurrence64(nxt.flip(0), dy.flip(0)).flip(0)
        before = torch.roll(h, 1, 0)
        before[first] = h0[has]
        out["dx"] = turn(keep * dh)
        out["dgate"] = turn(dh * (before - x) * f * keep)
        if s["h0"] is not None:
            dh0 = dlast.clone()
            dh0[has] = f[first] * dh[first]
            out["dh0"] = turn(dh0)
    return out


def _exact_logits(s):
    rows, vocab = s["logits"].shape
    z = s["logits"].double()
    off, prompt = s["off"].tolist(), s["prompt"].tolist()
    for r in range(rows):
        ids = s["history"][off[r]:off[r + 1]].long()
        in_all = torch.bincount(ids, minlength=vocab)
        c = torch.bincount(ids[prompt[r]:], minlength=vocab).double()
        rep = s["repetition"][r].double()
        z[r] = torch.where(in_all == 0, z[r], torch.where(z[r] > 0, z[r] / rep, z[r] * rep))
        z[r] -= s["presence"][r].double() * (c > 0) + s["frequency"][r].double() * c
    if s["bias"] is not None:
        z += s["bias"].double()
    if s["allowed"] is not None:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        ok = ((s["allowed"][:, :, None] >> bit) & 1).reshape(s["allowed"].shape[0], -1)[:, :vocab].bool()
        for r, st in enumerate(s["state"].tolist()):
            if st >= 0:
                z[r][~ok[st]] = float("-inf")
    return z


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "step":
            g = s["gate"].double()
            h = torch.sigmoid(g) * s["state"].double() + torch.sigmoid(-g) * s["x"].double()
            return h, h.clone()
        if case["kind"] == "scan":
            return _exact_scan(s)
        if case["kind"] == "w4":
            k, group = case["k"], case["group"]
            of = torch.arange(k, device="cuda") // group
            w = torch.stack([(s["q"] >> (4 * i)) & 15 for i in range(8)], 2).flatten(1)[:, :k].double()
            w = (w - (8.0 if s["zeros"] is None else s["zeros"].double()[:, of])) * s["scales"].double()[:, of]
            return s["x"].double() @ w.t().contiguous() + s["bias"].double()
        return _exact_logits(s)


def work(case):
    """Each input read once, each output written once."""
    size = 4 if case.get("dtype") == "float32" else 2
    if case["kind"] == "step":
        cells = float(case["rows"]) * case["dim"]
        return {"bytes": cells * (3 * size + 8), "flops": 10.0 * cells}
    if case["kind"] == "scan":
        mean = {"even": case["length"], "reads": 200, "long_reads": 2920}[case["layout"]]
        cells = float(case["rows"]) * mean * case["dim"]
        ends = 4.0 * case["rows"] * case["dim"] * ((2 if case["start"] else 1) * (2 if case["train"] else 1))
        # (a training step reads the outputs' gradients as well and writes those of values and gates)
        return {"bytes": cells * size * (6 if case["train"] else 3) + ends + 8.0 * case["rows"],
                "flops": cells * (35 if case["train"] else 10)}
    if case["kind"] == "w4":
        m, n, k = float(case["m"]), float(case["n"]), float(case["k"])
        groups = -(-case["k"] // case["group"])
        return {"bytes": n * k / 2 + n * groups * (3 if case["zeros"] else 2) + 2 * m * k + 4 * n +
                m * n * (4 if case["out"] == "float32" else 2), "flops": 2.0 * m * n * k}
    rows, vocab = float(case["rows"]), float(case["vocab"])
    masks = min(rows, case["states"]) * vocab / 8
    return {"bytes": rows * vocab * 2 * size + 4.0 * rows * case["history"] + masks + (4 * vocab if case["bias"] else 0),
            "flops": 6.0 * rows * vocab}
