"""A small recurrent DNA model from end to end: sequences -> BPE ids -> embeddings -> gated recurrence or linear attention ->
4-bit head -> penalties and a motif's grammar on the logits -> next tokens, the likeliest ones or a beam search, and a training
step of the same model.

    python examples/generate_dna.py --motif ATGNNNNNNNNNTAA --rows 4
    python examples/generate_dna.py --train 20
    python examples/generate_dna.py --mixer linear --beams 4

The weights are random (there is no checkpoint to load); what it shows is how the operators fit together.
"""
import argparse
import json
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from dnatok_amd import bpe_vocab, encoders, lm_ops  # noqa: E402

TOKENIZER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tests", "golden",
                         "bpe4096_tokenizer.json")


class Tokenizer:
    """The BPE encoder of a tokenizer.json, and its tokens' bytes."""

    def __init__(self, path=TOKENIZER):
        with open(path) as fh:
            model = json.load(fh)["model"]
        kernel = bpe_vocab.KernelVocab(bpe_vocab.split_merges(model["merges"]))
        self.encoder = encoders.BpeEncoder(kernel.pair_a, kernel.pair_b, kernel.new_id, len(kernel),
                                           out_remap=kernel.remap_to(model["vocab"], model["vocab"]["[UNK]"]))
        self.tokens = lm_ops.token_bytes(model["vocab"])

    def encode(self, sequences):
        """Packed ids int32 and offsets int64 on the GPU."""
        data, off, lens = encoders.bytes_from_strings(sequences)
        tok, lengths = self.encoder.encode(data, off, int(lens.max()))
        ids, offsets, _ = encoders.pack_ragged(tok, off, lengths)
        return ids[:int(offsets[-1])], offsets

    def decode(self, ids):
        return b"".join(self.tokens[i] or b"" for i in ids).decode("ascii")


class RecurrentLM(torch.nn.Module):
    """Layers of x + out(mixer(in(x))), and a head.  The mixer: a gated recurrence, or linear attention in heads that forget at
    different rates."""

    def __init__(self, vocab, dim=256, layers=2, mixer="gated", heads=4):
        super().__init__()
        self.dim, self.mixer, self.heads = dim, mixer, heads
        self.embed = torch.nn.Parameter(torch.randn(vocab, dim) * 0.5)
        width = 2 * dim if mixer == "gated" else 3 * dim
        self.inner = torch.nn.ParameterList(torch.randn(width, dim) / dim ** 0.5 for _ in range(layers))
        self.outer = torch.nn.ParameterList(torch.randn(dim, dim) / dim ** 0.5 for _ in range(layers))
        self.head = torch.nn.Parameter(torch.randn(vocab, dim) / dim ** 0.5)
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-1.0 - 8.0 * torch.arange(heads) / heads)))

    def in_heads(self, parts):
        """Queries, keys and values [tokens, heads, dim / heads] of a projection's output."""
        return (t.view(t.shape[0], self.heads, -1) for t in parts.split(self.dim, 1))

    def forward(self, ids, offsets):
        """Packed ids -> features [total, dim] in bfloat16 and each layer's states behind the rows."""
        x, states = lm_ops.embedding(ids, self.embed).bfloat16(), []
        for inner, outer in zip(self.inner, self.outer):
            parts = x @ inner.bfloat16().t()
            if self.mixer == "gated":
                y, last = lm_ops.gated_scan(parts[:, :self.dim], parts[:, self.dim:], offsets)
            else:
                y, last = lm_ops.linear_attention(*self.in_heads(parts), self.log_decay, offsets)
                y = y.flatten(1)
            x = x + y @ outer.bfloat16().t()
            states.append(last)
        return x, states


class Generator:
    """The model with 4-bit weights, one token of each row at a time."""

    def __init__(self, model, group=64):
        self.dim, self.embed, self.model = model.dim, model.embed.detach().bfloat16(), model
        self.inner = [lm_ops.W4Matrix.quantize(w, group) for w in model.inner]
        self.outer = [lm_ops.W4Matrix.quantize(w, group) for w in model.outer]
        self.head = lm_ops.W4Matrix.quantize(model.head, group)

    def step(self, token, states):
        """Features of one new token of each row; the states move on."""
        x = lm_ops.embedding(token, self.embed)
        for inner, outer, state in zip(self.inner, self.outer, states):
            parts = inner.matvec(x)
            if self.model.mixer == "gated":
                y, _ = lm_ops.gated_step(parts[:, :self.dim], parts[:, self.dim:], state, out_state=state)
            else:
                y, _ = lm_ops.linear_attention_step(*self.model.in_heads(parts), self.model.log_decay, state, out_state=state)
                y = y.flatten(1)
            x = x + outer.matvec(y)
        return x

    def last_features(self, model, ids, offsets):
        """The last token's features of each row, zeros for an empty one, and the states."""
        x, states = model(ids, offsets)
        return torch.cat([x.new_zeros((1, self.dim)), x])[torch.where(offsets[1:] > offsets[:-1], offsets[1:], 0)], states

    @torch.no_grad()
    def search(self, model, ids, offsets, steps, beams, grammar=None):
        """The ``beams`` likeliest continuations of each row, as far as the grammar allows any: int32 [B, beams, steps] (-1 behind
        their end) and their log probabilities float32 [B, beams], the best first.  A beam has ended where the grammar lets nothing
        follow any more."""
        rows = offsets.numel() - 1
        x, states = self.last_features(model, ids, offsets)
        scores = torch.zeros((rows, 1), device=ids.device)
        chosen = torch.empty((rows, 0), dtype=torch.int32, device=ids.device)
        state = torch.zeros(rows, dtype=torch.int32, device=ids.device)
        ended = torch.zeros(rows, dtype=torch.bool, device=ids.device)
        # (and of the state behind the last one, of rows that took a forbidden token: those have not ended, they are none)
        over = torch.nn.functional.pad((grammar.allowed == 0).all(1), (0, 1)) if grammar else None
        for _ in range(steps):
            logits = self.head.matvec(x, out_dtype=torch.float32)
            if grammar:
                lm_ops.process_logits(logits, allowed=grammar.allowed, state=state, out=logits)
            scores, token, parent = lm_ops.beam_select(logits, scores, beams, finished=ended.view(rows, -1), eos_id=0)
            chosen, state, ended, *states = lm_ops.reorder_rows([chosen, state, ended, *states], parent)
            token = torch.where(ended, -1, token.view(-1))
            chosen = torch.cat([chosen, token[:, None]], 1)
            if grammar:
                state = torch.where(ended, state, grammar.advance(state, token))
                ended = over[state.long()]
            x = self.step(token, states)
        return chosen.view(rows, -1, steps), scores

    @torch.no_grad()
    def generate(self, model, ids, offsets, steps, grammar=None, *, repetition=1.2, presence=0.1, frequency=0.05):
        """int32 [B, steps]: the likeliest allowed token each time; -1 once nothing is allowed."""
        rows = offsets.numel() - 1
        lengths = offsets[1:] - offsets[:-1]
        width = int(lengths.max()) + steps
        # each row's history has room to grow: ids of -1 count for nothing
        history = torch.full((rows, width), -1, dtype=torch.int32, device=ids.device)
        at = torch.arange(int(lengths.max()), device=ids.device)
        there = at[None, :] < lengths[:, None]
        history[:, :at.numel()][there] = ids
        room = torch.arange(rows + 1, device=ids.device) * width
        penalties = [torch.full((rows,), v, device=ids.device) for v in (repetition, presence, frequency)]
        x, states = self.last_features(model, ids, offsets)
        state = torch.zeros(rows, dtype=torch.int32, device=ids.device) if grammar else None
        out = []
        for i in range(steps):
            logits = self.head.matvec(x, out_dtype=torch.float32)
            lm_ops.process_logits(logits, history=history.view(-1), history_offsets=room,
                                  prompt_lengths=lengths.to(torch.int32), repetition=penalties[0], presence=penalties[1],
                                  frequency=penalties[2], allowed=grammar.allowed if grammar else None, state=state,
                                  out=logits)
            best, token = logits.max(1)
            token = torch.where(torch.isneginf(best), -1, token).to(torch.int32)
            out.append(token)
            history.scatter_(1, (lengths + i)[:, None], token[:, None])
            if grammar:
                state = torch.where(token < 0, state, grammar.advance(state, token.clamp(min=0)))
            x = self.step(token.clamp(min=0), states)
        return torch.stack(out, 1)


def train(model, ids, offsets, steps, lr=0.05):
    """Next-token prediction on the rows; the losses."""
    optimizer = torch.optim.SGD(model.parameters(), lr=lr)
    follows = torch.ones(ids.numel(), dtype=torch.bool, device=ids.device)
    follows[(offsets[1:] - 1)[offsets[1:] > offsets[:-1]]] = False     # (a row's last token has no successor)
    losses = []
    for _ in range(steps):
        x, _ = model(ids, offsets)
        logits = (x @ model.head.bfloat16().t()).float()
        loss = torch.nn.functional.cross_entropy(logits[:-1][follows[:-1]], ids[1:][follows[:-1]].long())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--motif", default="ATGNNNNNNNNNNNNTAA", help="what is generated spells this (IUPAC letters)")
    p.add_argument("--rows", type=int, default=4)
    p.add_argument("--train", type=int, default=0, help="training steps on the prompts first")
    p.add_argument("--mixer", choices=["gated", "linear"], default="gated", help="what the layers mix tokens with")
    p.add_argument("--beams", type=int, default=0, help="continuations to search over instead of taking the likeliest token")
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    torch.manual_seed(a.seed)
    gen = torch.Generator().manual_seed(a.seed)
    tok = Tokenizer()
    prompts = ["".join("ACGT"[i] for i in torch.randint(0, 4, (200 + 37 * r,), generator=gen)) for r in range(a.rows)]
    ids, offsets = tok.encode(prompts)
    model = RecurrentLM(len(tok.tokens), mixer=a.mixer).cuda()
    losses = train(model, ids, offsets, a.train)
    if losses:
        print("loss %.3f -> %.3f" % (losses[0], losses[-1]))
    grammar = lm_ops.TokenGrammar.from_iupac(a.motif, tok.tokens)
    if a.beams:
        chosen = Generator(model).search(model, ids, offsets, len(a.motif), a.beams, grammar)[0].flatten(0, 1).cpu().tolist()
    else:
        chosen = Generator(model).generate(model, ids, offsets, len(a.motif), grammar).cpu().tolist()
    sequences = [tok.decode(i for i in row if i >= 0) for row in chosen]
    for s in sequences:
        print(s)
    return losses, sequences


if __name__ == "__main__":
    main()
