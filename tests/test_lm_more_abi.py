"""The C entries of linear attention, embeddings and beam search refuse what their kernels cannot take before anything is launched (no
GPU needed), what the compiler made of their kernels, and the plain forms that the GPU's results are compared with."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from dnatok_amd import _lib, build
from tests.support import attention_reference as ref

P = 4096                                # an address that is never looked at
INVALID, TOO_LARGE = -1, -3
HELD = []                               # shapes whose addresses were handed out


def shape(**change):
    fields = dict(dtype=1, reverse=0, n_rows=2, total=128, heads=4, kv_heads=2, dim_k=16, dim_v=24, q_token=64, q_head=16, k_token=32,
                  k_head=16, v_token=48, v_head=24, dy_token=96, dy_head=24, scale=0.25, with_offsets=0)
    assert set(change) <= set(fields)
    HELD.append(_lib.LinearShape(**{**fields, **change}))
    return ctypes.addressof(HELD[-1])


def forward(offsets=None, q=P, work=P, work_bytes=1 << 40, states=None, **change):
    s = shape(**change)
    return _lib.lib().dnatok_linear_attention(s, q, P, P, P, offsets, None, P, P, states, work, work_bytes, None)


def backward(dy=P, work_bytes=1 << 40, states=P, **change):
    s = shape(**change)
    return _lib.lib().dnatok_linear_attention_backward(s, P, P, P, P, None, None, dy, None, states, P, P, P, None, P, work_bytes, None)


def step(**change):
    s = shape(**change)
    return _lib.lib().dnatok_linear_attention_step(s, P, P, P, P, P, P, P, None)


BAD = [dict(dtype=3), dict(dtype=-1), dict(n_rows=-1), dict(total=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(dim_k=0),
       dict(dim_v=-1), dict(scale=0.0), dict(scale=2.0 ** -41), dict(scale=-2.0 ** 41), dict(scale=float("nan")), dict(scale=float("inf")), dict(q_token=-64), dict(k_head=-16),
       dict(v_token=-1), dict(dy_head=-24)]
LARGE = [dict(dim_k=129), dict(dim_v=129), dict(q_token=2 ** 40), dict(k_token=2 ** 31 // 256), dict(v_token=2 ** 62), dict(heads=65536, kv_heads=1),
         dict(dy_token=2 ** 25)]


@pytest.mark.parametrize("call", [forward, backward, step])
def test_attention_refuses(call):
    assert [call(**c) for c in BAD] == [INVALID] * len(BAD)
    assert [call(**c) for c in LARGE] == [TOO_LARGE] * len(LARGE)


def test_attention_refuses_calls_that_do_not_fit():
    assert forward(offsets=P) == INVALID and forward(with_offsets=1) == INVALID        # the shape says otherwise
    assert forward(total=129) == INVALID and forward(n_rows=0) == INVALID              # rows that do not fill the axis; tokens without rows
    assert forward(q=None) == INVALID and backward(dy=None) == INVALID
    cut = dict(n_rows=1, total=1 << 20)
    assert _lib.lib().dnatok_linear_attention_work_bytes(shape(**cut), 0) > 0
    assert forward(work_bytes=16, **cut) == INVALID and forward(work=None, **cut) == INVALID and forward(work=P + 4, **cut) == INVALID
    assert backward(work_bytes=16, **cut) == INVALID and backward(states=None, **cut) == INVALID
    assert forward(n_rows=1 << 24, total=1 << 24) == TOO_LARGE
    single = dict(heads=1, kv_heads=1, n_rows=1 << 23, total=1 << 23)
    assert forward(**single) == TOO_LARGE and backward(**single) == TOO_LARGE          # a grid has less than 2^32 threads
    assert _lib.lib().dnatok_linear_attention(None, P, P, P, P, None, None, P, P, None, P, 0, None) == INVALID
    assert _lib.lib().dnatok_linear_attention_step(shape(n_rows=65536), P, P, P, P, P, P, P, None) == TOO_LARGE
    assert _lib.lib().dnatok_linear_attention_work_bytes(None, 1) == 0


def test_embedding_refuses():
    L, one = _lib.lib(), ctypes.c_float(1.0)
    at = ctypes.addressof(one)
    odd = [ctypes.c_float(float(x)) for x in ("inf", "nan")]

    def rows(ids=P, id_bytes=4, n=8, weight=P, stride=16, dtype=1, vocab=4, dim=16, scale=at, y=P):
        return L.dnatok_embedding(ids, id_bytes, n, weight, stride, dtype, vocab, dim, scale, y, None)

    def grad(ids=P, id_bytes=4, n=8, dy=P, stride=16, dtype=1, vocab=4, dim=16, scale=at, out=P, work=P, work_bytes=1 << 40):
        return L.dnatok_embedding_backward(ids, id_bytes, n, dy, stride, dtype, vocab, dim, scale, out, work, work_bytes, None)

    common = [*(dict(scale=ctypes.addressof(x)) for x in odd), dict(id_bytes=2), dict(n=-1), dict(vocab=-1), dict(dim=-1), dict(stride=-16), dict(dtype=7), dict(ids=None), dict(scale=None)]
    for call, more in ((rows, [dict(weight=None), dict(y=None)]), (grad, [dict(dy=None), dict(out=None), dict(n=500, work_bytes=8),
                                                                          dict(n=500, work=None), dict(n=500, work=P + 8)])):
        assert [call(**c) for c in common + more] == [INVALID] * len(common + more)
        assert [call(**c) for c in (dict(n=2 ** 31), dict(vocab=2 ** 31), dict(dim=2 ** 23))] == [TOO_LARGE] * 3
    assert rows(n=0) == 0 and rows(dim=0) == 0 and grad(vocab=0) == 0 and grad(dim=0) == 0       # nothing to do
    assert L.dnatok_embedding_work_bytes(0, 10, 10) == 0 and L.dnatok_embedding_work_bytes(500, 10, 10) > 0


def test_beam_search_refuses():
    L = _lib.lib()

    def select(logits=P, stride=100, dtype=0, groups=2, beams=3, vocab=100, scores=P, finished=None, eos=0, width=3, out=P, work=P,
               work_bytes=1 << 40):
        return L.dnatok_beam_select(logits, stride, dtype, groups, beams, vocab, scores, finished, eos, width, out, P, P, work, work_bytes, None)

    bad = [dict(dtype=5), dict(groups=-1), dict(beams=0), dict(vocab=0), dict(width=0), dict(stride=-1), dict(logits=None), dict(scores=None),
           dict(out=None), dict(work=None), dict(work_bytes=8), dict(work=P + 8), dict(finished=P, eos=100), dict(finished=P, eos=-1)]
    assert [select(**c) for c in bad] == [INVALID] * len(bad)
    assert [select(**c) for c in (dict(beams=129), dict(width=129), dict(vocab=2 ** 31), dict(groups=2 ** 31), dict(groups=2 ** 26, beams=1))] == [TOO_LARGE] * 5
    assert select(groups=0) == 0
    rows = (ctypes.c_int64 * 5)(P, P, 16, 16, 16)
    at = ctypes.addressof(rows)

    def reorder(tensors=at, n=1, parents=P, groups=2, beams=3, width=3):
        return L.dnatok_reorder_rows(tensors, n, parents, groups, beams, width, None)

    bad = [dict(n=-1), dict(groups=-1), dict(beams=0), dict(width=0), dict(tensors=None), dict(parents=None)]
    assert [reorder(**c) for c in bad] == [INVALID] * len(bad) and reorder(n=0) == 0 and reorder(groups=0) == 0
    for i, value in ((0, 0), (1, 0), (2, -1), (3, -16), (4, -16), (2, 2 ** 40)):
        changed = (ctypes.c_int64 * 5)(*rows)
        changed[i] = value
        assert reorder(tensors=ctypes.addressof(changed)) == INVALID, (i, value)


@pytest.mark.parametrize("src", ["linear_attention.hip", "linear_walk_f32.hip", "linear_walk_bf16.hip", "linear_walk_f16.hip", "embedding.hip",
                                 "beam.hip"])
def test_no_flat_accesses_and_no_packed_32_bit_arithmetic(src, tmp_path):
    hipcc = build.hipcc()
    if not (os.path.isabs(hipcc) and os.path.exists(hipcc)):
        pytest.skip("hipcc not found")
    out = tmp_path / (src + ".s")
    flags = [f for f in build.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.check_call([hipcc, *flags, "-I", build.CSRC, "-S", "--cuda-device-only", "-o", str(out),
                           os.path.join(build.CSRC, src)], stderr=subprocess.DEVNULL)
    code = [line.split(";")[0].strip() for line in out.read_text().splitlines()]
    bad = [c for c in code if re.search(r"\bflat_(load|store|atomic)|\bv_pk_(add|mul|fma)_f32", c)]
    assert not bad, f"{len(bad)}, e.g. {bad[:3]}"
    spilled, kernel = {}, None
    for c in code:
        if m := re.match(r"^(_Z\w+):", c):
            kernel = m.group(1)
        if re.search(r"\bscratch_store_dword", c):
            spilled[kernel] = spilled.get(kernel, 0) + 4 * {"x2": 2, "x3": 3, "x4": 4}.get(c.split()[0][-2:], 1)
    # registers that a kernel keeps in scratch memory: of the 16-bit walks with tiles of 96 and 128 in four waves, where rows end within
    # sixteen bytes most
    most = {"linear_walk_f32.hip": 64, "linear_walk_bf16.hip": 128, "linear_walk_f16.hip": 128}.get(src, 0)
    assert max(spilled.values(), default=0) <= most, spilled


@pytest.mark.parametrize("reverse", [False, True])
def test_the_attention_reference_against_autograd(reverse):
    g = torch.Generator().manual_seed(0)
    q, k, v, h0, dy, dlast = (torch.randn(s, generator=g, dtype=torch.float64) for s in
                              ((20, 4, 5), (20, 2, 5), (20, 2, 3), (3, 4, 5, 3), (20, 4, 3), (3, 4, 5, 3)))
    ld, off = -torch.rand(4, generator=g, dtype=torch.float64), [0, 7, 7, 20]
    leaves = [t.requires_grad_(True) for t in (q, k, v, h0)]
    y, last = [None] * 20, []
    for b in range(3):
        state = h0[b]
        for t in (reversed if reverse else list)(range(off[b], off[b + 1])):
            state = torch.exp(ld)[:, None, None] * state + k[t].repeat_interleave(2, 0)[:, :, None] * v[t].repeat_interleave(2, 0)[:, None]
            y[t] = (q[t][:, :, None] * state).sum(1) * 0.3
        last.append(state)
    grads = torch.autograd.grad((torch.stack(y), torch.stack(last)), leaves, (dy, dlast))
    got = ref.attention(q, k, v, ld, off, h0, 0.3, reverse, dy, dlast)
    for name, want in zip(("y", "last", "dq", "dk", "dv", "dh0"), (torch.stack(y), torch.stack(last), *grads)):
        assert (got[name] - want).abs().max() < 1e-12, name
