"""The 64-bit restatements that the model operators are tested against, against differences and closed forms;
and what the wrappers refuse without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

from dnatok_amd import _lib, lm_ops
from tests.support import lm_reference as ref


@pytest.mark.parametrize("reverse", [False, True])
def test_gradient_of_the_recurrence_against_differences(reverse):
    rng = np.random.default_rng(1)
    off = np.array([0, 5, 5, 12, 13])
    x, g, dy = (rng.standard_normal((13, 3)) for _ in range(3))
    h0, dlast = rng.standard_normal((4, 3)), rng.standard_normal((4, 3))

    def value(x, g, h0):
        y, last = ref.scan(x, g, off, h0, reverse)
        return (y * dy).sum() + (last * dlast).sum()

    grads = ref.scan_grad(x, g, off, dy, dlast, h0, reverse)[:3]
    args, eps = [x, g, h0], 1e-5
    for i, grad in enumerate(grads):
        for at in np.ndindex(grad.shape):
            shifted = [[a.copy() for a in args] for _ in range(2)]
            shifted[0][i][at] += eps
            shifted[1][i][at] -= eps
            diff = (value(*shifted[0]) - value(*shifted[1])) / (2 * eps)
            assert abs(diff - grad[at]) <= 1e-8                      # (eps^2 and 1e-16 / eps, times values of a few units)


def test_recurrence_closed_form():
    """A constant gate: geometric weights."""
    x = np.arange(1.0, 7.0)[:, None]
    y, last = ref.scan(x, np.zeros((6, 1)), np.array([0, 6]), np.array([[8.0]]))
    want = 8.0 * 0.5 ** 6 + sum(0.5 * 0.5 ** (6 - t) * t for t in range(1, 7))
    assert abs(last[0, 0] - want) < 1e-12 and y[5, 0] == last[0, 0]
    back, blast = ref.scan(x[::-1], np.zeros((6, 1)), np.array([0, 6]), np.array([[8.0]]), reverse=True)
    np.testing.assert_allclose(back[::-1], y)


def test_products_and_logits_by_hand():
    q = np.array([[0x76543210, -1]], dtype=np.int64).astype(np.int32)
    assert list(ref.unpack4(q, 10)[0]) == [0, 1, 2, 3, 4, 5, 6, 7, 15, 15]
    y = ref.w4(np.ones((1, 10)), q, np.array([[2.0]]), None, 10, 32)
    assert y[0, 0] == 2.0 * (sum(range(8)) - 64 + 2 * 7)
    z = ref.logits(np.array([[2.0, -2.0, 1.0, 0.0]]), np.array([0, 1, 1, 3, 9]), [0, 5], [1], [2.0], [0.5], [0.25], None,
                   np.array([[0b0111]]), np.array([0]))
    assert list(z[0]) == [1.0, -4.0 - 0.5 - 0.5, 1.0, -np.inf]


def test_argument_errors_without_a_gpu():
    L = _lib.lib()
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)
    scan = lambda dtype=0, rows=1, total=4, dim=4, x=p, off=p: L.dnatok_gated_scan(
        x, 4, p, 4, dtype, off, rows, total, dim, 0, None, p, None, None, None, 0, None)
    for kw, text in (({"dtype": 3}, b"type"), ({"dim": 0}, b"size"), ({"rows": -1}, b"size"), ({"rows": 0}, b"size"),
                     ({"x": None}, b"null"), ({"rows": 3, "off": None}, b"one length")):
        assert scan(**kw) == -1 and text in L.dnatok_last_error(), kw
    assert L.dnatok_gated_scan_backward(None, 4, p, 4, 0, p, 1, 4, 4, 0, None, p, 4, None, p, p, p, None, None, 0, None) == -1
    assert L.dnatok_gated_scan_backward(p, 4, p, 4, 0, p, 1, 1 << 20, 4, 0, None, p, 4, None, p, p, p, None, p, 64, None) == -4
    assert scan(total=1 << 20) == -4 and b"bytes" in L.dnatok_last_error()
    assert L.dnatok_gated_step(p, 4, p, 4, 0, None, 1, 4, None, p, None) == -1 and b"null" in L.dnatok_last_error()
    w4 = lambda dtype=1, stride=8, group=32, y=1, x=p, k=64: L.dnatok_w4_matvec(
        x, 64, dtype, p, stride, p, None, 1, 4, k, group, None, p, 4, y, None)
    for kw, text in (({"dtype": 0}, b"bfloat16"), ({"stride": 7}, b"overlap"), ({"group": 40}, b"32"), ({"group": 0}, b"32"),
                     ({"y": 2}, b"type"), ({"x": None}, b"null"), ({"k": 0}, b"size")):
        assert w4(**kw) == -1 and text in L.dnatok_last_error(), kw
    logits = lambda dtype=0, out=0, z=p, off=None, hist=None, allowed=None, stride=1, states=0, state=None: L.dnatok_logits_process(
        z, 8, dtype, 2, 8, hist, off, None, None, None, None, None, 0, allowed, stride, states, state, p, 8, out, None)
    for kw, text in (({"dtype": 5}, b"type"), ({"out": 1}, b"type"), ({"z": None}, b"null"), ({"hist": p}, b"offsets"),
                     ({"allowed": p, "states": 0}, b"mask"), ({"allowed": p, "states": 1, "stride": 0}, b"mask"),
                     ({"allowed": p, "states": 3}, b"one"), ({"state": p}, b"masks")):
        assert logits(**kw) == -1 and text in L.dnatok_last_error(), kw


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu():
    x = torch.randn(4, 8)
    with pytest.raises(ValueError, match="GPU"):
        lm_ops.gated_scan(x, x, torch.tensor([0, 4]))
    with pytest.raises(ValueError, match="GPU"):
        lm_ops.gated_step(x, x)
    with pytest.raises(ValueError, match="GPU"):
        lm_ops.W4Matrix(torch.zeros((4, 1), dtype=torch.int32), torch.ones(4, 1).bfloat16(), in_features=8, group=32)
    with pytest.raises(ValueError, match="GPU"):
        lm_ops.process_logits(x)


def test_token_grammar_by_hand():
    tokens = [b"A", b"C", b"G", b"T", b"AC", b"GT", b"ACG", None, b"TTT"]
    g = lm_ops.TokenGrammar.from_iupac("ANG", tokens, eos_id=7, device="cpu")
    assert g.n_states == 4 and g.allowed.shape == (4, 1) and g.next_state.shape == (5, 9)
    bits = lambda s: [v for v in range(9) if int(g.allowed[s, 0]) >> v & 1]
    assert bits(0) == [0, 4, 6] and bits(1) == [0, 1, 2, 3] and bits(2) == [2] and bits(3) == [7]
    # (state 1 allows CG, none of the tokens; GT has T where G must be)
    assert g.next_state[0].tolist() == [1, 4, 4, 4, 2, 4, 3, 4, 4]
    assert g.next_state[4].tolist() == [4] * 9                          # a row that took what was forbidden
    state = g.advance(torch.tensor([0, 0, -1, 4, 3], dtype=torch.int32), torch.tensor([4, 8, 3, 0, 7]))
    assert state.tolist() == [2, 4, -1, 4, 3]
    again = lm_ops.TokenGrammar.from_iupac("AY", tokens, repeat=True, device="cpu")
    assert again.n_states == 2 and again.next_state[0, 4] == 0 and again.next_state[0, 6] == 2


@pytest.mark.parametrize("vocab", [31, 32, 33, 200])
def test_token_grammar_against_following_every_byte(vocab):
    rng = np.random.default_rng(vocab)
    tokens = [None if rng.random() < 0.1 else bytes(rng.choice(list(b"ACGT"), rng.integers(1, 6))) for _ in range(vocab)]
    trans = np.full((6, 256), -1)
    trans[:, list(b"ACGT")] = rng.integers(-1, 6, (6, 4))
    g = lm_ops.TokenGrammar(trans, tokens, device="cpu")
    for s in range(6):
        for v, t in enumerate(tokens):
            at = s if t else -1
            for byte in t or b"":
                at = trans[at, byte] if at >= 0 else -1
            assert (int(g.allowed[s, v >> 5]) >> (v & 31) & 1) == (at >= 0)
            assert g.next_state[s, v] == (at if at >= 0 else 6)


def test_token_grammar_refusals():
    for bad in (lambda: lm_ops.TokenGrammar(np.zeros((2, 255)), [b"A"], device="cpu"),
                lambda: lm_ops.TokenGrammar(np.full((2, 256), 2), [b"A"], device="cpu"),
                lambda: lm_ops.TokenGrammar(np.zeros((2, 256)), [], device="cpu"),
                lambda: lm_ops.TokenGrammar(np.zeros((2, 256)), [b"A"], eos_id=1, device="cpu"),
                lambda: lm_ops.TokenGrammar.from_iupac("AXG", [b"A"], device="cpu"),
                lambda: lm_ops.TokenGrammar.from_iupac("", [b"A"], device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_token_bytes():
    assert lm_ops.token_bytes({"A": 1, "[PAD]": 0, "ACGN": 3, "<unk>": 2}) == [None, b"A", None, b"ACGN"]


def test_quick_calls_are_the_calls_of_ctypes():
    from dnatok_amd import _hostpack
    L = _lib.lib()
    address = ctypes.cast(L.dnatok_w4_matvec, ctypes.c_void_p).value
    args = (4096, 64, 1, 4096, 7, 4096, None, 1, 4, 64, 32, None, 4096, 4, 1, None)
    assert _hostpack.call(address, *args) == L.dnatok_w4_matvec(*args) == -1
    assert b"overlap" in L.dnatok_last_error()
    for bad in ((), (0, 1), (None,), (address, "x"), (address,) + (0,) * 25):
        with pytest.raises(TypeError):
            _hostpack.call(*bad)
