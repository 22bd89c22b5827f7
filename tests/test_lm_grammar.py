"""Grammars over a vocabulary's tokens: chosen tokens that are no token of the vocabulary, and arguments that name no state (CPU)."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops

TOKENS = [b"T", b"C", b"G", b"TT", b"AC", None, b"A"]


def grammar(**kw):
    return lm_ops.TokenGrammar.from_iupac("ACGT", TOKENS, device="cpu", **kw)


@pytest.mark.parametrize("token", [-1, -2, -7, -8, 7, 8, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_advance_with_what_is_no_token(token, dtype):
    """Nothing may follow, as after a forbidden token; rows without a grammar stay without."""
    g = grammar(repeat=True)
    state = torch.tensor([0, 1, 3, -1, g.n_states], dtype=torch.int32)
    after = g.advance(state, torch.full((5,), token, dtype=dtype))
    assert after.tolist() == [g.n_states, g.n_states, g.n_states, -1, g.n_states] and after.dtype == torch.int32


def test_advance_follows_tokens():
    g = grammar()
    state = torch.tensor([0, 0, 1, 0, 3, -5], dtype=torch.int32)
    token = torch.tensor([6, 4, 1, 1, 0, 2])
    assert g.advance(state, token).tolist() == [1, 2, 2, g.n_states, 4, -5]
    assert g.next_state.shape == (g.n_states + 1, len(TOKENS)) and g.next_state.dtype == torch.int32


def test_refusals():
    trans = np.full((2, 256), -1)
    for bad in (np.full((2, 256), 2 ** 32), np.full((2, 256), -2 ** 32), np.full((2, 256), 0.5), np.full((2, 256), np.nan),
                np.full((2, 256), 2), np.full((2, 256), -2), trans[:, :255], trans[:0]):
        with pytest.raises(ValueError):
            lm_ops.TokenGrammar(bad, TOKENS, device="cpu")
    for accepting in ([2], [-1], [0, 5]):
        with pytest.raises(ValueError):
            lm_ops.TokenGrammar(trans, TOKENS, accepting=accepting, eos_id=5, device="cpu")
    assert lm_ops.TokenGrammar(trans.astype(np.float64), TOKENS, device="cpu").n_states == 2
    g = lm_ops.TokenGrammar(trans, TOKENS, accepting=iter([1]), eos_id=5, device="cpu")
    assert g.advance(torch.tensor([0, 1], dtype=torch.int32), torch.tensor([5, 5])).tolist() == [2, 1]
