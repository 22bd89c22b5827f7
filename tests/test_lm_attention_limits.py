"""What the C entries of linear attention take that looks like too much (no GPU needed: a null buffer, which is looked at later, is what
they refuse)."""
import pytest

from dnatok_amd import _lib
from tests.test_lm_more_abi import INVALID, P, TOO_LARGE, backward, forward, shape

FAR = [dict(q_token=2 ** 40), dict(k_token=2 ** 23), dict(v_token=2 ** 62), dict(q_token=2 ** 24, k_token=2 ** 24, v_token=2 ** 24, dy_token=2 ** 24)]


def step(q=None, **change):
    return _lib.lib().dnatok_linear_attention_step(shape(**change), q, P, P, P, P, P, P, None)


@pytest.mark.parametrize("far", FAR)
def test_the_stride_of_a_single_token_is_that_of_no_address(far):
    one = dict(n_rows=1, total=1, **far)
    assert forward(q=None, **one) == INVALID and backward(dy=None, **one) == INVALID and step(**one) == INVALID
    assert forward(q=None, **{**one, "total": 2}) == TOO_LARGE and step(**{**one, "n_rows": 2}) == TOO_LARGE
    assert forward(**{**one, "q_token": -1}) == INVALID


@pytest.mark.parametrize("heads,rows", [(16, 600000), (64, 2 ** 22), (65535, 1000)])
def test_many_rows_of_many_heads(heads, rows):
    many = dict(heads=heads, kv_heads=1, n_rows=rows, total=rows)
    assert forward(q=None, **many) == INVALID and backward(dy=None, **many) == INVALID
    assert forward(q=None, **{**many, "n_rows": 2 ** 23, "total": 2 ** 23}) == TOO_LARGE
