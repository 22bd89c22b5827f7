"""Groups of more columns than the matrix has, up to sizes that 32 bits do not hold."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import w4_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [1024, 2 ** 31 - 32, 2 ** 31, 2 ** 32, 2 ** 32 + 32, 2 ** 40 + 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 7])
def test_w4_group_of_all_columns(m, dtype, group):
    k = 1000
    print(f"w4 m={m} {dtype} group={group}", flush=True)
    q, scales, z, x, b = w4_inputs(m, 90, k, 1024, dtype, True)
    want = lm_ops.W4Matrix(q, scales, z, in_features=k, group=1024).matvec(x, bias=b)
    assert torch.equal(lm_ops.W4Matrix(q, scales, z, in_features=k, group=group).matvec(x, bias=b), want)
