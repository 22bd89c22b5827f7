"""Products with 4-bit weights of rows of x at any stride: what lies between them changes nothing, to the last bit."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import DEV, check_w4

pytestmark = pytest.mark.gpu


# tiles of 16 rows with slices of 4 and of 8 blocks, tiles of 64 rows; depths that end with a slice, a block and inside one
@pytest.mark.parametrize("m,n", [(2, 40), (17, 40), (64, 10300)])
@pytest.mark.parametrize("k", [1024, 2048, 2112, 2040])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_w4_rows_of_x_at_any_stride(m, n, k, group, dtype):
    matrix, x, _ = check_w4(m, n, k, group, dtype, True, bias=False)
    want = matrix.matvec(x)
    for more in (8, 32, 64 - k % 64, 128 - k % 64, 5):
        wide = torch.full((m, k + more), float("nan"), dtype=dtype, device=DEV)
        for first in (0, more):
            part = wide[:, first:first + k]
            part.copy_(x)
            assert torch.equal(matrix.matvec(part), want), (more, first)
            part.fill_(float("nan"))


def test_w4_one_row_broadcast():
    matrix, x, _ = check_w4(1, 300, 1024, 64, torch.bfloat16, True, bias=False)
    two = matrix.matvec(torch.cat((x, x)))
    assert torch.equal(matrix.matvec(x.expand(19, 1024))[17], two[0])
