"""Products of 33 to 64 rows and more about the place where sixteen rows at a time give way to 64: as many workgroups of the former as
run at once, and one more."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import DEV, check_w4, w4_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(33, 170 * 64), (33, 170 * 64 + 1), (48, 171 * 64), (49, 128 * 64), (49, 128 * 64 + 1), (64, 128 * 64 + 64),
                                 (65, 102 * 64), (65, 103 * 64), (130, 57 * 64 + 5), (200, 40 * 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [130, 256])
def test_w4_about_512_workgroups(m, n, k, dtype):
    check_w4(m, n, k, 64, dtype, m % 2 == 0, torch.float32 if n % 2 else None)


@pytest.mark.parametrize("m,n", [(61, 10300), (40, 11000)])
def test_w4_of_64_rows_with_rows_of_weights_far_apart(m, n):
    k, group, stride = 1000, 64, 2 ** 16
    print(f"w4 m={m} n={n} k={k} stride={stride}", flush=True)
    q, scales, z, x, b = w4_inputs(m, n, k, group, torch.bfloat16, True)
    wide = torch.zeros(n * stride, dtype=torch.int32, device=DEV)
    far = wide.as_strided(q.shape, (stride, 1))
    far.copy_(q)
    got = lm_ops.W4Matrix(far, scales, z, in_features=k, group=group).matvec(x, bias=b)
    assert torch.equal(got, lm_ops.W4Matrix(q, scales, z, in_features=k, group=group).matvec(x, bias=b))
