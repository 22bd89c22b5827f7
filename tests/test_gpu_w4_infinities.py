"""Products with 4-bit weights of rows of x that hold infinities, NaN or numbers next to the largest: where the formula gives an
infinity the operator gives that one, NaN only where the formula has it (an infinity times a weight of 0 among them), and the other rows
are what they are without."""
import numpy as np
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support import lm_reference as ref
from tests.test_gpu_lm_ops import DEV, U, host, w4_inputs

pytestmark = pytest.mark.gpu
INF = float("inf")


# rows, outputs, columns, group: one row in LDS and too wide for it; blocks of sixteen rows by 1, 2 and 4 tiles, short and long
# slices; blocks of 64 rows; rows of x at the same place of their lines and elsewhere
SHAPES = [(1, 77, 1000, 64), (1, 40, 8200, 128), (2, 33, 416, 32), (17, 50, 2041, 128), (16, 8000, 512, 64), (16, 14500, 1152, 96),
          (61, 10300, 1000, 128), (64, 10240, 256, 64), (40, 10250, 320, 32)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group", SHAPES)
def test_w4_infinities_are_the_formulas(m, n, k, group, zeros, dtype):
    print(f"w4 infinities m={m} n={n} k={k} group={group} {dtype} zeros={zeros}", flush=True)
    q, scales, z, x, b = w4_inputs(m, n, k, group, dtype, zeros)
    matrix = lm_ops.W4Matrix(q, scales, z, in_features=k, group=group)
    clean = matrix.matvec(x, bias=b, out_dtype=torch.float32)
    big = 1e37 if dtype is torch.bfloat16 else 6e4
    plans = [{0: INF}, {k - 1: -INF}, {k // 2: INF, k // 3: -INF}, {5: float("nan")}, {k // 2: big, 1: -big}, {}]
    rows = sorted({0, m // 3, m // 2, m - 1})
    for shift in range(len(plans) if m == 1 else 2):
        bad = x.clone()
        for i, r in enumerate(rows):
            for at, v in plans[(i + 3 * shift) % len(plans) if m > 1 else shift].items():
                bad[r, at] = v
        got = matrix.matvec(bad, bias=b, out_dtype=torch.float32)
        hx, hs = host(bad), host(scales)
        with np.errstate(invalid="ignore"):
            want = ref.w4(hx[rows], q.cpu().numpy(), hs, None if z is None else z.cpu().numpy(), k, group, host(b))
        out = host(got)[rows]
        assert np.array_equal(np.isnan(out), np.isnan(want))
        infinite = np.isinf(want)
        assert np.array_equal(out[infinite], want[infinite])
        fine = np.isfinite(want)
        most = np.where(np.isfinite(hx), np.abs(hx), 0.0).sum(1)[rows][:, None]
        tol = 4 * min(group, k) ** 0.5 * U * 144 * hs.max() * most + 8 * U * np.abs(np.where(fine, want, 0.0))
        assert (np.abs(np.where(fine, out - np.where(fine, want, 0.0), 0.0)) <= tol).all()
        others = [r for r in range(m) if r not in rows]
        assert torch.equal(got[others], clean[others])
