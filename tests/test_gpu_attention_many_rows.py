"""Linear attention over as many rows and heads as take more than one launch (one has less than 2^32 threads)."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.support.attention_reference import U

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_short_reads():
    """600,000 rows of one token and 16 heads, room in front of them and behind: every result has a closed form."""
    rows, heads, front, behind = 600000, 16, 3, 70
    total = front + rows + behind
    g = torch.Generator(device=DEV).manual_seed(0)
    print("linear_attention of", rows, "rows of", heads, "heads", flush=True)
    q, k, dy = (torch.randn((total, heads, 4), generator=g, device=DEV).requires_grad_(i < 2) for i in range(3))
    v = torch.randn((total, heads, 4), generator=g, device=DEV).requires_grad_(True)
    ld = torch.linspace(-2.0, 0.0, heads, device=DEV)
    off = torch.arange(front, front + rows + 1, device=DEV)
    y, last = lm_ops.linear_attention(q, k, v, ld, off, scale=0.5)
    dlast = torch.randn(last.shape, generator=g, device=DEV)
    grads = torch.autograd.grad((y, last), (q, k, v), (dy, dlast))
    inner = slice(front, front + rows)

    def check(got, terms, count):
        """A sum of products, in 32 bits: a rounding of the sum of their sizes for each product and each sum."""
        off_by = (got.detach().double() - terms.sum(-1)).abs() - count * U * terms.abs().sum(-1)
        assert off_by.max().item() <= 0

    qd, kd, vd, gd = (t.detach()[inner].double() for t in (q, k, v, dy))
    for lo in range(0, rows, 100000):
        part = slice(lo, lo + 100000)
        a, b, c, d, e = qd[part], kd[part], vd[part], 0.5 * gd[part], dlast[part].double()
        rows_of = lambda t: t.detach()[inner][part]
        check(rows_of(y), 0.5 * (a * b)[:, :, None, :] * c[..., None], 20)
        check(last[part], (b[..., None] * c[:, :, None])[..., None], 20)
        check(rows_of(grads[2]), torch.cat([(a * b)[:, :, None, :] * d[..., None], b[:, :, None, :] * e.transpose(2, 3)], -1), 20)
        check(rows_of(grads[1]), torch.cat([(c * d)[:, :, None, :] * a[..., None], c[:, :, None, :] * e], -1), 20)
        check(rows_of(grads[0]), (c * d)[:, :, None, :] * b[..., None], 20)
    for t in (y, *grads):
        assert (t[:front] == 0).all() and (t[front + rows:] == 0).all()
