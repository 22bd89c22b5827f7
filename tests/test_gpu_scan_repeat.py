"""The recurrence gives the same bits from call to call, also where channels keep their state over many groups of tiles, so that
a tile may find the state in front of it in several ways."""
import pytest
import torch

from dnatok_amd import lm_ops
from tests.test_gpu_lm_ops import DEV, TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,reverse", [(256, False), (256, True), (7, False)])
def test_scan_of_slow_channels_is_the_same_every_time(dtype, dim, reverse):
    total = 300000
    print(f"gated_scan repeated dim={dim} {dtype} reverse={reverse}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    x, gate, dy = (torch.randn((total, dim), generator=g, device=DEV).to(dtype) for _ in range(3))
    gate += torch.linspace(-1.0, 10.0, dim, device=DEV).to(dtype)
    dlast = torch.randn((2, dim), generator=g, device=DEV)
    off = torch.tensor([0, 250001, total], device=DEV)
    x.requires_grad_(True), gate.requires_grad_(True)
    other = torch.empty(64 << 20, device=DEV)
    side = torch.cuda.Stream()
    first = None
    for i in range(12):
        if i % 3 == 2:                                                 # (with other work on the card now and then)
            with torch.cuda.stream(side):
                other.fill_(float(i))
        y, last = lm_ops.gated_scan(x, gate, off, reverse=reverse)
        out = (y, last) + torch.autograd.grad((y, last), (x, gate), (dy, dlast))
        if first is None:
            first = [t.detach().clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(first, out)), i
    side.synchronize()
