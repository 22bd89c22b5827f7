"""What a matrix of 4-bit weights hands to its C entry point (no GPU needed: the call is caught)."""
import pytest
import torch

from dnatok_amd import lm_ops


@pytest.mark.parametrize("k,group,handed", [(1000, 64, 64), (1000, 1024, 1024), (1000, 2 ** 32 + 32, 2 ** 30), (33, 2 ** 31, 2 ** 30)])
def test_group_fits_the_entry_point(monkeypatch, k, group, handed):
    calls = []
    monkeypatch.setattr(lm_ops, "_run", lambda name, device, *args: calls.append(args))
    monkeypatch.setattr(lm_ops, "_require_floats", lambda *a, **kw: None)
    groups = -(-k // group)
    matrix = lm_ops.W4Matrix(torch.zeros((4, -(-k // 8)), dtype=torch.int32), torch.zeros((4, groups)).bfloat16(), in_features=k,
                             group=group)
    matrix.matvec(torch.zeros((1, k)).bfloat16())
    assert calls[0][10] == handed and matrix.group == group
