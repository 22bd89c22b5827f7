"""What may be an output of the model operators' calls: which places it may share with an input, and that autograd learns of it (the
checks alone, on the CPU)."""
import pytest
import torch

from dnatok_amd import lm_ops


def ok(out, *inputs, **kw):
    lm_ops._require_out("op", out, *inputs, **kw)


def bad(out, *inputs, **kw):
    with pytest.raises(ValueError, match="overlap"):
        lm_ops._require_out("op", out, *inputs, **kw)


def test_rows_of_an_output_have_places_of_their_own():
    wide = torch.zeros(6, 20)
    ok(wide), ok(wide[:, 3:9]), ok(wide[::2]), ok(wide[:1].expand(1, 20)), ok(torch.zeros(4, 1)), ok(torch.zeros(1, 4).t())
    bad(torch.zeros(1, 20).expand(6, 20))
    bad(torch.zeros(40).as_strided((3, 20), (10, 1)))
    ok(torch.zeros(0, 5)), ok(torch.zeros(5, 0)), ok(torch.zeros(1, 5).as_strided((1, 5), (0, 1)))


def test_outputs_and_inputs_in_one_buffer():
    wide = torch.zeros(6, 20)
    ok(wide[:, :5], wide[:, 5:10]), ok(wide[:, 10:], wide[:, :10]), ok(wide[:3], wide[3:]), ok(wide[3:], wide[:3])
    bad(wide[:, :5], wide[:, 4:9]), bad(wide[:, 4:9], wide[:, :5]), bad(wide[:3], wide[2:5]), bad(wide[2:5], wide[:3])
    bad(wide[:, 15:], wide.view(-1)[18:118].view(5, 20)[:, :6])        # columns that reach around into the next row
    ok(wide[:, :5], wide[:, :5]), ok(wide, wide), ok(wide, None, torch.zeros(6, 20))
    bad(wide, wide, in_place=False), ok(wide[:, :5], wide[:, 5:10], in_place=False)
    bad(wide.view(12, 10)[:6], wide[:, :10])                           # from one place on, other places
    bad(wide.view(torch.bfloat16)[:, :20], wide)                       # another type
    bad(wide, wide[0]), ok(wide[1:], wide[0]), bad(wide[:2], wide.view(-1)[25:30])
    ok(wide[:1], wide[1:2]), bad(wide[:1, :5], wide[:1, 4:9]), ok(wide[:1, :5], wide[:1, 5:9])


def test_autograd_learns_that_an_output_was_written():
    w = torch.ones(3, 4, requires_grad=True)
    h = w * 2.0
    loss = (h * h).sum()                                               # keeps h
    with torch.no_grad():
        ok(h, h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        ok(torch.zeros(2, 2))
