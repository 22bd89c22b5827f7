"""Model operators on the rows that the encoders write: embeddings, a gated linear recurrence and linear attention
(training and single steps), products with 4-bit weights, logits on their way to the choice of a token, and beam
search.

Thin torch-tensor wrappers over the C ABI like :mod:`dnatok_amd.encoders`: every call runs HIP kernels of
libdnatok_hip.so on the current stream of its tensors' device, and none of them synchronises.  The
reference has no counterpart.
"""
from __future__ import annotations

import array
import ctypes
import functools
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

try:                                    # quick calls; without the C module ctypes makes them
    from ._hostpack import call as _quick_call
except ImportError:                     # pragma: no cover
    _quick_call = None

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    """A C entry point that takes integers and pointers and returns a status."""
    fn = getattr(_lib.lib(), name)
    if _quick_call is None:
        return fn
    return functools.partial(_quick_call, ctypes.cast(fn, ctypes.c_void_p).value)


def _run(name: str, device: torch.device, *args) -> None:
    """Calls an entry point on the current stream of ``device``, the last argument of all of them."""
    index = device.index
    if index == torch.cuda.current_device():
        stream = _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream().cuda_stream
        rc = _entry(name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = _entry(name)(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        _lib.check(rc, name)


def _no_tangent(name: str, *tensors) -> None:
    """Forward-mode derivatives are refused: a kernel would drop them."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no forward-mode derivative")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require_rows(t: torch.Tensor, name: str, shape, dtype: torch.dtype, device: torch.device) -> int:
    """A matrix whose rows' elements lie next to each other; returns the elements between rows."""
    if t.dtype is dtype and t.shape == shape and t.device == device:
        stride = t.stride()
        if stride[1] == 1 or shape[1] == 1:
            return stride[0]
    raise ValueError(f"{name} must be a {dtype} tensor {tuple(shape)} on {device} with contiguous rows")


def _require(t: Optional[torch.Tensor], name: str, shape, dtype: torch.dtype, device: torch.device) -> None:
    if t is not None and not (t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.device == device):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {device}")


def _require_out(name: str, out: torch.Tensor, *inputs: Optional[torch.Tensor], in_place: bool = True) -> None:
    """``out``, a matrix, has a place of its own for each element and shares none with an input, unless the two are one
    and the operator reads each element before it writes it (``in_place``).  What autograd kept of ``out`` is out of date from
    here on."""
    rows, cols = out.shape
    pitch, size = out.stride(0), out.element_size()
    if rows > 1 and pitch < cols:
        raise ValueError(f"{name}: rows of the output overlap")
    first, width = out.data_ptr(), cols * size
    end = first + (max(rows - 1, 0) * pitch + cols) * size
    for t in inputs:
        if t is None or t.numel() == 0 or out.numel() == 0:
            continue
        own = t.stride(0) if t.dim() == 2 and t.size(0) > 1 else 0
        wide = t.size(-1) * t.element_size()
        at = t.data_ptr()
        if at >= end or at + ((t.size(0) - 1) * own * t.element_size() if t.dim() == 2 else 0) + wide <= first:
            continue
        if in_place and t.dtype is out.dtype and t.shape == out.shape and at == first and (rows <= 1 or own == pitch):
            continue
        if rows > 1 and own * t.element_size() == pitch * size:       # columns of one matrix next to each other
            apart = (at - first) % (pitch * size)
            if apart >= width and apart + wide <= pitch * size:
                continue
        raise ValueError(f"{name}: the output overlaps an input")
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _require_floats(t: torch.Tensor, name: str, types=tuple(_DTYPES)) -> None:
    if not t.is_cuda or t.dtype not in types:
        raise ValueError(f"{name} must be on the GPU, of " + ", ".join(str(d) for d in types))


# ---- gated linear recurrence ------------------------------------------------------------------

class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, offsets, n_rows, h0, reverse):
        y, last, states = _scan_forward(x, gate, offsets, n_rows, h0, reverse, True)
        ctx.save_for_backward(x, gate, offsets, h0, states)
        ctx.n_rows, ctx.reverse = n_rows, reverse
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, gate, offsets, h0, states = ctx.saved_tensors
        total, dim = x.shape
        device, L = x.device, _lib.lib()
        if dy is not None and dim > 1 and dy.stride(1) != 1:
            dy = dy.contiguous()
        if dlast is not None:
            dlast = dlast.contiguous()
        dx = torch.empty((total, dim), dtype=x.dtype, device=device)
        dgate = torch.empty_like(dx)
        dh0 = torch.empty_like(h0) if h0 is not None and ctx.needs_input_grad[4] else None
        code = _DTYPES[x.dtype]
        need = L.dnatok_gated_scan_work_bytes(total, dim)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _run("dnatok_gated_scan_backward", device, x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0), code,
             _ptr(offsets), ctx.n_rows, total, dim, int(ctx.reverse), _ptr(h0), _ptr(dy),
             0 if dy is None else dy.stride(0), _ptr(dlast), states.data_ptr(), dx.data_ptr(), dgate.data_ptr(), _ptr(dh0),
             _ptr(work), need)
        return dx, dgate, None, None, dh0, None


def _scan_forward(x, gate, offsets, n_rows, h0, reverse, keep_states):
    total, dim = x.shape
    device, code, L = x.device, _DTYPES[x.dtype], _lib.lib()
    y = torch.empty((total, dim), dtype=x.dtype, device=device)
    last = torch.empty((n_rows, dim), dtype=torch.float32, device=device)
    states = None
    if keep_states:
        states = torch.empty(L.dnatok_gated_scan_states_bytes(total, dim) // 4, dtype=torch.float32, device=device)
    need = L.dnatok_gated_scan_work_bytes(total, dim)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _run("dnatok_gated_scan", device, x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0), code, _ptr(offsets), n_rows,
         total, dim, int(reverse), _ptr(h0), y.data_ptr(), last.data_ptr(), _ptr(states), _ptr(work), need)
    return y, last, states


def gated_scan(x: torch.Tensor, gate: torch.Tensor, offsets: Optional[torch.Tensor] = None, *,
               h0: Optional[torch.Tensor] = None, reverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence ``h_t = f_t h_(t-1) + (1 - f_t) x_t`` with ``f = sigmoid(gate)``, in every channel of
    every row.  Returns ``(y, last)``: the states in x's type and shape, and the state behind each row's last
    step, float32 [B, D].

    ``x`` and ``gate`` are packed rows [total, D] with ``offsets`` int64 [B + 1] as the encoders write
    them (ascending; rows may be empty, and there may be room behind the last one, as
    :func:`dnatok_amd.encoders.pack_ragged` leaves it: tokens in no row give zeros, also as gradients), or dense rows [B, T, D] without offsets (copied where they do not lie like packed
    ones); float32, bfloat16 or float16, the elements of
    a token next to each other (halves of one projection's output will do).  ``h0`` float32 [B, D] is the
    state in front of each row, zero if not given; ``reverse`` runs rows from their last token to their
    first.  States are held in 32 bits.  Differentiable (once) with respect to x, gate and h0."""
    _require_floats(x, "x")
    if x.dim() == 3 and offsets is None:
        b, t, d = x.shape
        if gate.shape != x.shape:
            raise ValueError("gate must have x's shape")
        y, last = _gated_scan(x.reshape(b * t, d), gate.reshape(b * t, d), None, b, h0, reverse)
        return y.view(b, t, d), last
    if x.dim() != 2 or offsets is None:
        raise ValueError("x must be [total, D] with offsets, or [B, T, D] without")
    if offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError("offsets must be int64 [B + 1]")
    _require(offsets, "offsets", offsets.shape, torch.int64, x.device)
    return _gated_scan(x, gate, offsets, offsets.numel() - 1, h0, reverse)


def _gated_scan(x, gate, offsets, n_rows, h0, reverse):
    total, dim = x.shape
    if dim == 0:
        raise ValueError("x has no channels")
    if n_rows == 0 and total:
        raise ValueError("tokens without rows")
    _require_rows(x, "x", x.shape, x.dtype, x.device)
    _require_rows(gate, "gate", x.shape, x.dtype, x.device)
    _require(h0, "h0", (n_rows, dim), torch.float32, x.device)
    _no_tangent("gated_scan", x, gate, h0)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, gate, offsets, n_rows, h0, reverse)
    return _scan_forward(x, gate, offsets, n_rows, h0, reverse, False)[:2]


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor] = None, *,
               out_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of :func:`gated_scan` for one token of each row: ``x`` and ``gate`` [B, D], ``state``
    float32 [B, D] (zero if not given).  Returns ``(y, new_state)``; ``out_state`` receives the new state and may be
    ``state`` itself.  Without gradients."""
    _require_floats(x, "x")
    shape, dtype, device = x.shape, x.dtype, x.device
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError("x must be [B, D]")
    xs = _require_rows(x, "x", shape, dtype, device)
    gs = _require_rows(gate, "gate", shape, dtype, device)
    _require(state, "state", shape, torch.float32, device)
    _require(out_state, "out_state", shape, torch.float32, device)
    _forward_only("gated_step", x, gate, state, out_state)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if out_state is None:
        out_state = torch.empty_like(y, dtype=torch.float32)
    else:
        _require_out("gated_step", out_state, x, gate, state)
    _run("dnatok_gated_step", device, x.data_ptr(), xs, gate.data_ptr(), gs, _DTYPES[dtype], _ptr(state), shape[0], shape[1],
         y.data_ptr(), out_state.data_ptr())
    return y, out_state


def _forward_only(name: str, *tensors) -> None:
    _no_tangent(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward pass: call it under torch.no_grad()")


# ---- linear attention -------------------------------------------------------------------------

_FAR_TOKENS = 1 << 23                   # elements between tokens that are too many (dnatok_linear_shape)
_STEP_ROWS = 65535                      # rows that one call of the step's entry takes


class _LinearPlan:
    """What calls of the same sizes have in common: their description for the C entries, and the sizes of their buffers."""

    def __init__(self, *fields):
        self.held = _lib.LinearShape(*fields)
        self.shape, L = ctypes.addressof(self.held), _lib.lib()
        self.states = L.dnatok_linear_attention_states_bytes(self.shape) // 4
        self.work, self.work_back = (L.dnatok_linear_attention_work_bytes(self.shape, i) for i in (0, 1))


@functools.lru_cache(maxsize=1024)
def _linear_plan(dtypes, devices, qs, q_stride, ks, k_stride, vs, v_stride, dy_stride, n_rows, scale, reverse, with_offsets) -> _LinearPlan:
    """Checks what linear attention takes for each token, q [N, H, Dk], k [N, G, Dk] and v [N, G, Dv]: once for calls of the
    same sizes."""
    if len(ks) != 3 or len(vs) != 3 or ks[0] != qs[0] or ks[2] != qs[2] or vs[:2] != ks[:2]:
        raise ValueError("q, k and v must be [.., H, Dk], [.., G, Dk] and [.., G, Dv] of the same tokens")
    (total, heads, dim_k), (_, kv_heads, dim_v) = qs, vs
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError("q's heads must be a multiple of k's and v's")
    if not 1 <= dim_k <= 128 or not 1 <= dim_v <= 128:
        raise ValueError("heads have 1 to 128 elements")
    for what, dtype, device, shape, stride in zip("qkv", dtypes, devices, (qs, ks, vs), (q_stride, k_stride, v_stride)):
        if dtype is not dtypes[0] or device != devices[0] or (shape[2] > 1 and stride[2] != 1):
            raise ValueError(f"{what} must be a {dtypes[0]} tensor on {devices[0]} with a head's elements next to each other")
    scale = dim_k ** -0.5 if scale is None else scale
    if not 2.0 ** -40 <= abs(scale) <= 2.0 ** 40:
        raise ValueError("scale must be 2^-40 to 2^40 in size")
    return _LinearPlan(_DTYPES[dtypes[0]], reverse, n_rows, total, heads, kv_heads, dim_k, dim_v, *q_stride[:2], *k_stride[:2],
                       *v_stride[:2], *dy_stride[:2], scale, with_offsets)


def _plan_of(q, k, v, n_rows, scale, reverse, with_offsets, dy=None) -> _LinearPlan:
    return _linear_plan((q.dtype, k.dtype, v.dtype), (q.device, k.device, v.device), q.shape, q.stride(), k.shape, k.stride(), v.shape,
                        v.stride(), (0, 0) if dy is None else dy.stride(), n_rows, None if scale is None else float(scale), reverse,
                        with_offsets)


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, offsets, n_rows, h0, scale, reverse):
        y, last, states = _linear_forward(q, k, v, log_decay, offsets, n_rows, h0, scale, reverse, True)
        ctx.save_for_backward(q, k, v, log_decay, offsets, h0, states)
        ctx.n_rows, ctx.scale, ctx.reverse = n_rows, scale, reverse
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        q, k, v, log_decay, offsets, h0, states = ctx.saved_tensors
        device, (total, heads, _), dim_v = q.device, q.shape, v.shape[2]
        if dy is None:
            dy = torch.zeros((1, 1, 1), dtype=q.dtype, device=device).expand(total, heads, dim_v)
        if (dim_v > 1 and dy.stride(2) != 1) or dy.stride(0) >= _FAR_TOKENS:     # (wherever autograd has put it)
            dy = dy.contiguous()
        if dlast is not None:
            dlast = dlast.contiguous()
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v))
        dh0 = torch.empty_like(h0) if h0 is not None and ctx.needs_input_grad[6] else None
        plan = _plan_of(q, k, v, ctx.n_rows, ctx.scale, int(ctx.reverse), int(offsets is not None), dy)
        need = plan.work_back
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _run("dnatok_linear_attention_backward", device, plan.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
             _ptr(offsets), _ptr(h0), dy.data_ptr(), _ptr(dlast), _ptr(states), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
             _ptr(dh0), _ptr(work), need)
        return dq, dk, dv, None, None, None, dh0, None, None


def _linear_forward(q, k, v, log_decay, offsets, n_rows, h0, scale, reverse, keep_states):
    (total, heads, dim_k), device, dim_v = q.shape, q.device, v.shape[2]
    plan = _plan_of(q, k, v, n_rows, scale, int(reverse), int(offsets is not None))
    y = torch.empty((total, heads, dim_v), dtype=q.dtype, device=device)
    last = torch.empty((n_rows, heads, dim_k, dim_v), dtype=torch.float32, device=device)
    states, need = None, plan.work
    if keep_states:
        states, need = torch.empty(plan.states, dtype=torch.float32, device=device), 0
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _run("dnatok_linear_attention", device, plan.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _ptr(offsets),
         _ptr(h0), y.data_ptr(), last.data_ptr(), _ptr(states), _ptr(work), need)
    return y, last, states


def _require_decay(name: str, log_decay: torch.Tensor, heads: int, device: torch.device) -> None:
    _require(log_decay, "log_decay", (heads,), torch.float32, device)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} has no gradient for log_decay")


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     offsets: Optional[torch.Tensor] = None, *, h0: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, reverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Linear attention with a decay for each head: ``S_t = exp(log_decay) S_(t-1) + k_t v_t^T`` and ``y_t = scale q_t S_t`` in
    every head of every row.  Returns ``(y, last)``: y [total, H, Dv] in q's type, and the states behind each row's last
    step, float32 [B, H, Dk, Dv].

    ``q`` [total, H, Dk], ``k`` [total, G, Dk] and ``v`` [total, G, Dv] are packed rows with ``offsets`` int64 [B + 1] as for
    :func:`gated_scan` (rows may be empty; tokens in no row give zeros, also as gradients), or dense rows [B, T, .., ..]
    without offsets (copied where they do not lie like packed ones); float32, bfloat16 or float16, the elements of a head
    next to each other (parts of one projection's output will do), tokens less than 2^23 elements apart; less than 2^23 rows and
    pieces of 512 tokens.  H is a multiple of G: neighbouring heads share keys and
    values.  Dk and Dv go up to 128.  ``log_decay`` float32 [H] is at most 0 (-inf: nothing is kept); ``scale`` is a number of
    2^-40 to 2^40 in size, Dk ** -0.5 if not given.  ``h0`` float32 [B, H, Dk, Dv] is the state in front of each row, zero if not given; ``reverse``
    runs rows from their last token to their first.  States and sums are held in 32 bits.  Infinities and NaN go on as the
    recurrence has them, forwards and in gradients, step by step where there are any (5 to 25 times the time).  Differentiable (once)
    with respect to q, k, v and h0."""
    _require_floats(q, "q")
    if q.dim() == 4 and offsets is None:
        if k.dim() != 4 or v.dim() != 4 or k.shape[:2] != q.shape[:2] or v.shape[:2] != q.shape[:2]:
            raise ValueError("q, k and v must be [.., H, Dk], [.., G, Dk] and [.., G, Dv] of the same tokens")
        b, t = q.shape[:2]
        y, last = _linear_attention(*(x.reshape(b * t, x.shape[2], x.shape[3]) for x in (q, k, v)), log_decay, None, b, h0, scale,
                                    reverse)
        return y.view(b, t, *y.shape[1:]), last
    if q.dim() != 3 or offsets is None:
        raise ValueError("q must be [total, H, Dk] with offsets, or [B, T, H, Dk] without")
    if offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError("offsets must be int64 [B + 1]")
    _require(offsets, "offsets", offsets.shape, torch.int64, q.device)
    return _linear_attention(q, k, v, log_decay, offsets, offsets.numel() - 1, h0, scale, reverse)


def _linear_attention(q, k, v, log_decay, offsets, n_rows, h0, scale, reverse):
    _plan_of(q, k, v, n_rows, scale, int(reverse), int(offsets is not None))
    if n_rows == 0 and q.shape[0]:
        raise ValueError("tokens without rows")
    _require_decay("linear_attention", log_decay, q.shape[1], q.device)
    _require(h0, "h0", (n_rows, q.shape[1], q.shape[2], v.shape[2]), torch.float32, q.device)
    _no_tangent("linear_attention", q, k, v, log_decay, h0)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (h0 is not None and h0.requires_grad)):
        return _LinearAttention.apply(q, k, v, log_decay, offsets, n_rows, h0, scale, reverse)
    return _linear_forward(q, k, v, log_decay, offsets, n_rows, h0, scale, reverse, False)[:2]


def _extent(t: torch.Tensor) -> Tuple[int, int]:
    """The first byte of a tensor and the one behind its last."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else first


def _require_apart(name: str, out: torch.Tensor, *inputs: Optional[torch.Tensor], same: Optional[torch.Tensor] = None) -> None:
    """``out``, which is contiguous, shares no memory with the inputs; ``same`` may be all of it, but no part."""
    first, end = _extent(out)
    for t in inputs:
        lo, hi = (0, 0) if t is None else _extent(t)
        if lo < end and first < hi and not (t is same and lo == first and hi == end and t.is_contiguous()):
            raise ValueError(f"{name}: the output overlaps an input")
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                          out_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of :func:`linear_attention` for one token of each row: ``q`` [B, H, Dk], ``k`` [B, G, Dk], ``v`` [B, G, Dv],
    ``state`` float32 [B, H, Dk, Dv] (zero if not given).  Returns ``(y, new_state)``; ``out_state`` receives the new state
    and may be ``state`` itself.  Tokens that lie 2^23 elements apart or more (the last ones of long prompts) are copied.  Without
    gradients."""
    _require_floats(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [B, H, Dk]")
    device, given, rows = q.device, (q, k, v), q.shape[0]
    if rows > 1:                             # (the C entries take no tokens that lie farther apart)
        q, k, v = (t.contiguous() if t.dim() == 3 and t.stride(0) >= _FAR_TOKENS else t for t in given)
    plan = _plan_of(q, k, v, rows, scale, 0, 0)
    shape = (*q.shape, v.shape[2])
    _require_decay("linear_attention_step", log_decay, shape[1], device)
    _require(state, "state", shape, torch.float32, device)
    _require(out_state, "out_state", shape, torch.float32, device)
    _forward_only("linear_attention_step", q, k, v, log_decay, state, out_state)
    y = q.new_empty((shape[0], shape[1], shape[3]))
    if out_state is None:
        out_state = torch.empty(shape, dtype=torch.float32, device=device)
    else:
        _require_apart("linear_attention_step", out_state, *given, log_decay, state, same=state)
    if rows <= _STEP_ROWS:
        _run("dnatok_linear_attention_step", device, plan.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
             _ptr(state), y.data_ptr(), out_state.data_ptr())
        return y, out_state
    for first in range(0, rows, _STEP_ROWS):
        here = slice(first, first + _STEP_ROWS)
        plan = _plan_of(q[here], k[here], v[here], min(_STEP_ROWS, rows - first), scale, 0, 0)
        _run("dnatok_linear_attention_step", device, plan.shape, q[here].data_ptr(), k[here].data_ptr(), v[here].data_ptr(),
             log_decay.data_ptr(), None if state is None else state[here].data_ptr(), y[here].data_ptr(), out_state[here].data_ptr())
    return y, out_state


# ---- embeddings -------------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _host_float(value: float) -> Tuple[ctypes.c_float, int]:
    """A number in host memory, and its address."""
    held = ctypes.c_float(value)
    return held, ctypes.addressof(held)


@functools.lru_cache(maxsize=1024)
def _embedding_work(n: int, vocab: int, dim: int) -> int:
    return _lib.lib().dnatok_embedding_work_bytes(n, vocab, dim)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.shape, ctx.dtype = scale, weight.shape, weight.dtype
        return _embed(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (ids,), (vocab, dim), device = ctx.saved_tensors, ctx.shape, dy.device
        n = ids.numel()
        dy = dy.reshape(n, dim)
        if dim > 1 and dy.stride(1) != 1:
            dy = dy.contiguous()
        grad = torch.empty((vocab, dim), dtype=ctx.dtype, device=device)
        need = _embedding_work(n, vocab, dim)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        held, at = _host_float(ctx.scale)
        _run("dnatok_embedding_backward", device, ids.data_ptr(), ids.element_size(), n, dy.data_ptr(), dy.stride(0),
             _DTYPES[ctx.dtype], vocab, dim, at, grad.data_ptr(), _ptr(work), need)
        return None, grad, None


def _embed(ids, weight, scale):
    vocab, dim = weight.shape
    y = torch.empty((*ids.shape, dim), dtype=weight.dtype, device=weight.device)
    held, at = _host_float(scale)
    _run("dnatok_embedding", weight.device, ids.data_ptr(), ids.element_size(), ids.numel(), weight.data_ptr(), weight.stride(0),
         _DTYPES[weight.dtype], vocab, dim, at, y.data_ptr())
    return y


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale weight[ids]``: the rows of ``weight`` [V, D] (float32, bfloat16 or float16) for ``ids`` int32 or int64 of any
    shape, as the encoders pack or pad them.  An id outside 0 .. V - 1 (-1 for none) gives a row of zeros, and has no part in
    the gradient.  Differentiable (once) with respect to the weight: its gradient is a 32-bit sum over each id's tokens,
    rounded once, the same to the last bit from call to call."""
    _require_floats(weight, "weight")
    if weight.dim() != 2:
        raise ValueError("weight must be [V, D]")
    _require_rows(weight, "weight", weight.shape, weight.dtype, weight.device)
    if ids.dtype not in (torch.int32, torch.int64) or ids.device != weight.device:
        raise ValueError(f"ids must be int32 or int64 on {weight.device}")
    scale = float(scale)
    if not abs(scale) < 3.4e38:
        raise ValueError("scale must be a finite number")
    _no_tangent("embedding", weight)
    ids = ids.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(ids, weight, scale)
    return _embed(ids, weight, scale)


# ---- products with 4-bit weights --------------------------------------------------------------

class W4Matrix:
    """A weight matrix [N, K] of 4-bit whole numbers with a scale per group of ``group`` columns:
    ``W[n, k] = (q[n, k] - zero[n, k // group]) * scale[n, k // group]``.

    ``q`` int32 [N, ceil(K / 8)] holds eight values to a word, the lowest bits first; ``scales`` [N, ceil(K / group)]
    are bfloat16 or float16, the type of the activations; ``zeros`` uint8 [N, ceil(K / group)] hold 0 .. 15
    (8 everywhere if not given); ``group`` is a multiple of 32 (C ABI: dnatok_w4_matvec)."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
                 in_features: int, group: int):
        _require_floats(scales, "scales", (torch.bfloat16, torch.float16))
        self.in_features, self.group = int(in_features), int(group)
        if self.in_features <= 0 or self.group <= 0 or self.group % 32:
            raise ValueError("in_features must be positive and group a multiple of 32")
        if q.dim() != 2:
            raise ValueError("q must be int32 [N, ceil(K / 8)]")
        self.out_features = q.shape[0]
        groups = -(-self.in_features // self.group)
        _require_rows(q, "q", (self.out_features, -(-self.in_features // 8)), torch.int32, scales.device)
        _require(scales, "scales", (self.out_features, groups), scales.dtype, scales.device)
        _require(zeros, "zeros", (self.out_features, groups), torch.uint8, scales.device)
        self.q, self.scales, self.zeros = q, scales, zeros
        self._group = min(self.group, 1 << 30)         # (32 bits at the C entry; more columns than a matrix has)

    @classmethod
    def quantize(cls, weight: torch.Tensor, group: int = 128, *, symmetric: bool = True,
                 dtype: torch.dtype = torch.bfloat16) -> "W4Matrix":
        """Rounds a weight [N, K] to 4 bits, group by group: to the whole numbers -8 .. 7 times the scale that
        fits the group's largest value, or between the group's smallest and largest value with a zero point."""
        n, k = weight.shape
        groups = -(-k // group)
        w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group - k)).view(n, groups, group)
        if symmetric:
            scale = (w.abs().amax(2) / 7.0).to(dtype)
            zero = torch.full_like(scale, 8.0, dtype=torch.float32)
        else:
            lo, hi = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
            scale = ((hi - lo) / 15.0).to(dtype)
            zero = torch.where(scale > 0, (-lo / scale.float()).round(), torch.zeros_like(lo)).clamp(0, 15)
        step = torch.where(scale > 0, scale, torch.ones_like(scale)).float()
        q = ((w / step[:, :, None]).round() + zero[:, :, None]).clamp(0, 15).to(torch.int64).view(n, -1)[:, :k]
        q = torch.nn.functional.pad(q, (0, -k % 8)).view(n, -1, 8)
        words = (q << torch.arange(0, 32, 4, device=q.device)).sum(2)
        words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        return cls(words, scale, None if symmetric else zero.to(torch.uint8), in_features=k, group=group)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weights [N, K] as numbers."""
        shift = torch.arange(0, 32, 4, device=self.q.device, dtype=torch.int32)
        w = ((self.q[:, :, None] >> shift) & 15).flatten(1)[:, :self.in_features].float()
        zero = torch.full_like(self.scales, 8.0) if self.zeros is None else self.zeros
        each = torch.arange(self.in_features, device=self.q.device) // self.group
        return ((w - zero.float()[:, each]) * self.scales.float()[:, each]).to(dtype)

    def matvec(self, x: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x W^T + bias`` for the few rows of ``x`` [M, K] (or one vector [K]), which has the scales' type:
        one token of each sequence.  ``bias`` is float32 [N]; the result has x's type or ``out_dtype`` =
        float32, and goes to ``out``, which shares no memory with them, if given.  Without gradients."""
        squeeze = x.dim() == 1
        if squeeze:
            x = x.unsqueeze(0)
        if x.dim() != 2:
            raise ValueError("x must be [M, K] or [K]")
        device = self.scales.device
        m, n, k = x.shape[0], self.out_features, self.in_features
        xs = _require_rows(x, "x", (m, k), self.scales.dtype, device)
        _require(bias, "bias", (n,), torch.float32, device)
        _forward_only("W4Matrix.matvec", x, bias, self.scales, out)
        if out_dtype is None:
            out_dtype = x.dtype if out is None else out.dtype
        if out_dtype not in (x.dtype, torch.float32):
            raise ValueError("out_dtype must be x's type or float32")
        given = out is not None
        if not given:
            out = x.new_empty((m, n), dtype=out_dtype)
        elif squeeze:
            out = out.unsqueeze(0)
        ys = _require_rows(out, "out", (m, n), out_dtype, device)
        if given:
            _require_out("W4Matrix.matvec", out, x, bias, in_place=False)
        _run("dnatok_w4_matvec", device, x.data_ptr(), xs, _DTYPES[x.dtype], self.q.data_ptr(), self.q.stride(0),
             self.scales.data_ptr(), _ptr(self.zeros), m, n, k, self._group, _ptr(bias), out.data_ptr(), ys,
             _DTYPES[out_dtype])
        return out[0] if squeeze else out


# ---- logits -----------------------------------------------------------------------------------

def _per_row(v, name: str, rows: int, device: torch.device) -> Optional[torch.Tensor]:
    if v is None or isinstance(v, torch.Tensor):
        _require(v, name, (rows,), torch.float32, device)
        return v
    return torch.full((rows,), float(v), dtype=torch.float32, device=device)


def process_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                   history_offsets: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None,
                   repetition: Union[None, float, torch.Tensor] = None,
                   presence: Union[None, float, torch.Tensor] = None,
                   frequency: Union[None, float, torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Penalties for tokens that a row's history holds, biases and a grammar's mask on logits [B, V].

    ``history`` int32 and ``history_offsets`` int64 [B + 1] are packed ids as the encoders write them (prompt
    first, then what was generated; ids outside the vocabulary count for nothing) and ``prompt_lengths``
    int32 [B] says how many of a row's ids are its prompt.  A token that the history holds anywhere has its logit
    divided by ``repetition`` where positive and multiplied where not; ``presence`` + ``frequency`` x count is
    taken off tokens that were generated.  The three are numbers or float32 [B].  ``bias`` float32 [V] or
    [B, V] is added.  ``allowed`` int32 [S, ceil(V / 32)] holds bit masks (see :class:`TokenGrammar`) and
    ``state`` int32 [B] each row's mask, negative for none; tokens without their bit become -inf, all of them
    where a mask is empty.  The result has the logits' type or ``out_dtype`` = float32; ``out`` may be the logits.  Without
    gradients."""
    _require_floats(logits, "logits")
    if logits.dim() != 2:
        raise ValueError("logits must be [B, V]")
    device, (rows, vocab) = logits.device, logits.shape
    stride = _require_rows(logits, "logits", logits.shape, logits.dtype, device)
    if (history is None) != (history_offsets is None):
        raise ValueError("history and history_offsets go together")
    if history is None and any(v is not None for v in (prompt_lengths, repetition, presence, frequency)):
        raise ValueError("penalties need a history")
    if history is not None:
        _require(history, "history", (history.numel(),), torch.int32, device)
        _require(history_offsets, "history_offsets", (rows + 1,), torch.int64, device)
        if history.numel() == 0:                       # (an empty tensor has no address)
            history = history_offsets = None
    _require(prompt_lengths, "prompt_lengths", (rows,), torch.int32, device)
    bias_stride = 0
    if bias is not None and bias.dim() == 2:
        bias_stride = _require_rows(bias, "bias", (rows, vocab), torch.float32, device)
    else:
        _require(bias, "bias", (vocab,), torch.float32, device)
    n_states = allowed_stride = 0
    if allowed is not None:
        if allowed.dim() != 2 or allowed.shape[0] == 0:
            raise ValueError("allowed must be int32 [S, ceil(V / 32)]")
        n_states = allowed.shape[0]
        allowed_stride = _require_rows(allowed, "allowed", (n_states, -(-vocab // 32)), torch.int32, device)
        if state is None and n_states not in (1, rows):
            raise ValueError("allowed without state must hold one mask, or one of each row")
    elif state is not None:
        raise ValueError("state needs allowed")
    _require(state, "state", (rows,), torch.int32, device)
    _forward_only("process_logits", logits, bias, out,
                  *(v for v in (repetition, presence, frequency) if isinstance(v, torch.Tensor)))
    if out_dtype is None:
        out_dtype = logits.dtype if out is None else out.dtype
    if out_dtype not in (logits.dtype, torch.float32):
        raise ValueError("out_dtype must be the logits' type or float32")
    given = out is not None
    if not given:
        out = torch.empty_like(logits, dtype=out_dtype, memory_format=torch.contiguous_format)
    out_stride = _require_rows(out, "out", (rows, vocab), out_dtype, device)
    if given:
        _require_out("process_logits", out, logits, bias)
    repetition = _per_row(repetition, "repetition", rows, device)
    presence = _per_row(presence, "presence", rows, device)
    frequency = _per_row(frequency, "frequency", rows, device)
    _run("dnatok_logits_process", device, logits.data_ptr(), stride, _DTYPES[logits.dtype], rows, vocab, _ptr(history),
         _ptr(history_offsets), _ptr(prompt_lengths), _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(bias),
         bias_stride, _ptr(allowed), allowed_stride, n_states, _ptr(state), out.data_ptr(), out_stride, _DTYPES[out_dtype])
    return out


# the letters of a motif (IUPAC), and the bases that each stands for
IUPAC = {"A": "A", "C": "C", "G": "G", "T": "T", "R": "AG", "Y": "CT", "S": "CG", "W": "AT", "K": "GT", "M": "AC",
         "B": "CGT", "D": "AGT", "H": "ACT", "V": "ACG", "N": "ACGT"}


def token_bytes(vocab) -> list:
    """A tokenizer's vocabulary (token -> id) as the bytes of each id; None for ids whose token is not made of
    bases."""
    tokens = [None] * (max(vocab.values(), default=-1) + 1)
    for token, i in vocab.items():
        if token and not token.strip("ACGTN"):
            tokens[i] = token.encode("ascii")
    return tokens


class TokenGrammar:
    """A finite automaton over bytes, as bit masks and next states over a vocabulary's tokens.

    ``transitions`` [S, 256] holds the next state for each state and byte, -1 for none; ``tokens`` the bytes
    of each id (None: never allowed, see :func:`token_bytes`).  A token is allowed in a state if all its bytes can be
    followed from there; ``eos_id`` in the states of ``accepting`` only.  ``allowed`` int32 [S, ceil(V / 32)] is what
    :func:`process_logits` takes; ``advance`` follows the tokens that were chosen.  State S, behind the last one, is
    that of a row which took a forbidden token: nothing may follow."""

    def __init__(self, transitions, tokens: Sequence[Optional[bytes]], *, accepting: Sequence[int] = (),
                 eos_id: Optional[int] = None, device="cuda"):
        trans = np.asarray(transitions)
        if trans.ndim != 2 or trans.shape[1] != 256 or trans.shape[0] == 0:
            raise ValueError("transitions must be [S, 256]")
        s, v = trans.shape[0], len(tokens)
        if v == 0:
            raise ValueError("no tokens")
        if not np.array_equal(trans, np.trunc(trans)) or trans.min() < -1 or trans.max() >= s:
            raise ValueError("transitions must be whole numbers, and lead to states that are there")
        trans = trans.astype(np.int32)
        accepting = list(accepting)
        if any(not 0 <= a < s for a in accepting):
            raise ValueError("accepting names states that are not there")
        if eos_id is not None and not 0 <= eos_id < v:
            raise ValueError("eos_id is not in the vocabulary")
        lengths = np.array([0 if t is None else len(t) for t in tokens])
        table = np.zeros((v, max(1, lengths.max())), dtype=np.uint8)
        for i, t in enumerate(tokens):
            if t:
                table[i, :len(t)] = np.frombuffer(t, dtype=np.uint8)
        dead = np.concatenate([trans, np.full((1, 256), -1, dtype=np.int32)])     # (row -1: dead stays dead)
        state = np.where(lengths > 0, np.arange(s, dtype=np.int32)[:, None], -1)
        for at in range(table.shape[1]):
            state = np.where(lengths > at, dead[state, table[:, at]], state)
        if eos_id is not None:
            state[:, eos_id] = -1
            for a in accepting:
                state[a, eos_id] = a
        self.n_states, self.vocab = s, v
        bits = np.zeros((s, -(-v // 32) * 32), dtype=np.uint8)
        bits[:, :v] = state >= 0
        words = np.packbits(bits, axis=1, bitorder="little").view("<u4").view(np.int32)
        # (a column behind the last token, for what is no token)
        following = np.full((s + 1, v + 1), s, dtype=np.int32)
        following[:s, :v] = np.where(state < 0, s, state)
        self.allowed = torch.from_numpy(np.ascontiguousarray(words)).to(device)
        self._following = torch.from_numpy(following).to(device)
        self.next_state = self._following[:, :v]

    @classmethod
    def from_iupac(cls, pattern: str, tokens: Sequence[Optional[bytes]], *, repeat: bool = False,
                   eos_id: Optional[int] = None, device="cuda") -> "TokenGrammar":
        """Sequences that spell ``pattern`` (IUPAC letters), once, or again and again with ``repeat``.  State i: i letters
        of the pattern are there; the sequence may end where the pattern does."""
        n = len(pattern)
        if n == 0 or any(c not in IUPAC for c in pattern.upper()):
            raise ValueError("pattern must be IUPAC letters")
        states = n if repeat else n + 1
        trans = np.full((states, 256), -1, dtype=np.int32)
        for i, c in enumerate(pattern.upper()):
            for base in IUPAC[c]:
                trans[i, ord(base)] = (i + 1) % states
        return cls(trans, tokens, accepting=[0] if repeat else [n], eos_id=eos_id, device=device)

    def advance(self, state: torch.Tensor, token: torch.Tensor) -> torch.Tensor:
        """The states of rows in ``state`` int32 [B] that took ``token`` [B]; negative states stay.  A token that is not in the
        vocabulary (-1 for none) is a forbidden one."""
        at = state.clamp(0, self.n_states).long()
        return torch.where(state < 0, state, self._following[at, token.clamp(-1, self.vocab).long()])


# ---- beam search ------------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _beam_work(groups: int, beams: int, vocab: int, width: int) -> int:
    return _lib.lib().dnatok_beam_work_bytes(groups, beams, vocab, width)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, width: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None, eos_id: Optional[int] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One step of a beam search: of all continuations of each group's beams, valued ``score + log_softmax(logits)``, the
    ``width`` best (as many as there are beams if not given).  Returns ``(scores, tokens, parents)``, float32 and int32
    [B, width], the best first: ``parents`` are the beams within the group that were continued.

    ``logits`` [B * K, V] are float32, bfloat16 or float16, a group's beams next to each other; ``scores`` float32 [B, K] are
    the beams' values so far (-inf for a beam that is none).  Equal ones are taken by beam, then by token; values are compared in
    64 bits, those of one beam by their logits.  ``finished`` bool [B, K] marks beams that have ended: their only
    continuation is ``eos_id``, at no cost.  Forbidden tokens (-inf, see :func:`process_logits`) and what is NaN are no continuations;
    where fewer than ``width`` are left, the score is -inf, the token -1 (as :meth:`TokenGrammar.advance` takes it) and the
    parent the place modulo K.  Up to 128 beams, before and after.  :func:`reorder_rows` moves the beams' states.  Without
    gradients."""
    _require_floats(logits, "logits")
    if logits.dim() != 2 or scores.dim() != 2 or scores.shape[1] == 0 or logits.shape[1] == 0:
        raise ValueError("logits must be [B * K, V] and scores [B, K]")
    device, (groups, beams), vocab = logits.device, scores.shape, logits.shape[1]
    width = beams if width is None else int(width)
    if not 1 <= width <= 128 or beams > 128:
        raise ValueError("1 to 128 beams, before and after")
    stride = _require_rows(logits, "logits", (groups * beams, vocab), logits.dtype, device)
    _require(scores, "scores", (groups, beams), torch.float32, device)
    _require(finished, "finished", (groups, beams), torch.bool, device)
    if finished is not None and (eos_id is None or not 0 <= eos_id < vocab):
        raise ValueError("finished needs an eos_id in the vocabulary")
    _forward_only("beam_select", logits, scores)
    new = torch.empty_like(scores) if width == beams else torch.empty((groups, width), dtype=torch.float32, device=device)
    tokens, parents = torch.empty((2, groups, width), dtype=torch.int32, device=device).unbind(0)
    need = _beam_work(groups, beams, vocab, width)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _run("dnatok_beam_select", device, logits.data_ptr(), stride, _DTYPES[logits.dtype], groups, beams, vocab, scores.data_ptr(),
         _ptr(finished), eos_id if finished is not None else 0, width, new.data_ptr(), tokens.data_ptr(), parents.data_ptr(), _ptr(work),
         need)
    return new, tokens, parents


def reorder_rows(tensors: Sequence[torch.Tensor], parents: torch.Tensor, *,
                 out: Optional[Sequence[torch.Tensor]] = None) -> list:
    """The rows of ``tensors``, each [B * K, ..] of any type (states of the recurrences, histories), in the order of the beams
    that :func:`beam_select` chose: row ``b * W + j`` of a result is row ``b * K + parents[b, j]``; ``parents`` int32 [B, W].
    A parent that is no beam gives zeros.  Rows are contiguous; ``out`` receives the results and shares no memory with
    the tensors, or with itself.  Without gradients."""
    tensors = list(tensors)
    if parents.dim() != 2 or not parents.is_cuda:
        raise ValueError("parents must be int32 [B, W] on the GPU")
    device, (groups, width) = parents.device, parents.shape
    _require(parents, "parents", (groups, width), torch.int32, device)
    given = out is not None
    out = list(out) if given else []
    if given and len(out) != len(tensors):
        raise ValueError("out must have as many tensors")
    if not tensors:
        return out
    beams = None
    for t in tensors:
        if t.dim() < 1 or t.device != device or t.is_complex() or not (t.is_contiguous() or t[:1].is_contiguous()):
            raise ValueError(f"tensors must be [B * K, ..] on {device} with contiguous rows")
        here = t.shape[0] // groups if groups else 1
        if (beams is not None and here != beams) or here * groups != t.shape[0]:
            raise ValueError("tensors must have as many rows as there are beams")
        beams = here
    if groups * width and not beams:
        raise ValueError("no beams to choose from")
    _forward_only("reorder_rows", *tensors, *out)
    if given:
        for t, o in zip(tensors, out):
            _require(o, "out", (groups * width, *t.shape[1:]), t.dtype, device)
        for i, o in enumerate(out):
            _require_apart("reorder_rows", o, parents, *tensors, *out[:i])
    else:
        out = [torch.empty((groups * width, *t.shape[1:]), dtype=t.dtype, device=device) for t in tensors]
    if groups * width == 0:
        return out
    rows = array.array("q")                        # dnatok_rows of include/dnatok_hip.h
    for t, o in zip(tensors, out):
        size = t.element_size()
        row = t.numel() // t.shape[0] * size
        rows.extend((t.data_ptr(), o.data_ptr(), row, t.stride(0) * size, row))
    _run("dnatok_reorder_rows", device, rows.buffer_info()[0], len(tensors), parents.data_ptr(), groups, beams, width)
    return out
