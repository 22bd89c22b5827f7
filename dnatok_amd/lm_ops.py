"""Model operators on the rows that the encoders write: a gated linear recurrence (training and
single steps), products with 4-bit weights, and logits on their way to the choice of a token.

Thin torch-tensor wrappers over the C ABI like :mod:`dnatok_amd.encoders`: every call runs HIP kernels of
libdnatok_hip.so on the current stream of its tensors' device, and none of them synchronises.  The
reference has no counterpart.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_NO_GUARD = contextlib.nullcontext()


def _stream(device: torch.device) -> int:
    # (see encoders._stream: the raw handle is much cheaper than the Stream object)
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _on(device: torch.device):
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _require_rows(t: torch.Tensor, name: str, shape, dtype: torch.dtype, device: torch.device) -> int:
    """A matrix whose rows' elements lie next to each other; returns the elements between rows."""
    if t.device != device or t.dtype != dtype or t.shape != shape or not (t.stride(-1) == 1 or t.shape[-1] == 1):
        raise ValueError(f"{name} must be a {dtype} tensor {tuple(shape)} on {device} with contiguous rows")
    return t.stride(0)


def _require(t: Optional[torch.Tensor], name: str, shape, dtype: torch.dtype, device: torch.device) -> None:
    if t is not None and (t.device != device or t.dtype != dtype or t.shape != shape or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {device}")


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
        with _on(device):
            _lib.check(L.dnatok_gated_scan_backward(
                x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0), code, _ptr(offsets), ctx.n_rows, total, dim,
                int(ctx.reverse), _ptr(h0), _ptr(dy), 0 if dy is None else dy.stride(0), _ptr(dlast), states.data_ptr(),
                dx.data_ptr(), dgate.data_ptr(), _ptr(dh0), _ptr(work), need, _stream(device)),
                "dnatok_gated_scan_backward")
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
    with _on(device):
        _lib.check(L.dnatok_gated_scan(
            x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0), code, _ptr(offsets), n_rows, total, dim,
            int(reverse), _ptr(h0), y.data_ptr(), last.data_ptr(), _ptr(states), _ptr(work), need, _stream(device)),
            "dnatok_gated_scan")
    return y, last, states


def gated_scan(x: torch.Tensor, gate: torch.Tensor, offsets: Optional[torch.Tensor] = None, *,
               h0: Optional[torch.Tensor] = None, reverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence ``h_t = f_t h_(t-1) + (1 - f_t) x_t`` with ``f = sigmoid(gate)``, in every channel of
    every row.  Returns ``(y, last)``: the states in x's type and shape, and the state behind each row's last
    step, float32 [B, D].

    ``x`` and ``gate`` are packed rows [total, D] with ``offsets`` int64 [B + 1] as the encoders write
    them (rows may be empty), or dense rows [B, T, D] without offsets; float32, bfloat16 or float16, the elements of
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
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, gate, offsets, n_rows, h0, reverse)
    return _scan_forward(x, gate, offsets, n_rows, h0, reverse, False)[:2]


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: Optional[torch.Tensor] = None, *,
               out_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of :func:`gated_scan` for one token of each row: ``x`` and ``gate`` [B, D], ``state``
    float32 [B, D] (zero if not given).  Returns ``(y, new_state)``; ``out_state`` receives the new state and may be
    ``state`` itself.  Without gradients."""
    _require_floats(x, "x")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError("x must be [B, D]")
    device = x.device
    xs = _require_rows(x, "x", x.shape, x.dtype, device)
    gs = _require_rows(gate, "gate", x.shape, x.dtype, device)
    _require(state, "state", x.shape, torch.float32, device)
    _require(out_state, "out_state", x.shape, torch.float32, device)
    _forward_only("gated_step", x, gate, state)
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    if out_state is None:
        out_state = torch.empty(x.shape, dtype=torch.float32, device=device)
    with _on(device):
        _lib.check(_lib.lib().dnatok_gated_step(x.data_ptr(), xs, gate.data_ptr(), gs, _DTYPES[x.dtype], _ptr(state),
                                                x.shape[0], x.shape[1], y.data_ptr(), out_state.data_ptr(),
                                                _stream(device)), "dnatok_gated_step")
    return y, out_state


def _forward_only(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward pass: call it under torch.no_grad()")


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
        float32.  Without gradients."""
        squeeze = x.dim() == 1
        if squeeze:
            x = x.unsqueeze(0)
        if x.dim() != 2:
            raise ValueError("x must be [M, K] or [K]")
        device = self.scales.device
        m, n, k = x.shape[0], self.out_features, self.in_features
        xs = _require_rows(x, "x", (m, k), self.scales.dtype, device)
        _require(bias, "bias", (n,), torch.float32, device)
        _forward_only("W4Matrix.matvec", x, bias)
        if out_dtype is None:
            out_dtype = x.dtype if out is None else out.dtype
        if out_dtype not in (x.dtype, torch.float32):
            raise ValueError("out_dtype must be x's type or float32")
        if out is None:
            out = torch.empty((m, n), dtype=out_dtype, device=device)
        elif squeeze:
            out = out.unsqueeze(0)
        ys = _require_rows(out, "out", (m, n), out_dtype, device)
        with _on(device):
            _lib.check(_lib.lib().dnatok_w4_matvec(
                x.data_ptr(), xs, _DTYPES[x.dtype], self.q.data_ptr(), self.q.stride(0), self.scales.data_ptr(),
                _ptr(self.zeros), m, n, k, self.group, _ptr(bias), out.data_ptr(), ys, _DTYPES[out_dtype],
                _stream(device)), "dnatok_w4_matvec")
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
    _forward_only("process_logits", logits, bias)
    if out_dtype is None:
        out_dtype = logits.dtype if out is None else out.dtype
    if out_dtype not in (logits.dtype, torch.float32):
        raise ValueError("out_dtype must be the logits' type or float32")
    if out is None:
        out = torch.empty((rows, vocab), dtype=out_dtype, device=device)
    out_stride = _require_rows(out, "out", (rows, vocab), out_dtype, device)
    repetition = _per_row(repetition, "repetition", rows, device)
    presence = _per_row(presence, "presence", rows, device)
    frequency = _per_row(frequency, "frequency", rows, device)
    with _on(device):
        _lib.check(_lib.lib().dnatok_logits_process(
            logits.data_ptr(), stride, _DTYPES[logits.dtype], rows, vocab, _ptr(history), _ptr(history_offsets),
            _ptr(prompt_lengths), _ptr(repetition), _ptr(presence), _ptr(frequency), _ptr(bias), bias_stride,
            _ptr(allowed), allowed_stride, n_states, _ptr(state), out.data_ptr(), out_stride, _DTYPES[out_dtype],
            _stream(device)), "dnatok_logits_process")
    return out
