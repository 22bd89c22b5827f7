"""Model operators on the rows that the encoders write: a gated linear recurrence (training and
single steps), products with 4-bit weights, and logits on their way to the choice of a token.

Thin torch-tensor wrappers over the C ABI like :mod:`dnatok_amd.encoders`: every call runs HIP kernels of
libdnatok_hip.so on the current stream of its tensors' device, and none of them synchronises.  The
reference has no counterpart.
"""
from __future__ import annotations

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
