"""The rules between a decoder's logits and the choice of a token, on the device.

`LogitsRules` holds what applies to each row of a batch: the tokens it has
already (repetition, frequency and presence penalties, repeated n-grams), a
row of a bias table, a row of a table of grammar masks. `process` writes the
logits after the rules; `topk` goes on to the log-probabilities of the k best
tokens without writing them (k = 1: the greedy choice). The definition is in
include/vkb200.h (vkb_logits_rules).

Tensors are torch CUDA tensors and stay the caller's: a rules object keeps them
alive and reads what they hold when a call runs, so a program makes it once and
updates the tensors in place. The work runs on the context's stream; tensors of
another stream are ordered by the caller, as for any other kernel.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check, VkbError  # noqa: F401

_L = _lib.load()
TOPK_MAX = _lib.LOGITS_TOPK_MAX


def _bad(message: str):
    raise VkbError(_lib.ERROR_INVALID_ARGUMENT, message)


def _tensor(t, name: str, dtypes, ndim: int):
    """Checks a CUDA tensor whose last axis is contiguous; returns its data pointer (None for None)."""
    if t is None:
        return None
    if not t.is_cuda:
        _bad(f"{name}: not on a CUDA device")
    if t.dtype not in dtypes:
        _bad(f"{name}: dtype {t.dtype} is not one of {', '.join(str(d) for d in dtypes)}")
    if t.dim() != ndim:
        _bad(f"{name}: {t.dim()} axes where {ndim} are wanted")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        _bad(f"{name}: its last axis must be contiguous")
    return t.data_ptr()


def _device(tensors) -> int | None:
    """The GPU that all of these (None among them) are on; None where there is no tensor."""
    on = {t.get_device() for t in tensors if t is not None}
    if len(on) > 1:
        _bad(f"tensors of one call on different GPUs: {sorted(on)}")
    return on.pop() if on else None


def _at_home(ctx, device, name: str):
    """Refuses tensors of another GPU than the context's."""
    if device is not None and device != ctx.device:
        _bad(f"{name}: on GPU {device}, the context is on GPU {ctx.device}")


def _ld(t) -> int:
    """The stride between rows, in elements; at least a row where there is one row only (its stride says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class LogitsRules:
    """What applies to the rows of a batch; everything is optional.

    history int32 [rows, n] and history_len int32 [rows]: token ids of each row;
    repetition, frequency, presence f32 [rows]; no_repeat_ngram: n (0 = off);
    bias f32 [n_bias, vocab] with bias_row int32 [rows] (None: row 0; -1: none);
    mask int32 or uint32 [n_mask, ceil(vocab / 32)] with mask_row int32 [rows]."""

    def __init__(self, history=None, history_len=None, repetition=None, frequency=None, presence=None,
                 no_repeat_ngram: int = 0, bias=None, bias_row=None, mask=None, mask_row=None):
        i32, f32 = (torch.int32,), (torch.float32,)
        self.tensors = (history, history_len, repetition, frequency, presence, bias, bias_row, mask, mask_row)
        s = _lib.LogitsRules()
        s.hist = _tensor(history, "history", i32, 2)
        s.hist_ld = 0 if history is None else _ld(history) if history.shape[1] else 0
        if history is not None and s.hist_ld < history.shape[1]:
            _bad("history: its rows overlap")
        s.hist_cols = 0 if history is None else history.shape[1]
        s.hist_len = _tensor(history_len, "history_len", i32, 1)
        s.repetition = _tensor(repetition, "repetition", f32, 1)
        s.frequency = _tensor(frequency, "frequency", f32, 1)
        s.presence = _tensor(presence, "presence", f32, 1)
        s.no_repeat_ngram = int(no_repeat_ngram)
        s.bias = _tensor(bias, "bias", f32, 2)
        s.bias_row = _tensor(bias_row, "bias_row", i32, 1)
        s.mask = _tensor(mask, "mask", (torch.int32, torch.uint32), 2)
        s.mask_row = _tensor(mask_row, "mask_row", i32, 1)
        if bias is not None:
            s.n_bias, s.bias_ld = bias.shape[0], _ld(bias)
        if mask is not None:
            s.n_mask, s.mask_ld = mask.shape[0], _ld(mask)
        self._per_row = [(n, t) for n, t in (("history", history), ("history_len", history_len), ("repetition", repetition),
                                             ("frequency", frequency), ("presence", presence), ("bias_row", bias_row),
                                             ("mask_row", mask_row)) if t is not None]
        self._bias_width = None if bias is None else bias.shape[1]
        self._mask_words = None if mask is None else mask.shape[1]
        self._checked = None
        self.device = _device(self.tensors)
        self.struct = s
        self.ref = C.byref(s)

    def check(self, rows: int, vocab: int, device: int | None = None):
        """Whether the rules fit a batch of this shape, on this GPU (None: whichever they are on)."""
        if self._checked == (rows, vocab, device):
            return
        if device is not None and self.device is not None and self.device != device:
            _bad(f"rules: on GPU {self.device}, the context is on GPU {device}")
        for name, t in self._per_row:
            if t.shape[0] < rows:
                _bad(f"{name}: {t.shape[0]} rows for {rows} rows of logits")
        if self._bias_width is not None and self._bias_width < vocab:
            _bad(f"bias: rows of {self._bias_width} values for a vocabulary of {vocab}")
        if self._mask_words is not None and self._mask_words < (vocab + 31) // 32:
            _bad(f"mask: rows of {self._mask_words} words for a vocabulary of {vocab}")
        self._checked = (rows, vocab, device)


_DTYPES = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16}


def _matrix(t, name: str):
    """(pointer, dtype code, rows, columns, row stride) of an f32 or f16 CUDA matrix with contiguous rows."""
    dt = _DTYPES.get(t.dtype)
    if dt is None or not t.is_cuda or t.dim() != 2:
        _tensor(t, name, tuple(_DTYPES), 2)
    rows, cols = t.shape
    ld, unit = t.stride()
    if unit != 1 and cols > 1:
        _bad(f"{name}: its last axis must be contiguous")
    return t.data_ptr(), dt, rows, cols, ld if rows > 1 else cols


def process(ctx, logits, rules: LogitsRules | None = None, out=None):
    """The logits ([rows, vocab], f32 or f16) after the rules, in their own type; out may be logits."""
    p, dt, rows, vocab, ld = _matrix(logits, "logits")
    if logits.get_device() != ctx.device:
        _at_home(ctx, logits.get_device(), "logits")
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        to, out_ld = out.data_ptr(), vocab
    else:
        to, out_dt, out_rows, out_vocab, out_ld = _matrix(out, "out")
        if (out_rows, out_vocab, out_dt) != (rows, vocab, dt):
            _bad("out: another shape or dtype than logits")
        _at_home(ctx, out.get_device(), "out")
    ref = None
    if rules is not None:
        if rules._checked != (rows, vocab, ctx.device):
            rules.check(rows, vocab, ctx.device)
        ref = rules.ref
    status = _L.vkb_logits_process(ctx.h, p, dt, rows, vocab, ld, ref, to, out_ld)
    if status:
        check(status)
    return out


def topk(ctx, logits, k: int, rules: LogitsRules | None = None, ids=None, logprobs=None):
    """(ids int32 [rows, k], log-probabilities f32 [rows, k]) of the k best tokens after the rules, the
    best first, ties by the lower id; id -1 at -inf where fewer than k tokens are left."""
    p, dt, rows, vocab, ld = _matrix(logits, "logits")
    if logits.get_device() != ctx.device:
        _at_home(ctx, logits.get_device(), "logits")
    if not 1 <= k <= TOPK_MAX:
        _bad(f"k must be in 1..{TOPK_MAX}, got {k}")
    for t, name, dtype in ((ids, "ids", torch.int32), (logprobs, "logprobs", torch.float32)):
        if t is not None and (t.dtype != dtype or tuple(t.shape) != (rows, k) or not t.is_contiguous() or not t.is_cuda):
            _bad(f"{name}: a contiguous {dtype} CUDA tensor of shape [{rows}, {k}] is wanted")
        if t is not None:
            _at_home(ctx, t.get_device(), name)
    if ids is None:
        ids = torch.empty((rows, k), dtype=torch.int32, device=logits.device)
    if logprobs is None:
        logprobs = torch.empty((rows, k), dtype=torch.float32, device=logits.device)
    ref = None
    if rules is not None:
        if rules._checked != (rows, vocab, ctx.device):
            rules.check(rows, vocab, ctx.device)
        ref = rules.ref
    status = _L.vkb_logits_topk(ctx.h, p, dt, rows, vocab, ld, ref, k, ids.data_ptr(), logprobs.data_ptr())
    if status:
        check(status)
    return ids, logprobs
