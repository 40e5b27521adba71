"""Beam search's selection over beams and vocabulary (``csrc/beam.cu``).  CPU tensors run reference formulas."""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple

import torch

from .. import _native as N
from . import flash
from .kernels import SPLITK_COUNTERS, SPLITK_WS_BYTES
from .paged import _BF16, _F32, _current_device, _here, _no_grad, _raw_stream, _scratch

c_void_p, c_int = ctypes.c_void_p, ctypes.c_int

MAX_BEAMS = 32
MAX_ROWS = 1 << 20


# The C struct's fields in order (see ops/paged.py).
_BEAM_ARGS = struct.Struct("9P 2q 10i")

_declared = False


def _lib():
    global _declared
    lib = N.load()
    if not _declared:
        lib.dptb_beam_step.argtypes, lib.dptb_beam_step.restype = [ctypes.c_char_p, c_void_p], c_int
        _declared = True
    return lib


def beam_step_reference(logits, scores, finished=None, eos=-1):
    """64-bit formulas over all continuations, sorted by value, then by beam, and within a beam by logit and token."""
    items, beams = scores.shape
    x = logits.double().view(items, beams, -1)
    vocab = x.shape[-1]
    ids = torch.arange(vocab, device=x.device)
    lp = torch.log_softmax(x, -1)
    start = scores.double()[..., None]
    fine = lp.isfinite().any(-1, keepdim=True) & ~lp.isnan().any(-1, keepdim=True) & start.isfinite()
    total = torch.where(fine, start + lp, -math.inf)
    if finished is not None:
        only = torch.where((ids == eos) & start.isfinite(), start, -math.inf)
        total = torch.where(finished[..., None], only, total)
        fine = fine & ~finished[..., None]
    within = torch.where(fine, torch.sort(x, dim=-1, descending=True, stable=True).indices, ids)
    total, order = torch.sort(total.gather(2, within).view(items, -1), dim=-1, descending=True, stable=True)
    total, order = total[:, :beams], order[:, :beams]
    beam, token = order // vocab, within.view(items, -1).gather(1, order)
    done = token == eos
    if finished is not None:
        done = done | finished.gather(1, beam)
    parents = beam + beams * torch.arange(items, device=x.device)[:, None]
    return total.float(), parents.int(), token, done


def beam_step(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None,
              eos: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """One step of beam search for ``items`` searches of ``beams`` beams: of all ``beams * vocab`` continuations of an item the
    best ``beams``, by ``scores [items, beams]`` (fp32) plus the log-probability that ``logits [items * beams, vocab]`` (bf16 or
    fp32) gives the token; equal ones in the order of the beams, and within a beam of the logits, then of the tokens.

    A beam of ``finished [items, beams]`` (bool) goes on with ``eos`` alone, at its old score.  A beam whose score is not finite and a
    row of logits that is no distribution (a NaN, an infinity, nothing but -inf) have continuations worth -inf only, so a search starts
    with the scores ``0, -inf, -inf, ...``.

    Returns ``(scores, parents, tokens, finished)``, each ``[items, beams]``, best first: ``parents`` (int32) are rows of ``logits``,
    as ``fork_pages`` takes them, ``tokens`` int64.  Up to 32 beams."""
    dev, last = logits.get_device(), -1 if eos is None else eos
    if not (dev >= 0 and scores.dim() == 2 and logits.dim() == 2) or _beam_is_off(logits, scores, finished, eos, dev):
        _check_beam(logits, scores, finished, eos)
        if dev < 0:
            return beam_step_reference(logits, scores, finished, last)
        if logits.stride(1) != 1 and logits.shape[1] > 1:
            logits = logits.contiguous()
        scores = scores.contiguous()
        finished = None if finished is None else finished.contiguous()
    (items, beams), vocab = scores.shape, logits.shape[1]
    out_scores, out_parents = torch.empty_like(scores), torch.empty_like(scores, dtype=torch.int32)
    out_tokens, out_finished = torch.empty_like(scores, dtype=torch.long), torch.empty_like(scores, dtype=torch.bool)
    lib, stream = _lib(), _raw_stream(dev)
    ws, counters = _scratch(dev, stream)
    N.check(lib.dptb_beam_step(_BEAM_ARGS.pack(
        logits.data_ptr(), scores.data_ptr(), 0 if finished is None else finished.data_ptr(), out_scores.data_ptr(),
        out_parents.data_ptr(), out_tokens.data_ptr(), out_finished.data_ptr(), ws.data_ptr(), counters.data_ptr(), logits.stride(0), SPLITK_WS_BYTES,
        items, beams, vocab, last, logits.dtype is _F32, SPLITK_COUNTERS, 0, 0, 0, 0), stream), "beam_step")
    return out_scores, out_parents, out_tokens, out_finished


def _beam_is_off(logits, scores, finished, eos, dev) -> bool:
    """Whether ``_check_beam`` has to look: everything it asks for, at the price of a call on each step."""
    (items, beams), (rows, vocab) = scores.shape, logits.shape
    return not (
        scores.dtype is _F32 and (logits.dtype is _BF16 or logits.dtype is _F32) and rows == items * beams and 0 < vocab <= 1 << 30 and
        0 < beams <= MAX_BEAMS and rows <= MAX_ROWS and scores.is_contiguous() and logits.stride(1) == 1 and
        (eos is None or 0 <= eos < vocab) and scores.get_device() == dev and _current_device() == dev and
        (finished is None or eos is not None and finished.dtype is torch.bool and finished.shape == scores.shape and
         finished.get_device() == dev and finished.is_contiguous()) and flash._raw_call() and
        not ((logits.requires_grad or scores.requires_grad) and torch.is_grad_enabled()))


def _check_beam(logits, scores, finished, eos) -> None:
    what = "beam_step"
    if scores.dim() != 2 or scores.dtype != torch.float32:
        raise ValueError(f"{what}: scores must be fp32 [items, beams], got {scores.dtype} {list(scores.shape)}")
    items, beams = scores.shape
    if logits.dim() != 2 or logits.shape[0] != items * beams or logits.shape[1] == 0:
        raise ValueError(f"{what}: logits {list(logits.shape)} are not [{items} * {beams}, vocab]")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: logits must be float32 or bfloat16, got {logits.dtype}")
    if not 0 < beams <= MAX_BEAMS or items * beams > MAX_ROWS or logits.shape[1] > 1 << 30:
        raise ValueError(f"{what}: 1 to {MAX_BEAMS} beams, at most {MAX_ROWS} rows and {1 << 30} tokens, got {items} x {beams} x {logits.shape[1]}")
    if finished is not None and (finished.shape != scores.shape or finished.dtype != torch.bool):
        raise ValueError(f"{what}: finished must be bool {list(scores.shape)}")
    if eos is not None and not 0 <= eos < logits.shape[1]:
        raise ValueError(f"{what}: eos {eos} is no token of {logits.shape[1]}")
    if finished is not None and eos is None:
        raise ValueError(f"{what}: finished beams need an eos to go on with")
    _here(what, logits, scores, finished)
    _no_grad(what, logits, scores)
