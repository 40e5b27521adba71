"""A key / value cache in pages: attention over it, the append to it and the operations on who holds which page
(``csrc/paged_attention.cu``, ``csrc/pages.cu``).

``k_pages`` / ``v_pages`` are ``[pages, kv_heads, page, head_dim]`` (any strides, features contiguous), ``table [rows, width]``
lists the pages of every sequence in order, with -1 behind the last, and ``lens [rows]`` counts its tokens; both are int32.  A
page may stand in several rows.  It is free when no row lists it.

The operations on pages run on the device and return new tables; nothing is read back.  What only the device can see, a page
number outside the pool or a pool without a free page, is recorded in the status word: the kernels skip such a page, and
``_native.raise_on_device_error`` raises.  CPU tensors run reference formulas with the same contracts, which raise at once.

None of this has gradients: tensors that want them, or carry a tangent, are refused, and so are torch.func transforms.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple, Union

import torch

from .. import _native as N
from . import flash, kernels

c_void_p, c_int = ctypes.c_void_p, ctypes.c_int
# (called for CUDA tensors only; looking for devices here would fix which are visible as soon as the package is imported)
_current_device, _raw_stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
_increment_version = torch._C._increment_version
_F32, _BF16, _I32 = torch.float32, torch.bfloat16, torch.int32

MAX_HEAD_DIM = 256
MAX_ROWS = 4096           # rows of a table in one call
MAX_PAGES = 1 << 19
TOO_LARGE = -4


# Arguments of the entry points, in the order and with the padding of their C structs (a ctypes.Structure takes 1.6 us to fill, a
# packed one 0.25; a step of decoding makes a call or two a layer).
_ATTN_ARGS = struct.Struct("6P 11q 8i f4x Pq P iII4x")
_APPEND_ARGS = struct.Struct("8P 8q 10i d")
_FORK_ARGS = struct.Struct("9P q 6i")
_COMPACT_ARGS = struct.Struct("5P q 3i4x")
_COPY_ARGS = struct.Struct("3P 2q 2i")

_declared = False


def _lib():
    global _declared
    lib = N.load()
    if not _declared:
        for name in ("dptb_paged_attention", "dptb_paged_append", "dptb_fork_pages", "dptb_compact_pages", "dptb_copy_pages"):
            fn = getattr(lib, name)
            fn.argtypes, fn.restype = [ctypes.c_char_p, c_void_p], c_int
        _declared = True
    return lib


def _scratch(dev: int, stream: int):
    """``splitk_workspace`` of the stream, which is what it is looked up by."""
    if not torch._C._cuda_isCurrentStreamCapturing():
        held = kernels._SPLITK_WS.get((dev, stream))
        if held is not None:
            return held[0], held[1]
    return kernels.splitk_workspace(torch.device("cuda", dev))


# ------------------------------------------------------------------------------------------------------------ checks
def _here(what: str, first: torch.Tensor, *others) -> None:
    """One device for all, and the current one if it is a CUDA device: kernels go to its current stream."""
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on different devices ({dev} and {t.device})")
    if first.is_cuda and dev.index != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors are on {dev}, the current device is {torch.cuda.current_device()}")


def _no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradients; call it under torch.no_grad()")
    if torch._C._are_functorch_transforms_active():
        raise ValueError(f"{what} has no derivatives and is not for torch.func transforms")
    if torch.autograd.forward_ad._current_level >= 0 and any(
            t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no derivatives; a tensor carries a tangent")


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether elements may share a place: an axis that does not step over all that the smaller steps reach."""
    reach = 1
    for step, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if step < reach:
            return t.numel() > 0
        reach += (n - 1) * step
    return False


def _meets(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the stretches of memory from first to last element meet."""
    def end(t):
        return t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    return a.numel() > 0 and b.numel() > 0 and a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _ints(what: str, name: str, t: torch.Tensor, *shape) -> None:
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: {name} must be int32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} must be {list(shape)}, got {list(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{what}: {name} must have a contiguous last axis")


def _table(what: str, table: torch.Tensor) -> None:
    if table.dim() != 2:
        raise ValueError(f"{what}: the table must be [rows, width], got {list(table.shape)}")
    _ints(what, "the table", table, *table.shape)
    if table.shape[0] > MAX_ROWS:
        raise ValueError(f"{what}: at most {MAX_ROWS} rows, got {table.shape[0]}")


def _pages(what: str, k: torch.Tensor, v: torch.Tensor) -> None:
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"{what}: k_pages and v_pages must be [pages, kv_heads, page, head_dim] both, got {list(k.shape)} "
                         f"and {list(v.shape)}")
    if k.dtype not in (torch.bfloat16, torch.float32) or v.dtype != k.dtype:
        raise TypeError(f"{what}: pages must be float32 or bfloat16 both, got {k.dtype} and {v.dtype}")
    pages, heads, page, hd = k.shape
    if not 0 < hd <= MAX_HEAD_DIM or heads == 0 or page == 0 or pages > MAX_PAGES:
        raise ValueError(f"{what}: pages of {list(k.shape)}: heads of 1 to {MAX_HEAD_DIM} features, at most {MAX_PAGES} pages")
    for t in (k, v):
        if t.stride(3) != 1 and hd > 1:
            raise ValueError(f"{what}: the features of a page must be contiguous")


# ------------------------------------------------------------------------------------------------------------ attention
def paged_attention_reference(q, k_pages, v_pages, table, lens, scale=None):
    """fp32 formulas, a row at a time."""
    rows, heads, hd = q.shape
    pages, hkv, page, _ = k_pages.shape
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(rows, heads, hd, dtype=torch.float32, device=q.device)
    for r, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        held = table[r, :-(-n // page)].long()
        if n > table.shape[1] * page or bool((held < 0).any()) or bool((held >= pages).any()):
            raise ValueError(f"paged_attention: row {r} of {n} tokens lists a page that is not in the pool")
        k, v = (t[held].transpose(0, 1).reshape(hkv, -1, hd)[:, :n].float() for t in (k_pages, v_pages))
        s = q[r].float().view(hkv, heads // hkv, hd) @ k.transpose(1, 2) * scale
        out[r] = (torch.softmax(s, -1) @ v).view(heads, hd)
    return out.to(q.dtype)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per row, ``q [rows, heads, head_dim]``, over the ``lens[r]`` tokens of its pages (the new one
    among them).  Query heads share key heads in groups of ``heads // kv_heads``; a row of no tokens gives zeros.  bf16 or fp32, one type for all; sums in
    fp32.  ``scale`` is ``head_dim ** -0.5`` unless given.  Returns ``[rows, heads, head_dim]``: ``out``, if given, which may lie over the
    queries or any other argument."""
    dev = q.get_device()
    sizes = None if dev < 0 or out is not None else _attention_sizes(q, k_pages, v_pages, table, lens, dev)
    if sizes is None:
        _check_attention(q, k_pages, v_pages, table, lens, out)
        if dev < 0:
            o = paged_attention_reference(q, k_pages, v_pages, table, lens, scale)
            return o if out is None else out.copy_(o)
        if q.stride(2) != 1 and q.shape[2] > 1:
            q = q.contiguous()
        sizes = q.shape, k_pages.shape, table.shape[1], q.stride(), k_pages.stride(), v_pages.stride(), table.stride(0), q.dtype
    (rows, heads, hd), (pages, hkv, page, _), width, (q_row, q_head, _), (kp, kh, kt, _), (vp, vh, vt, _), t_row, dtype = sizes
    given = out
    if given is not None and (any(_meets(out, t) for t in (k_pages, v_pages, table, lens)) or _meets(out, q) and not (
            out.data_ptr() == q.data_ptr() and out.stride() == q.stride())):     # (a query itself is read before its result is written)
        out = None
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((rows, heads, hd))
        o_row, o_head = heads * hd, hd
    else:
        o_row, o_head, _ = out.stride()
    stream = _raw_stream(dev)
    ws, counters = _scratch(dev, stream)
    rc = _lib().dptb_paged_attention(_ATTN_ARGS.pack(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(),
        q_row, q_head, o_row, o_head, kp, kh, kt, vp, vh, vt, t_row,
        rows, heads, hkv, hd, page, width, pages, dtype is _F32, hd ** -0.5 if scale is None else scale,
        ws.data_ptr(), kernels.SPLITK_WS_BYTES // 4, counters.data_ptr(), kernels.SPLITK_COUNTERS, 0, 0), stream)
    if rc == TOO_LARGE:
        raise ValueError(f"paged_attention: {rows} rows of up to {width * page} tokens and {heads} heads in one call are too many")
    N.check(rc, "paged_attention")
    if given is not None:
        if given is not out:
            return given.copy_(out)
        _increment_version((out,))
    return out


def _attention_sizes(q, k_pages, v_pages, table, lens, dev):
    """Shapes and strides of a call without ``out`` that has all that ``_check_attention`` asks for, which takes longer; else None."""
    q_shape, k_shape, t_shape, dtype = q.shape, k_pages.shape, table.shape, q.dtype
    if len(q_shape) != 3 or len(k_shape) != 4 or len(t_shape) != 2 or v_pages.shape != k_shape:
        return None
    (rows, heads, hd), (pages, hkv, page, k_hd), (t_rows, width) = q_shape, k_shape, t_shape
    q_by, k_by, v_by, (t_row, t_one) = q.stride(), k_pages.stride(), v_pages.stride(), table.stride()
    if ((dtype is _BF16 or dtype is _F32) and k_pages.dtype is dtype and v_pages.dtype is dtype and
            table.dtype is _I32 and lens.dtype is _I32 and k_hd == hd and t_rows == rows and lens.shape == (rows,) and
            0 < hd <= MAX_HEAD_DIM and 0 < hkv and heads % hkv == 0 and 0 < page and pages <= MAX_PAGES and rows <= MAX_ROWS and
            q_by[2] == 1 and k_by[3] == 1 and v_by[3] == 1 and (t_one == 1 or width <= 1) and (rows <= 1 or lens.stride(0) == 1) and
            k_pages.get_device() == dev and v_pages.get_device() == dev and table.get_device() == dev and
            lens.get_device() == dev and _current_device() == dev and flash._raw_call() and
            not (torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad))):
        return q_shape, k_shape, width, q_by, k_by, v_by, t_row, dtype
    return None


def _check_attention(q, k_pages, v_pages, table, lens, out) -> None:
    what = "paged_attention"
    _pages(what, k_pages, v_pages)
    _table(what, table)
    if q.dim() != 3 or q.shape[0] != table.shape[0] or q.shape[2] != k_pages.shape[3] or q.shape[1] % k_pages.shape[1]:
        raise ValueError(f"{what}: queries {list(q.shape)} do not go with a table of {list(table.shape)} and pages of "
                         f"{list(k_pages.shape)}")
    if q.dtype != k_pages.dtype:
        raise TypeError(f"{what}: queries are {q.dtype}, pages {k_pages.dtype}")
    rows, heads, hd = q.shape
    _ints(what, "lens", lens, rows)
    _here(what, q, k_pages, v_pages, table, lens, out)
    _no_grad(what, q, k_pages, v_pages, out)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 and hd > 1):
        raise ValueError(f"{what}: out must be {list(q.shape)} {q.dtype} with contiguous features")
    if out is not None and _overlaps_itself(out):
        raise ValueError(f"{what}: places of out {list(out.shape)} with strides {list(out.stride())} overlap")


# ------------------------------------------------------------------------------------------------------------ append
def paged_append_reference(qkv, k_pages, v_pages, table, positions, heads, rows, rotary_dim, rope_base):
    pages, hkv, page, hd = k_pages.shape
    x = qkv.reshape(-1, heads + 2 * hkv, hd)
    half = rotary_dim // 2
    pos = positions.double()
    angle = pos[:, None] * rope_base ** (-2.0 * torch.arange(half, dtype=torch.float64, device=x.device) / max(rotary_dim, 1))
    angle = torch.where(pos[:, None] >= 0, angle, 0.0)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    y = x.clone()
    a, b = x[:, :heads + hkv, :half].float(), x[:, :heads + hkv, half:rotary_dim].float()
    y[:, :heads + hkv, :half] = (a * cos - b * sin).to(x.dtype)
    y[:, :heads + hkv, half:rotary_dim] = (b * cos + a * sin).to(x.dtype)
    for t, p in enumerate(positions.tolist()):
        if p < 0:
            continue
        r = t if rows is None else int(rows[t])
        at = int(table[r, p // page]) if 0 <= r < table.shape[0] and p // page < table.shape[1] else -1
        if not 0 <= at < pages:
            raise ValueError(f"paged_append: token {t} has no page at position {p} of row {r}")
        k_pages[at, :, p % page] = y[t, heads:heads + hkv]
        v_pages[at, :, p % page] = y[t, heads + hkv:]
    return y[:, :heads].contiguous(), y[:, heads:heads + hkv].contiguous()


def paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
                 heads: int, rows: Optional[torch.Tensor] = None, rotary_dim: Optional[int] = None, rope_base: float = 10000.0,
                 keys: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Keys and values of a projection output ``qkv [tokens, (heads + 2 kv_heads) head_dim]`` to their places in the pages: token
    ``t`` is token ``positions[t]`` of row ``rows[t]`` (of row ``t`` without ``rows``); int32.  A negative position is padding
    and writes nothing.  Queries and keys are turned by the half-split rotary embedding over ``rotary_dim`` features (all of
    them unless given; 0: not at all).  Returns the turned queries ``[tokens, heads, head_dim]``, and with ``keys`` the turned keys
    too; ``qkv``, which shares no memory with the pages, stays as it is.  No two tokens may have one place."""
    dev, rotary = qkv.get_device(), k_pages.shape[-1] if rotary_dim is None else rotary_dim
    sizes = None if dev < 0 else _append_sizes(qkv, k_pages, v_pages, table, positions, heads, rows, rotary, rope_base, dev)
    if sizes is None:
        _check_append(qkv, k_pages, v_pages, table, positions, heads, rows, rotary, rope_base)
        if dev < 0:
            q, k = paged_append_reference(qkv, k_pages, v_pages, table, positions, heads, rows, rotary, rope_base)
            return (q, k) if keys else q
        if qkv.stride(1) != 1:
            qkv = qkv.contiguous()
        sizes = qkv.shape[0], k_pages.shape, table.shape, qkv.stride(0), k_pages.stride(), v_pages.stride(), table.stride(0), qkv.dtype
    tokens, (pages, hkv, page, hd), (table_rows, width), x_row, (kp, kh, kt, _), (vp, vh, vt, _), t_row, dtype = sizes
    q = qkv.new_empty((tokens, heads, hd))
    k = qkv.new_empty((tokens, hkv, hd)) if keys else None
    N.check(_lib().dptb_paged_append(_APPEND_ARGS.pack(
        qkv.data_ptr(), q.data_ptr(), k.data_ptr() if keys else 0, k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(),
        positions.data_ptr(), 0 if rows is None else rows.data_ptr(), x_row, kp, kh, kt, vp, vh, vt, t_row,
        tokens, heads, hkv, hd, rotary, page, width, pages, table_rows, dtype is _F32, rope_base), _raw_stream(dev)), "paged_append")
    _increment_version((k_pages, v_pages))
    return (q, k) if keys else q


def _append_sizes(qkv, k_pages, v_pages, table, positions, heads, rows, rotary, rope_base, dev):
    """Shapes and strides of a call that has all that ``_check_append`` asks for, which takes longer, and pages in one of the usual orders;
    else None."""
    x_shape, k_shape, t_shape, dtype = qkv.shape, k_pages.shape, table.shape, qkv.dtype
    if len(x_shape) != 2 or len(k_shape) != 4 or len(t_shape) != 2 or v_pages.shape != k_shape:
        return None
    (tokens, features), (pages, hkv, page, hd), (table_rows, width) = x_shape, k_shape, t_shape
    (x_row, x_one), k_by, v_by, (t_row, t_one) = qkv.stride(), k_pages.stride(), v_pages.stride(), table.stride()
    kp, kh, kt, k_one = k_by
    if ((dtype is _BF16 or dtype is _F32) and k_pages.dtype is dtype and v_pages.dtype is dtype and table.dtype is _I32 and
            positions.dtype is _I32 and positions.shape == (tokens,) and (tokens <= 1 or positions.stride(0) == 1) and
            0 < hd <= MAX_HEAD_DIM and 0 < hkv and 0 < page and pages <= MAX_PAGES and table_rows <= MAX_ROWS and
            (kt >= hd and kh >= (page - 1) * kt + hd or kh >= hd and kt >= (hkv - 1) * kh + hd) and
            kp >= (hkv - 1) * kh + (page - 1) * kt + hd and v_by == k_by and
            heads > 0 and features == (heads + 2 * hkv) * hd and 0 <= rotary <= hd and rotary % 2 == 0 and rope_base > 0 and
            x_one == 1 and k_one == 1 and (t_one == 1 or width <= 1) and
            k_pages.get_device() == dev and v_pages.get_device() == dev and table.get_device() == dev and
            positions.get_device() == dev and _current_device() == dev and
            (table_rows == tokens if rows is None else rows.dtype is _I32 and rows.shape == (tokens,) and
             rows.get_device() == dev and (tokens <= 1 or rows.stride(0) == 1)) and flash._raw_call() and
            k_pages.data_ptr() != v_pages.data_ptr() and            # (that transforms' wrappers do not have)
            not (torch.is_grad_enabled() and (qkv.requires_grad or k_pages.requires_grad or v_pages.requires_grad))):
        return tokens, k_shape, t_shape, x_row, k_by, v_by, t_row, dtype
    return None


def _check_append(qkv, k_pages, v_pages, table, positions, heads, rows, rotary, rope_base) -> None:
    what = "paged_append"
    _pages(what, k_pages, v_pages)
    _table(what, table)
    hkv, hd = k_pages.shape[1], k_pages.shape[3]
    if rotary < 0 or rotary % 2 or rotary > hd:
        raise ValueError(f"{what}: rotary_dim must be even and in [0, {hd}], got {rotary}")
    if heads <= 0 or qkv.dim() != 2 or qkv.shape[1] != (heads + 2 * hkv) * hd:
        raise ValueError(f"{what}: qkv {list(qkv.shape)} is not [tokens, ({heads} + 2 * {hkv}) * {hd}]")
    if qkv.dtype != k_pages.dtype:
        raise TypeError(f"{what}: qkv is {qkv.dtype}, pages {k_pages.dtype}")
    if not rope_base > 0:
        raise ValueError(f"{what}: rope_base must be positive")
    tokens = qkv.shape[0]
    _ints(what, "positions", positions, tokens)
    if rows is not None:
        _ints(what, "rows", rows, tokens)
    elif tokens != table.shape[0]:
        raise ValueError(f"{what}: {tokens} tokens without `rows` for a table of {table.shape[0]} rows")
    _here(what, qkv, k_pages, v_pages, table, positions, rows)
    _no_grad(what, qkv, k_pages, v_pages)
    if _overlaps_itself(k_pages) or _overlaps_itself(v_pages) or k_pages.numel() > 0 and k_pages.data_ptr() == v_pages.data_ptr():
        raise ValueError(f"{what}: places of the pages overlap: {list(k_pages.shape)} with strides {list(k_pages.stride())} and "
                         f"{list(v_pages.stride())}")


# ------------------------------------------------------------------------------------------------------------ pages
def fork_pages_reference(table, lens, pages, page, parents, grow):
    t_in, l_in, width = table.tolist(), lens.tolist(), table.shape[1]
    who = list(range(len(t_in))) if parents is None else parents.tolist()
    more = grow.tolist() if isinstance(grow, torch.Tensor) else [grow if 0 <= p < len(l_in) and l_in[p] > 0 else 0 for p in who]
    held, old, new = [], [], []
    for p, g in zip(who, more):
        if p >= len(t_in):
            raise ValueError(f"fork_pages: parent {p} of {len(t_in)} rows")
        n = max(0, l_in[p]) if p >= 0 else 0
        row = t_in[p][:-(-n // page)] if n else []
        if n + max(g, 0) > width * page or any(not 0 <= x < pages for x in row) or len(row) < -(-n // page):
            raise ValueError(f"fork_pages: a row of {n} tokens, {g} more, in {width} pages of {page}: {row}")
        held.append(row)
        old.append(n)
        new.append(n + max(g, 0))
    grows = [b > a and a % page != 0 for a, b in zip(old, new)]
    used = {x for row in held for x in row}
    others = {x for row, g in zip(held, grows) for x in (row[:-1] if g else row)}
    free = iter([x for x in range(pages) if x not in used])
    keeper, src, dst = {}, [-1] * len(who), [-1] * len(who)
    try:
        for r, row in enumerate(held):
            row = list(row)
            if grows[r] and (row[-1] in others or keeper.setdefault(row[-1], r) != r):
                src[r], row[-1] = row[-1], next(free)
                dst[r] = row[-1]
            while len(row) * page < new[r]:
                row.append(next(free))
            held[r] = row + [-1] * (width - len(row))
    except StopIteration:
        raise ValueError(f"fork_pages: a pool of {pages} pages has no free one left") from None
    make = lambda x, *shape: torch.tensor(x, dtype=torch.int32, device=table.device).view(*shape)  # noqa: E731
    return make(held, len(who), width), make(new, -1), make(src, -1), make(dst, -1)


def fork_pages(table: torch.Tensor, lens: torch.Tensor, pages: int, page: int, parents: Optional[torch.Tensor] = None,
               grow: Union[int, torch.Tensor] = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The rows of a cache anew: row ``r`` becomes row ``parents[r]`` (itself without ``parents``; -1: empty, which frees its
    pages), longer by ``grow`` tokens: an int for every row that holds tokens, or int32 ``[rows]``, which starts empty rows as well.
    Pages of a ``pages``-page pool (``page`` tokens each) are taken for them, free ones of the lowest numbers first, row by row;
    a part-filled last page that others list too is replaced by a copy of the row's own, except for the first row that grows into it.
    Returns ``(table, lens, src, dst)``: the new table and lengths, and for every row the page to copy and its copy (-1: none), which
    ``copy_pages`` takes before anything is appended.  The old table is left as it is."""
    dev, each = table.get_device(), isinstance(grow, torch.Tensor)
    if dev < 0 or _fork_is_off(table, lens, pages, page, parents, grow, each, dev):
        _check_fork(table, lens, pages, page, parents, grow, each)
        if dev < 0:
            return fork_pages_reference(table, lens, pages, page, parents, grow)
    rows_in, width = table.shape
    rows = rows_in if parents is None else parents.shape[0]
    new_table = torch.empty_like(table) if rows == rows_in and table.is_contiguous() else table.new_empty((rows, width))
    like = lens if parents is None else parents
    new_lens, src, dst = torch.empty_like(like), torch.empty_like(like), torch.empty_like(like)
    stream = _raw_stream(dev)
    N.check(_lib().dptb_fork_pages(_FORK_ARGS.pack(
        table.data_ptr(), lens.data_ptr(), 0 if parents is None else parents.data_ptr(), grow.data_ptr() if each else 0,
        new_table.data_ptr(), new_lens.data_ptr(), src.data_ptr(), dst.data_ptr(), _scratch(dev, stream)[0].data_ptr(), table.stride(0),
        rows_in, rows, width, pages, page, 0 if each else grow), stream), "fork_pages")
    return new_table, new_lens, src, dst


def _fork_is_off(table, lens, pages, page, parents, grow, each, dev) -> bool:
    """Whether ``_check_fork`` has to look : everything it asks for, in less time."""
    if table.dim() != 2 or parents is not None and parents.dim() != 1:
        return True
    rows_in = table.shape[0]
    rows = rows_in if parents is None else parents.shape[0]
    return not (
        table.dtype is _I32 and lens.dtype is _I32 and lens.shape == (rows_in,) and rows_in <= MAX_ROWS and rows <= MAX_ROWS and
        0 <= pages <= MAX_PAGES and 0 < page and (table.stride(1) == 1 or table.shape[1] <= 1) and (rows_in <= 1 or lens.stride(0) == 1) and
        (parents is None or parents.dtype is _I32 and parents.get_device() == dev and (rows <= 1 or parents.stride(0) == 1)) and
        (grow.dtype is _I32 and grow.shape == (rows,) and grow.get_device() == dev and (rows <= 1 or grow.stride(0) == 1) if each
         else 0 <= grow < 1 << 31) and lens.get_device() == dev and _current_device() == dev)


def _check_fork(table, lens, pages, page, parents, grow, each) -> None:
    what = "fork_pages"
    _table(what, table)
    rows_in = table.shape[0]
    _ints(what, "lens", lens, rows_in)
    rows = rows_in if parents is None else parents.numel()
    if parents is not None:
        _ints(what, "parents", parents, rows)
    if each:
        _ints(what, "grow", grow, rows)
    elif not 0 <= grow < 1 << 31:
        raise ValueError(f"{what}: rows grow by 0 or more tokens, got {grow}")
    if rows > MAX_ROWS or not 0 <= pages <= MAX_PAGES or page <= 0:
        raise ValueError(f"{what}: {rows} rows (at most {MAX_ROWS}), {pages} pages (at most {MAX_PAGES}) of {page} tokens")
    _here(what, table, lens, parents, grow if each else None)


def compact_pages_reference(table, pages):
    held = sorted({p for p in table.flatten().tolist() if p >= 0})
    if held and held[-1] >= pages:
        raise ValueError(f"compact_pages: page {held[-1]} of a pool of {pages}")
    live, on = len(held), set(held)
    moves = dict(zip([p for p in held if p >= live], [p for p in range(live) if p not in on]))
    make = lambda x: torch.tensor(x, dtype=torch.int32, device=table.device)  # noqa: E731
    new = make([moves.get(p, p) if p >= 0 else -1 for p in table.flatten().tolist()]).view(table.shape)
    blank = [-1] * (pages // 2 - len(moves))
    return new, make(list(moves) + blank), make(list(moves.values()) + blank), make([live])


def compact_pages(table: torch.Tensor, pages: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``n`` listed pages of a pool numbered 0 to ``n - 1``: those numbered ``n`` and above move, in order, to the unlisted
    numbers below.  Returns ``(table, src, dst, live)``: the table in the new numbers, the moves (``[pages // 2]``, -1 behind
    the last) for ``copy_pages``, and ``n`` as an int32 ``[1]``."""
    dev = table.get_device()
    if dev < 0 or _compact_is_off(table, pages, dev):
        _check_compact(table, pages)
        if dev < 0:
            return compact_pages_reference(table, pages)
    rows, width = table.shape
    new = torch.empty_like(table) if table.is_contiguous() else table.new_empty((rows, width))
    live = table.new_empty((1,))
    src = table.new_empty((pages // 2,))
    dst = torch.empty_like(src)
    N.check(_lib().dptb_compact_pages(_COMPACT_ARGS.pack(
        table.data_ptr(), new.data_ptr(), src.data_ptr(), dst.data_ptr(), live.data_ptr(), table.stride(0), rows, width, pages),
        _raw_stream(dev)), "compact_pages")
    return new, src, dst, live


def _compact_is_off(table, pages, dev) -> bool:
    return not (table.dim() == 2 and table.dtype is _I32 and table.shape[0] <= MAX_ROWS and 0 <= pages <= MAX_PAGES and
                (table.stride(1) == 1 or table.shape[1] <= 1) and _current_device() == dev)


def _check_compact(table, pages) -> None:
    _table("compact_pages", table)
    if not 0 <= pages <= MAX_PAGES:
        raise ValueError(f"compact_pages: a pool of {pages} pages (at most {MAX_PAGES})")
    _here("compact_pages", table)


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """In place: page ``dst[i]`` of ``pool [..., pages, kv_heads, page, head_dim]`` (contiguous; every layer's keys and values at
    once) becomes a copy of page ``src[i]``; pairs with a -1 are passed over.  A page that is copied to must be in no other pair."""
    dev, shape = pool.get_device(), pool.shape
    if dev < 0 or _copy_is_off(pool, src, dst, dev):
        _check_copy(pool, src, dst)
    pages = shape[-4]
    outer = math.prod(shape[:-4])
    if dev < 0:
        real = (src >= 0) & (dst >= 0)
        x, y = src[real].long(), dst[real].long()
        if bool((x >= pages).any()) or bool((y >= pages).any()):
            raise ValueError(f"copy_pages: a page outside the pool of {pages}")
        flat = pool.view(outer, pages, -1)
        flat[:, y] = flat[:, x]
        return
    if outer > 65535:
        raise ValueError(f"copy_pages: at most 65535 pools at once, got {outer}")
    N.check(_lib().dptb_copy_pages(_COPY_ARGS.pack(
        pool.data_ptr(), src.data_ptr(), dst.data_ptr(), outer, shape[-3] * shape[-2] * shape[-1] * pool.element_size(),
        src.shape[0], pages), _raw_stream(dev)), "copy_pages")
    _increment_version((pool,))


def _copy_is_off(pool, src, dst, dev) -> bool:
    return not (
        pool.dim() >= 4 and pool.is_contiguous() and (pool.dtype is _BF16 or pool.dtype is _F32) and src.dim() == 1 and
        src.dtype is _I32 and dst.dtype is _I32 and src.shape == dst.shape and src.get_device() == dev and
        dst.get_device() == dev and (src.shape[0] <= 1 or src.stride(0) == 1 and dst.stride(0) == 1) and
        _current_device() == dev and flash._raw_call() and not (pool.requires_grad and torch.is_grad_enabled()))


def _check_copy(pool, src, dst) -> None:
    what = "copy_pages"
    if pool.dim() < 4 or not pool.is_contiguous():
        raise ValueError(f"{what}: the pool must be a contiguous [..., pages, kv_heads, page, head_dim], got {list(pool.shape)}")
    if pool.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: pages must be float32 or bfloat16, got {pool.dtype}")
    if src.dim() != 1:
        raise ValueError(f"{what}: src and dst must be lists of pages")
    _ints(what, "src", src, *src.shape)
    _ints(what, "dst", dst, *src.shape)
    _here(what, pool, src, dst)
    _no_grad(what, pool)
