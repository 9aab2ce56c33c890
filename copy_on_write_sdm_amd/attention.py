"""The attention layers of a stack on the device: whole prompts, and single
tokens over a paged cache held in 8 bits.

The reference runs its attention layers in its model (CausalSelfAttention,
copy_on_write_sdm/model.py:47-189) over a dense K/V cache in the activations'
type; ``prefill_faithful_sdm_stack`` and ``decode_faithful_sdm_stack`` take
them as the caller's callables.  These are the operators such a callable
needs:

* ``prompt_attention``    causal attention over packed prompts of different
                          lengths, with grouped heads;
* ``extend_page_tables``  the page tables and token slots of a step, from the
                          requests' lengths and new tokens;
* ``write_kv_cache``      keys and values into their slots, in 8 bits;
* ``cached_attention``    each request's newest tokens over the cache.

A page holds ``page_tokens`` tokens of one request in one layer: keys as
[pages, heads, page_tokens, width], values transposed, [pages, heads, width,
page_tokens], in float8 (e4m3), with one power of two for each page and head
by which the codes count, [pages, heads].  The width is a head's, padded with
zeros to 32, 64, 96, 128, 192 or 256 (``cache_width``).

Kernels: csrc/prompt_attention.hip and csrc/kv_cache.hip.  Float32, float16
and bfloat16; there is no backward pass (inputs that require a gradient are
refused, where gradients are recorded) and no CPU path.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Sequence

import torch

from . import _native as nat

CODES = torch.float8_e4m3fn
_INT32, _FLOAT32 = torch.int32, torch.float32
MAX_REQUESTS = 4_096
_FAR = 1 << 23        # elements between rows from which prompts are copied
PAGE_TOKENS = (16, 32, 64, 128, 256)
CACHE_WIDTHS = (32, 64, 96, 128, 192, 256)


_PADDED = {w: next(c for c in CACHE_WIDTHS if c >= w) for w in range(8, 257, 8)}


def cache_width(head_width: int) -> int:
    """The row width of a cache for heads of ``head_width``."""

    padded = _PADDED.get(head_width)
    if padded is None:
        raise ValueError("attention head width must be a multiple of 8, at most 256")
    return padded


def _need_device(tensor: torch.Tensor, what: str) -> None:
    if not tensor.is_cuda:
        raise RuntimeError(f"{what} must be on the GPU: the attention kernels have no CPU path")


def _need_no_gradient(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any([t.requires_grad for t in tensors]):
        raise RuntimeError("the attention operators have no backward pass: call them under "
                           "torch.no_grad(), or with detached inputs")


def _float_type(dtype: torch.dtype) -> int:
    code = nat.FLOAT_TYPES.get(dtype)
    if code is None:
        raise TypeError("attention takes float32, float16 or bfloat16")
    return code


def _scale(scale: float | None, width: int) -> float:
    if scale is None:
        return width ** -0.5
    if not 0.0 < scale < math.inf:
        raise ValueError("the attention scale must be positive")
    return scale


def _rows(tensor: torch.Tensor, step: int, far: float = math.inf
          ) -> tuple[torch.Tensor, int, tuple[int, ...]]:
    """``tensor``, its address and its strides where its rows can be loaded 16
    bytes (``step`` elements) at a time, as a slice of a fused projection can,
    and lie less than ``far`` elements apart; else those of a contiguous copy."""

    strides, address = tensor.stride(), tensor.data_ptr()
    together = 0
    for s in strides[:-1]:
        together |= s
    if strides[-1] == 1 and not together % step and not address % 16 and strides[0] < far:
        return tensor, address, strides
    copy = tensor.contiguous()
    if copy.data_ptr() % 16:        # contiguous as it was, only its address is odd
        copy = copy.clone()
    # of its sizes, not its own: a tensor is contiguous whatever the strides of
    # its axes of one element
    strides = [1]
    for size in reversed(copy.shape[1:]):
        strides.append(strides[-1] * size)
    return copy, copy.data_ptr(), tuple(reversed(strides))


def _int32(tensor: torch.Tensor, numbers: int, device: int, what: str) -> None:
    if tensor.dtype is not _INT32 or tensor.numel() != numbers or not tensor.is_contiguous():
        raise ValueError(f"{what} must be {numbers} contiguous int32 numbers")
    if tensor.get_device() != device:
        raise ValueError(f"{what} must be on the other inputs' device")


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                     offsets: torch.Tensor, *, longest: int | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention over packed prompts: query [T, heads, D], key and
    value [T, kv_heads, D] (any strides between rows and heads; ``heads`` a
    multiple of ``kv_heads``, query head h reads key head ``h // (heads //
    kv_heads)``), and int32 offsets [S + 1] on the device: sequence s holds
    rows offsets[s] to offsets[s + 1] - 1.  Returns [T, heads, D] in the
    query's type; rows of no sequence are zero.  ``longest`` bounds the
    sequences' lengths (T when not given) and sizes the launch: a bound that
    is too small or too large costs time, not correctness.  ``scale`` defaults
    to D ** -0.5."""

    if query.ndim != 3 or key.ndim != 3 or value.shape != key.shape:
        raise ValueError("attention takes query [T,heads,D] and key and value [T,kv_heads,D]")
    rows, heads, width = query.shape
    key_rows, kv_heads, key_width = key.shape
    if key_rows != rows or key_width != width:
        raise ValueError("attention query, key and value do not align")
    if not kv_heads or not heads or heads % kv_heads:
        raise ValueError("query heads must be a multiple of the key heads")
    cache_width(width)
    _need_no_gradient(query, key, value)
    dtype = query.dtype
    code = _float_type(dtype)
    if key.dtype is not dtype or value.dtype is not dtype:
        raise TypeError("attention query, key and value share one type")
    _need_device(query, "attention inputs")
    device, index = query.device, query.get_device()
    if key.get_device() != index or value.get_device() != index:
        raise ValueError("attention inputs must be on one device")
    sequences = offsets.numel() - 1
    if sequences < 0 or offsets.ndim != 1:
        raise ValueError("attention offsets must be a vector of sequences + 1")
    _int32(offsets, sequences + 1, index, "attention offsets")
    if longest is None:
        longest = rows
    elif longest < 0:
        raise ValueError("the longest sequence cannot be negative")
    factor = _scale(scale, width)
    if not sequences:
        return torch.zeros(rows, heads, width, device=device, dtype=dtype)
    out = query.new_empty((rows, heads, width))
    if not rows:
        return out
    step = 8 if code else 4
    query, q, (q_row, q_head, _) = _rows(query, step, _FAR)
    key, k, (k_row, k_head, _) = _rows(key, step, _FAR)
    value, v, (v_row, v_head, _) = _rows(value, step, _FAR)
    a = nat.PromptAttention(q, k, v, q_row, q_head, k_row, k_head, v_row, v_head,
                            offsets.data_ptr(), out.data_ptr(), rows, sequences, longest, heads,
                            kv_heads, width, code, factor)
    rc = nat.lib().cowsdm_prompt_attention(a, nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_prompt_attention")
    return out


class PageTableStep(NamedTuple):
    """What ``extend_page_tables`` returns, all int32 on the device: the
    requests' new lengths [B], the free pages left [1], the offsets of their
    new tokens in the packed order [B + 1], each new token's position in its
    request and its slot [tokens], and whether something ran short [1]."""

    lengths: torch.Tensor
    free_count: torch.Tensor
    offsets: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    overflow: torch.Tensor


def extend_page_tables(lengths: torch.Tensor, added: torch.Tensor, page_tables: torch.Tensor,
                       free_pages: torch.Tensor, free_count: torch.Tensor, *, page_tokens: int,
                       tokens: int, out: Sequence[torch.Tensor] | None = None) -> PageTableStep:
    """Room for ``added`` [B] new tokens of requests that hold ``lengths``
    [B]: pages popped from the top of the free stack (``free_pages``, of which
    the first ``free_count`` [1] are free) in request order go into
    ``page_tables`` [B, columns] in place, and every new token gets its
    position and slot (page * page_tokens + position % page_tokens; -1 where
    the table holds no page).  ``tokens`` is the size of the
    packed token outputs, at least the sum of ``added``; entries past it are
    -1.  Where the pages, the columns or ``tokens`` do not suffice, or a count
    is negative, ``overflow`` is 1, positions and slots are -1 and the tables
    stay as they were.  ``out``: the tensors to write, in the order of
    ``PageTableStep``, none of them an input."""

    if lengths.ndim != 1 or page_tables.ndim != 2 or free_pages.ndim != 1:
        raise ValueError("page tables take lengths [B], page_tables [B,columns], free_pages [P]")
    _need_device(lengths, "page tables")
    batch, device, index = lengths.numel(), lengths.device, lengths.get_device()
    columns, pages = page_tables.shape[1], free_pages.numel()
    _int32(lengths, batch, index, "lengths")
    _int32(added, batch, index, "added tokens")
    _int32(page_tables, batch * columns, index, "page tables")
    _int32(free_pages, pages, index, "free pages")
    _int32(free_count, 1, index, "the free count")
    if page_tables.shape[0] != batch:
        raise ValueError("page tables must have a row for every request")
    if page_tokens not in PAGE_TOKENS:
        raise ValueError("a page holds 16, 32, 64, 128 or 256 tokens")
    if tokens < 0:
        raise ValueError("the token count cannot be negative")
    if batch > MAX_REQUESTS:
        raise ValueError(f"page tables take at most {MAX_REQUESTS} requests")
    if out is None:
        sizes = (batch, 1, batch + 1, tokens, tokens, 1)
        step = PageTableStep(*torch.empty(sum(sizes), dtype=_INT32, device=device).split(sizes))
    else:
        step = out if isinstance(out, PageTableStep) else PageTableStep(*out)
        a, b, c, d, e, f = step
        if not (a.dtype is b.dtype is c.dtype is d.dtype is e.dtype is f.dtype is _INT32
                and a.numel() == batch and b.numel() == 1 and c.numel() == batch + 1
                and d.numel() == e.numel() == tokens and f.numel() == 1
                and a.is_contiguous() and b.is_contiguous() and c.is_contiguous()
                and d.is_contiguous() and e.is_contiguous() and f.is_contiguous()
                and a.get_device() == b.get_device() == c.get_device() == d.get_device()
                == e.get_device() == f.get_device() == index):
            raise ValueError(f"page table outputs must be contiguous int32 of {batch}, 1, "
                             f"{batch + 1}, {tokens}, {tokens} and 1 numbers on the inputs' "
                             "device")
        if batch and step.lengths.data_ptr() == lengths.data_ptr():
            raise ValueError("the new lengths cannot be written over the old")
        if step.free_count.data_ptr() == free_count.data_ptr():
            raise ValueError("the new free count cannot be written over the old")
    rc = nat.lib().cowsdm_page_tables_extend(
        lengths.data_ptr(), added.data_ptr(), batch, page_tables.data_ptr(), columns,
        free_pages.data_ptr(), pages, free_count.data_ptr(), page_tokens, tokens,
        step.lengths.data_ptr(), step.free_count.data_ptr(), step.offsets.data_ptr(),
        step.positions.data_ptr(), step.slots.data_ptr(), step.overflow.data_ptr(), nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_page_tables_extend")
    return step


def _cache(key_pages: torch.Tensor, key_scales: torch.Tensor, value_pages: torch.Tensor,
           value_scales: torch.Tensor, width: int, device: int) -> nat.KVCache:
    """The C view of one layer's cache, after checking its tensors."""

    if key_pages.ndim != 4:
        raise ValueError("cache keys must be [pages,heads,page_tokens,width]")
    pages, heads, page_tokens, padded = key_pages.shape
    if (value_pages.shape != (pages, heads, padded, page_tokens)
            or key_scales.shape != (pages, heads) or value_scales.shape != (pages, heads)):
        raise ValueError("cache tensors do not align")
    if (key_pages.dtype is not CODES or value_pages.dtype is not CODES
            or key_scales.dtype is not _FLOAT32 or value_scales.dtype is not _FLOAT32):
        raise TypeError("cache codes are float8_e4m3fn and scales float32")
    if page_tokens not in PAGE_TOKENS:
        raise ValueError("a page holds 16, 32, 64, 128 or 256 tokens")
    if padded != _PADDED.get(width):
        raise ValueError(f"a cache for heads of {width} is {cache_width(width)} wide")
    if not (key_pages.is_contiguous() and key_scales.is_contiguous()
            and value_pages.is_contiguous() and value_scales.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if not (key_pages.get_device() == key_scales.get_device() == value_pages.get_device()
            == value_scales.get_device() == device):
        raise ValueError("cache tensors must be on the inputs' device")
    return nat.KVCache(pages, heads, page_tokens, padded, key_pages.data_ptr(),
                       key_scales.data_ptr(), value_pages.data_ptr(), value_scales.data_ptr())


def write_kv_cache(key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor,
                   key_pages: torch.Tensor, key_scales: torch.Tensor, value_pages: torch.Tensor,
                   value_scales: torch.Tensor) -> None:
    """Keys and values [T, heads, D] (any strides between rows and heads) into
    their slots [T] (int32; -1: not written) of one layer's cache, in place.

    A page and head has one scale for its keys and one for its values: the
    least power of two (from 2^-100 to 2^119) under which every finite
    magnitude is at most 448.  Writing a page's first token sets it from the
    tokens of the call; a page that goes on keeps the larger of its own and
    that one, and where it grows the page's other codes are taken to it,
    exactly but for the smallest.  Codes round to nearest even; e4m3 has no
    infinity, so infinities become NaN.  A page's tokens of one call follow
    one another, as ``extend_page_tables`` gives them."""

    if key.ndim != 3 or value.shape != key.shape:
        raise ValueError("cache writes take key and value [T,heads,D]")
    tokens, heads, width = key.shape
    _need_no_gradient(key, value)
    _need_device(key, "cache writes")
    device = key.get_device()
    code = _float_type(key.dtype)
    if value.dtype is not key.dtype:
        raise TypeError("cache keys and values share one type")
    if value.get_device() != device:
        raise ValueError("cache writes must be on one device")
    _int32(slots, tokens, device, "cache slots")
    cache = _cache(key_pages, key_scales, value_pages, value_scales, width, device)
    if cache.heads != heads:
        raise ValueError("cache and keys differ in heads")
    if tokens == 0:
        return
    step = 8 if code else 4
    key, k, (k_row, k_head, _) = _rows(key, step)
    value, v, (v_row, v_head, _) = _rows(value, step)
    rc = nat.lib().cowsdm_kv_write(cache, k, k_row, k_head, v, v_row, v_head, code, width,
                                   slots.data_ptr(), tokens, nat.stream_handle(key.device))
    if rc:
        nat.check(rc, "cowsdm_kv_write")


def cached_workspace_bytes(batch: int, tokens: int, heads: int, kv_heads: int, width: int,
                           longest: int) -> int:
    """The workspace of a ``cached_attention`` call: 0 where its launch does
    not split the cache."""

    return nat.lib().cowsdm_cached_attention_workspace_bytes(batch, tokens, heads, kv_heads,
                                                             cache_width(width), longest)


def cached_attention(query: torch.Tensor, key_pages: torch.Tensor, key_scales: torch.Tensor,
                     value_pages: torch.Tensor, value_scales: torch.Tensor,
                     page_tables: torch.Tensor, lengths: torch.Tensor, *,
                     longest: int | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of each request's newest tokens over one layer's cache: query
    [B, n, heads, D] holds the last n of its ``lengths`` [B] tokens (written
    before), and row i sees positions 0 to length - n + i.  Grouped heads as
    in ``prompt_attention``.  Returns [B, n, heads, D] in the query's type.
    Tokens whose table entry is no page of the pool are left out, and a row
    that sees nothing is zero.  ``longest`` bounds the lengths (the
    tables' columns when not given): a bound that is too small costs time, not
    correctness."""

    if query.ndim != 4:
        raise ValueError("cached attention takes query [B,n,heads,D]")
    batch, tokens, heads, width = query.shape
    _need_no_gradient(query)
    _need_device(query, "attention inputs")
    device, index = query.device, query.get_device()
    code = _float_type(query.dtype)
    cache = _cache(key_pages, key_scales, value_pages, value_scales, width, index)
    if heads == 0 or heads % cache.heads:
        raise ValueError("query heads must be a multiple of the cache's heads")
    if page_tables.ndim != 2:
        raise ValueError("page tables must be [B,columns]")
    columns = page_tables.shape[1]
    if page_tables.shape[0] != batch:
        raise ValueError("page tables must have a row for every request")
    _int32(page_tables, batch * columns, index, "page tables")
    _int32(lengths, batch, index, "lengths")
    room = columns * cache.page_tokens
    if longest is None or longest > room:
        longest = room
    if longest < 0:
        raise ValueError("the longest length cannot be negative")
    factor = _scale(scale, width)
    out = query.new_empty((batch, tokens, heads, width))
    if not batch or not tokens:
        return out
    query, q_at, (q_request, q_token, q_head, _) = _rows(query, 8 if code else 4)
    need = nat.lib().cowsdm_cached_attention_workspace_bytes(batch, tokens, heads, cache.heads,
                                                             cache.width, longest)
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    q = nat.CachedQuery(
        q_at, q_request, q_token, q_head, page_tables.data_ptr(), lengths.data_ptr(),
        out.data_ptr(), batch, tokens, heads, width, columns, longest, code, factor)
    rc = nat.lib().cowsdm_cached_attention(cache, q, nat.ptr(workspace), need,
                                     nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_cached_attention")
    return out
