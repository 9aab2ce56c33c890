"""The life of a paged cache's pages besides their extension
(``extend_page_tables``): requests that share the first tokens of others,
finished requests' pages, and the pool's pages moved together.

* ``fork_page_tables``     new requests that hold the first tokens of others:
                           whole pages are shared, the page in which the
                           tokens end is a new one;
* ``release_page_tables``  the pages of finished requests, as far as no other
                           request holds them;
* ``compact_page_tables``  the pages in use at the pool's lowest numbers;
* ``copy_pages``           the pages that a fork or a move has to copy, in
                           every layer.

``page_shares`` [pages] counts the requests that hold a page beyond the first:
zeros where nothing is shared.  A page that requests share is full, so that
extension and cache writes never touch one.  What the table operators return
is new, and their inputs stay as they are but for the free stack, onto which a
release pushes above its count, over the numbers that forks and extensions have
popped.  A caller that keeps the tensors from before a call can go back to them,
but after a release only as far as the free count was no larger than the one that
it was called with.

Kernels: csrc/pages.hip.  All on the device, without a read by the host; there
is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat
from .attention import (CODES, MAX_REQUESTS, PAGE_TOKENS, CACHE_WIDTHS, _int32, _need_device)

_INT32, _FLOAT32 = torch.int32, torch.float32


class PageFork(NamedTuple):
    """What ``fork_page_tables`` returns, int32 on the device: the children's
    lengths [n] and tables [n, columns], all pages' shares [pages], the free
    pages left [1], the page to copy for each child and where to (``copy_pages``;
    -1: none) [n], and whether something was wrong or ran short [1]."""

    lengths: torch.Tensor
    page_tables: torch.Tensor
    page_shares: torch.Tensor
    free_count: torch.Tensor
    sources: torch.Tensor
    targets: torch.Tensor
    overflow: torch.Tensor


class PageRelease(NamedTuple):
    """What ``release_page_tables`` returns, int32 on the device: the
    requests' lengths [B] (0 where released), all pages' shares [pages] and the
    free pages [1]."""

    lengths: torch.Tensor
    page_shares: torch.Tensor
    free_count: torch.Tensor


class PageMoves(NamedTuple):
    """What ``compact_page_tables`` returns, int32 on the device: the tables
    [B, columns], all pages' shares [pages], the free stack [pages] and its
    count [1], and the moves that ``copy_pages`` makes: from and to [pages //
    2], ascending, -1 past the last."""

    page_tables: torch.Tensor
    page_shares: torch.Tensor
    free_pages: torch.Tensor
    free_count: torch.Tensor
    sources: torch.Tensor
    targets: torch.Tensor


def _check_tables(lengths: torch.Tensor, page_tables: torch.Tensor, page_shares: torch.Tensor,
                  page_tokens: int) -> tuple[int, int, int, int]:
    if lengths.ndim != 1 or page_tables.ndim != 2 or page_shares.ndim != 1:
        raise ValueError("page tables take lengths [B], page_tables [B,columns], "
                         "page_shares [pages]")
    _need_device(lengths, "page tables")
    index = lengths.get_device()
    batch, columns = page_tables.shape
    pages = page_shares.shape[0]
    if batch != lengths.shape[0]:
        raise ValueError("page tables must have a row for every request")
    _int32(lengths, batch, index, "lengths")
    _int32(page_tables, batch * columns, index, "page tables")
    _int32(page_shares, pages, index, "page shares")
    if page_tokens not in PAGE_TOKENS:
        raise ValueError("a page holds 16, 32, 64, 128 or 256 tokens")
    return batch, columns, pages, index


def fork_page_tables(lengths: torch.Tensor, page_tables: torch.Tensor, page_shares: torch.Tensor,
                     free_pages: torch.Tensor, free_count: torch.Tensor, parents: torch.Tensor,
                     tokens: torch.Tensor, *, page_tokens: int) -> PageFork:
    """New requests, child i with the first ``tokens[i]`` tokens of request
    ``parents[i]`` (int32 [n] both; a request may be named more than once, and
    hold more tokens than that).  The child's whole pages are the parent's and
    get one more sharer each.  Where its tokens end inside a page, it gets one
    of its own from the top of the free stack, in the children's order, and
    that page of the parent's is to be copied there (``copy_pages`` with
    ``sources`` and ``targets``; tokens past the child's length come with it
    and are not read).  Where a parent or a token count is out of range or
    the pages do not suffice, ``overflow`` is 1, the children are empty and
    nothing else changes."""

    batch, columns, pages, index = _check_tables(lengths, page_tables, page_shares, page_tokens)
    if parents.ndim != 1 or tokens.shape != parents.shape:
        raise ValueError("forked requests must be one parent and token count each")
    n, device = parents.numel(), lengths.device
    _int32(free_pages, pages, index, "free pages")
    _int32(free_count, 1, index, "the free count")
    _int32(parents, n, index, "parents")
    _int32(tokens, n, index, "shared tokens")
    if n > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests are forked at once")
    sizes = (n, n * columns, pages, 1, n, n, 1)
    held, tables, shares, count, sources, targets, overflow = torch.split_with_sizes(
        torch.empty(sum(sizes), dtype=_INT32, device=device), sizes)
    fork = PageFork(held, tables.view(n, columns), shares, count, sources, targets, overflow)
    rc = nat.lib().cowsdm_page_tables_fork(
        lengths.data_ptr(), page_tables.data_ptr(), batch, columns, page_shares.data_ptr(),
        free_pages.data_ptr(), pages, free_count.data_ptr(), parents.data_ptr(),
        tokens.data_ptr(), n, page_tokens, held.data_ptr(), tables.data_ptr(), shares.data_ptr(),
        count.data_ptr(), sources.data_ptr(), targets.data_ptr(), overflow.data_ptr(),
        nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_page_tables_fork")
    return fork


def release_page_tables(lengths: torch.Tensor, page_tables: torch.Tensor,
                        page_shares: torch.Tensor, free_pages: torch.Tensor,
                        free_count: torch.Tensor, requests: torch.Tensor, *,
                        page_tokens: int) -> PageRelease:
    """The pages of the named requests (int32 [n]; a second naming and a
    number that is no request count for nothing) let go: each loses as many
    sharers as named requests hold it, and one that no request holds any more
    goes onto the free stack, in place above its count.  They go in the order
    of the list and then of the columns, a shared page where its last named
    holder lists it.  Lengths of the named become 0; the tables are not
    written."""

    batch, columns, pages, index = _check_tables(lengths, page_tables, page_shares, page_tokens)
    if requests.ndim != 1:
        raise ValueError("released requests must be a vector")
    n, device = requests.numel(), lengths.device
    _int32(free_pages, pages, index, "free pages")
    _int32(free_count, 1, index, "the free count")
    _int32(requests, n, index, "released requests")
    if n > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests are released at once")
    lib = nat.lib()
    need = lib.cowsdm_page_tables_release_workspace_bytes(pages, columns, n)
    sizes = (batch, pages, 1, need // 4)
    new_lengths, shares, count, workspace = torch.split_with_sizes(
        torch.empty(sum(sizes), dtype=_INT32, device=device), sizes)
    rc = lib.cowsdm_page_tables_release(
        lengths.data_ptr(), page_tables.data_ptr(), batch, columns, page_shares.data_ptr(),
        free_pages.data_ptr(), pages, free_count.data_ptr(), requests.data_ptr(), n, page_tokens,
        new_lengths.data_ptr(), shares.data_ptr(), count.data_ptr(), workspace.data_ptr(), need,
        nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_page_tables_release")
    return PageRelease(new_lengths, shares, count)


def compact_page_tables(lengths: torch.Tensor, page_tables: torch.Tensor,
                        page_shares: torch.Tensor, *, page_tokens: int) -> PageMoves:
    """The U pages that the requests hold, numbered below U: those numbered U
    or more go, in ascending order, to the numbers below U that no request
    holds.  ``copy_pages`` with ``sources`` and ``targets`` then moves what is in
    them.  The free stack is the other numbers, U on top.  Table entries past
    a request's pages become -1, as entries that are no page of the pool do."""

    batch, columns, pages, index = _check_tables(lengths, page_tables, page_shares, page_tokens)
    device, lib = lengths.device, nat.lib()
    need = lib.cowsdm_page_tables_compact_workspace_bytes(pages)
    sizes = (batch * columns, pages, pages, 1, pages // 2, pages // 2, need // 4)
    tables, shares, stack, count, sources, targets, workspace = torch.split_with_sizes(
        torch.empty(sum(sizes), dtype=_INT32, device=device), sizes)
    moves = PageMoves(tables.view(batch, columns), shares, stack, count, sources, targets)
    rc = lib.cowsdm_page_tables_compact(
        lengths.data_ptr(), page_tables.data_ptr(), batch, columns, page_shares.data_ptr(), pages,
        page_tokens, tables.data_ptr(), shares.data_ptr(), stack.data_ptr(), count.data_ptr(),
        sources.data_ptr(), targets.data_ptr(), workspace.data_ptr(), need,
        nat.stream_handle(device))
    if rc:
        nat.check(rc, "cowsdm_page_tables_compact")
    return moves


def copy_pages(key_pages: torch.Tensor, key_scales: torch.Tensor, value_pages: torch.Tensor,
               value_scales: torch.Tensor, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Pages ``sources`` [n] copied to pages ``targets`` [n] (int32; entries that
    are no page of the pool are left out), codes and scales, in place: of one
    layer's cache (``cached_attention``'s tensors) or of all layers', with the
    layers as a first axis.  Targets differ from each other, and none of them
    is a source: what such pages hold afterwards is not defined."""

    if key_pages.ndim not in (4, 5):
        raise ValueError("cache keys must be [pages,heads,page_tokens,width], of all layers "
                         "with the layers before")
    _need_device(key_pages, "cache pages")
    shape = key_pages.shape
    *lead, pages, heads, page_tokens, width = shape
    layers = lead[0] if lead else 1
    each = shape[:-2]
    if (value_pages.shape != (*each, width, page_tokens) or key_scales.shape != each
            or value_scales.shape != each):
        raise ValueError("cache tensors do not align")
    if (key_pages.dtype is not CODES or value_pages.dtype is not CODES
            or key_scales.dtype is not _FLOAT32 or value_scales.dtype is not _FLOAT32):
        raise TypeError("cache codes are float8_e4m3fn and scales float32")
    if page_tokens not in PAGE_TOKENS:
        raise ValueError("a page holds 16, 32, 64, 128 or 256 tokens")
    if width not in CACHE_WIDTHS:
        raise ValueError("a cache is 32, 64, 96, 128, 192 or 256 wide")
    if not (key_pages.is_contiguous() and key_scales.is_contiguous()
            and value_pages.is_contiguous() and value_scales.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    index = key_pages.get_device()
    if not (key_scales.get_device() == value_pages.get_device() == value_scales.get_device()
            == index):
        raise ValueError("cache tensors must be on one device")
    if sources.ndim != 1 or targets.shape != sources.shape:
        raise ValueError("copied pages must be one source and target each")
    n = sources.numel()
    _int32(sources, n, index, "source pages")
    _int32(targets, n, index, "target pages")
    if not n or not layers or not pages or not heads:
        return
    cache = nat.KVCache(pages, heads, page_tokens, width, key_pages.data_ptr(),
                        key_scales.data_ptr(), value_pages.data_ptr(), value_scales.data_ptr())
    rc = nat.lib().cowsdm_pages_copy(cache, layers, sources.data_ptr(), targets.data_ptr(), n,
                                     nat.stream_handle(key_pages.device))
    if rc:
        nat.check(rc, "cowsdm_pages_copy")
