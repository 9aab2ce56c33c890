"""The paged 8-bit K/V cache of a stack's attention layers, with its request
lifecycle, and the attention callables over it that
``prefill_faithful_sdm_stack`` and ``decode_faithful_sdm_stack`` take.

The reference keeps each attention layer's keys and values dense, in the
activations' type, for every request's whole capacity
(``_allocate_dense_cache``, inference.py:293-306).  Here a request holds pages
of one pool for the tokens that it has, in a byte an element; the page tables
are shared by the layers, whose requests are equally long.
"""

from __future__ import annotations

from contextlib import contextmanager
from typing import Callable, Sequence

import torch

from .attention import (CODES, PAGE_TOKENS, PageTableStep, cache_width, cached_attention,
                        extend_page_tables, prompt_attention, write_kv_cache)
from . import _native as nat


class PagedKVCache:
    """Requests' pages and every layer's keys and values in them.

    The requests are rows of ``page_tables`` and ``lengths``, in the order of
    the decode state's batch.  How many tokens each holds is known on the host
    as well, so that running out of pages or columns is refused before a
    launch, without reading the device.  Calls on one cache must be
    stream-ordered."""

    def __init__(self, layers: int, heads: int, head_width: int, *, capacity: int, pages: int,
                 page_tokens: int = 64, device: torch.device | str = "cuda"):
        """Room for requests of up to ``capacity`` tokens over ``pages`` pages."""

        if layers <= 0 or heads <= 0 or capacity <= 0 or pages <= 0:
            raise ValueError("KV cache layers, heads, capacity and pages must be positive")
        if page_tokens not in PAGE_TOKENS:
            raise ValueError("a page holds 16, 32, 64, 128 or 256 tokens")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("the KV cache must be on the GPU: it has no CPU path")
        width = cache_width(head_width)
        self.heads, self.head_width, self.page_tokens = heads, head_width, page_tokens
        self.capacity = capacity
        # zeros, so that no slot ever holds NaN by chance
        self.key_pages = torch.zeros(layers, pages, heads, page_tokens, width,
                                     dtype=torch.uint8, device=device).view(CODES)
        self.value_pages = torch.zeros(layers, pages, heads, width, page_tokens,
                                       dtype=torch.uint8, device=device).view(CODES)
        self.key_scales = torch.ones(layers, pages, heads, device=device)
        self.value_scales = torch.ones(layers, pages, heads, device=device)
        columns = -(-capacity // page_tokens)
        self.page_tables = torch.empty(0, columns, dtype=torch.int32, device=device)
        self.lengths = torch.empty(0, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)
        self._lengths: list[int] = []
        self._released: set[int] = set()
        self._free = pages
        self._before: tuple | None = None       # what the last extend may be taken back to
        self._added: dict[tuple[int, ...], torch.Tensor] = {}

    @property
    def layers(self) -> int:
        return self.key_pages.shape[0]

    @property
    def requests(self) -> int:
        return len(self._lengths)

    @property
    def device(self) -> torch.device:
        return self.lengths.device

    @property
    def free(self) -> int:
        """Pages that no request holds."""

        return self._free

    def request_lengths(self) -> list[int]:
        """The tokens that each request holds."""

        return list(self._lengths)

    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.page_tokens)

    def admit(self, requests: int) -> list[int]:
        """``requests`` more rows, without tokens, after the others; their indices."""

        if requests < 0:
            raise ValueError("admitted requests cannot be negative")
        first = self.requests
        rows = torch.full((requests, self.page_tables.shape[1]), -1, dtype=torch.int32,
                          device=self.device)
        tables = torch.cat((self.page_tables, rows))
        lengths = torch.cat((self.lengths, self.lengths.new_zeros(requests)))
        self.page_tables, self.lengths = tables, lengths
        self._lengths = self._lengths + [0] * requests
        self._before = None
        self._added.clear()
        return list(range(first, first + requests))

    def _now(self) -> tuple:
        """What ``extend`` and ``admit`` replace, none of it in place: a table's
        entries past the pages that its request holds are not read."""

        return self.page_tables, self.lengths, self.free_count, self._lengths, self._free

    def _back_to(self, before: tuple) -> None:
        self.page_tables, self.lengths, self.free_count, self._lengths, self._free = before
        self._before = None
        self._added.clear()

    def take_back(self) -> None:
        """Takes the last ``extend`` back, as long as no other change has
        followed it: its pages are free again, and what ``write`` has put into
        its slots lies past the lengths, where nothing reads.  (A page that it
        went on in keeps a scale that those tokens raised.)"""

        if self._before is None:
            raise ValueError("there is no KV cache step to take back")
        self._back_to(self._before)

    def extend(self, added: int | Sequence[int]) -> PageTableStep:
        """Pages for ``added`` more tokens of every request (one number for
        all, or one each); ``write`` then fills their slots."""

        counts = [added] * self.requests if isinstance(added, int) else [int(n) for n in added]
        if len(counts) != self.requests or min(counts, default=0) < 0:
            raise ValueError("added tokens must be one count per request, none negative")
        if any(n and r in self._released for r, n in enumerate(counts)):
            raise ValueError("released requests must be removed before further decode")
        lengths = [n + m for n, m in zip(self._lengths, counts)]
        if max(lengths, default=0) > self.capacity:
            raise ValueError("decode state has reached its fixed capacity")
        need = sum(self._pages(n) for n in lengths) - sum(self._pages(n) for n in self._lengths)
        if need > self._free:
            raise ValueError(f"KV cache pages are exhausted: {need} needed, {self._free} free")
        key = tuple(counts)
        tensor = self._added.get(key)
        if tensor is None:
            if len(self._added) >= 8:
                self._added.clear()
            tensor = self._added[key] = torch.tensor(counts, dtype=torch.int32,
                                                     device=self.device)
        step = extend_page_tables(self.lengths, tensor, self.page_tables, self.free_pages,
                                  self.free_count, page_tokens=self.page_tokens,
                                  tokens=sum(counts))
        self._before = self._now()
        self.lengths, self.free_count = step.lengths, step.free_count
        self._lengths, self._free = lengths, self._free - need
        return step

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor,
              slots: torch.Tensor) -> None:
        """One layer's keys and values [T, heads, D] into a step's slots."""

        write_kv_cache(key, value, slots, self.key_pages[layer], self.key_scales[layer],
                       self.value_pages[layer], self.value_scales[layer])

    def attend(self, layer: int, query: torch.Tensor, *, scale: float | None = None
               ) -> torch.Tensor:
        """``cached_attention`` of every request's newest tokens [B, n, heads, D]."""

        return cached_attention(query, self.key_pages[layer], self.key_scales[layer],
                                self.value_pages[layer], self.value_scales[layer],
                                self.page_tables, self.lengths,
                                longest=max(self._lengths, default=0), scale=scale)

    def release(self, requests: Sequence[int]) -> int:
        """The pages of finished requests go back to the pool; their rows stay
        until ``compact``.  Returns the pages freed."""

        named = [int(r) for r in requests]
        if (len(set(named)) != len(named) or any(not 0 <= r < self.requests for r in named)
                or self._released & set(named)):
            raise ValueError("released sequence is invalid, duplicated, or inactive")
        if not named:
            return 0
        rows = torch.tensor(named, dtype=torch.int32, device=self.device)
        nat.check(nat.lib().cowsdm_pages_release(
            self.lengths.data_ptr(), self.page_tables.data_ptr(), self.requests,
            self.page_tables.shape[1], rows.data_ptr(), len(named), self.free_pages.data_ptr(),
            self.free_pages.numel(), self.free_count.data_ptr(), self.page_tokens,
            nat.stream_handle(self.device)), "cowsdm_pages_release")
        freed = sum(self._pages(self._lengths[r]) for r in named)
        self._before = None
        for r in named:
            self._lengths[r] = 0
        self._released |= set(named)
        self._free += freed
        return freed

    def compact(self) -> list[int]:
        """Closes the rows of released requests; the others keep their order
        and their pages.  Returns the survivors' former indices."""

        kept = [r for r in range(self.requests) if r not in self._released]
        if self._released:
            index = torch.tensor(kept, dtype=torch.int64, device=self.device)
            tables, lengths = (t.index_select(0, index) for t in (self.page_tables, self.lengths))
            self.page_tables, self.lengths = tables, lengths
            self._before = None
            self._lengths = [self._lengths[r] for r in kept]
            self._released = set()
            self._added.clear()
        return kept

    def storage_bytes(self) -> dict[str, int]:
        """Bytes of the codes, their scales and the tables, and of the codes and
        scales in pages that requests hold."""

        codes = self.key_pages.numel() + self.value_pages.numel()
        scales = 4 * (self.key_scales.numel() + self.value_scales.numel())
        pages = self.free_pages.numel()
        used = pages - self._free
        return {
            "kv_codes": codes,
            "kv_scales": scales,
            "kv_tables": 4 * (self.page_tables.numel() + self.lengths.numel() + pages + 1),
            "kv_live": (codes + scales) // pages * used,
        }


Project = Callable[[int, torch.Tensor, torch.Tensor],
                   "tuple[torch.Tensor, torch.Tensor, torch.Tensor]"]
Finish = Callable[[int, torch.Tensor, torch.Tensor], torch.Tensor]


class PagedAttention:
    """A stack's "A" layers over a ``PagedKVCache``: ``prefill`` is
    ``prefill_faithful_sdm_stack``'s ``attention_block`` and ``decode``
    ``decode_faithful_sdm_stack``'s ``attention_decode``.  The caller gives
    what belongs to the model:

    * ``project(layer, tokens [T, width], positions [T])`` -> query
      [T, heads, D], key and value [T, kv_heads, D] (norm, projections and any
      rotation by position);
    * ``finish(layer, tokens [T, width], mixed [T, heads, D])`` -> the block's
      residual stream [T, width] (output projection, residual add, MLP).

    ``layers`` are the positions of the "A" layers in the layout, in the order
    in which they run.  A prefill admits its requests after those that the cache holds, as
    ``FaithfulSDMDecodeState.admit`` appends them to the batch; ``release`` and
    ``compact`` of the cache go with the state's.  The state's own dense caches
    of these layers hold no heads.

    A step is a token, or a prompt, through all of these layers.  The stack's
    prefill and decode open it before their first layer runs, so that one that
    the cache has no room for changes nothing, and take it back when any layer
    raises: the cache then stands where the decode state does, and the step can
    be run again.  Called by itself, the first layer's call opens the step, a
    layer that raises takes it back, and ``abort`` does so for what fails
    between the layers.  What SDM layers have written before a failure is
    theirs and stays."""

    def __init__(self, cache: PagedKVCache, layers: Sequence[int], project: Project,
                 finish: Finish, *, scale: float | None = None):
        self.cache, self.layers = cache, tuple(layers)
        if not self.layers or len(self.layers) > cache.layers:
            raise ValueError("the cache needs a layer for every attention layer")
        self.project, self.finish, self.scale = project, finish, scale
        self._step: PageTableStep | None = None
        self._next = 0              # the layer of the step that runs next
        self._prompt = False
        self._before: tuple | None = None       # where the cache stood before the step

    # ------------------------------------------------------------- the steps

    def _open(self, step: PageTableStep, prompt: bool) -> None:
        self._step, self._next, self._prompt = step, 0, prompt
        self._before = self.cache._before

    def _unfinished(self) -> bool:
        return self._step is not None and self._next < len(self.layers)

    def _none_unfinished(self) -> None:
        if self._unfinished():
            raise ValueError(f"the last step has not run attention layer "
                             f"{self.layers[self._next]}: abort() takes it back")

    def _begin_prefill(self, batch: int, time: int) -> None:
        self._none_unfinished()
        cache, before = self.cache, self.cache._now()
        try:
            cache.admit(batch)
            step = cache.extend([0] * len(before[3]) + [time] * batch)
        except BaseException:
            # no room: the cache is as it was
            cache._back_to(before)
            raise
        cache._before = before
        self._open(step, True)

    def _begin_decode(self, batch: int, position: "int | Sequence[int] | torch.Tensor") -> None:
        self._none_unfinished()
        held = self.cache._lengths
        if isinstance(position, int):
            at = [position] * batch
        else:
            at = position.tolist() if isinstance(position, torch.Tensor) else list(position)
        if at != held:
            raise ValueError("decode positions do not match the KV cache")
        self._open(self.cache.extend(1), False)

    def abort(self) -> None:
        """Takes the last step back, whichever of its layers have run; nothing
        where there is none, or the cache has changed since."""

        before, self._before, self._step = self._before, None, None
        if before is not None and self.cache._before is before:
            self.cache.take_back()

    @contextmanager
    def _whole_step(self, begin: Callable[..., None], *args):
        begin(*args)
        try:
            yield
            if self._unfinished():
                raise ValueError(f"attention layer {self.layers[self._next]} is not in the layout")
        except BaseException:
            self.abort()
            raise

    def prefill_step(self, batch: int, time: int):
        """A context that opens the step of a prompt and takes it back when its
        body raises or leaves an attention layer out."""

        return self._whole_step(self._begin_prefill, batch, time)

    def decode_step(self, batch: int, position: "int | Sequence[int] | torch.Tensor"):
        """The same of one token of every request, which stand at ``position``
        (one for all, or one each)."""

        return self._whole_step(self._begin_decode, batch, position)

    def _enter(self, layer: int, prompt: bool, begin: Callable[..., None], *args
               ) -> tuple[int, PageTableStep]:
        """The layer's index and step, opened by its first layer if need be."""

        if layer not in self.layers:
            raise ValueError(f"layer {layer} is not one of the attention layers {self.layers}")
        index = self.layers.index(layer)
        if not self._unfinished() and index == 0:
            begin(*args)
        if not self._unfinished() or index != self._next or prompt is not self._prompt:
            raise ValueError(f"attention layer {layer} is not the next of its step")
        return index, self._step

    # ------------------------------------------------------------ the layers

    @torch.no_grad()
    def prefill(self, layer: int, tokens: torch.Tensor):
        """``attention_block``: tokens [B, T, width] of B new requests."""

        batch, time, width = tokens.shape
        index, step = self._enter(layer, True, self._begin_prefill, batch, time)
        try:
            rows = tokens.reshape(batch * time, width)
            query, key, value = self.project(layer, rows, step.positions)
            self.cache.write(index, key, value, step.slots)
            mixed = prompt_attention(query, key, value, step.offsets, longest=time,
                                     scale=self.scale)
            out = self.finish(layer, rows, mixed).reshape(batch, time, width)
            none = tokens.new_empty(batch, 0, time, self.cache.head_width)
        except BaseException:
            self.abort()
            raise
        self._next = index + 1
        return out, none, none

    @torch.no_grad()
    def decode(self, layer: int, tokens: torch.Tensor, key_cache: torch.Tensor,
               value_cache: torch.Tensor, position: "int | torch.Tensor") -> torch.Tensor:
        """``attention_decode``: one more token [B, 1, width] of every request."""

        batch, _, width = tokens.shape
        index, step = self._enter(layer, False, self._begin_decode, batch, position)
        try:
            rows = tokens.reshape(batch, width)
            query, key, value = self.project(layer, rows, step.positions)
            self.cache.write(index, key, value, step.slots)
            mixed = self.cache.attend(index, query.unsqueeze(1), scale=self.scale)
            out = self.finish(layer, rows, mixed.squeeze(1)).reshape(batch, 1, width)
        except BaseException:
            self.abort()
            raise
        self._next = index + 1
        return out


def paged_owner(attention) -> PagedAttention | None:
    """The ``PagedAttention`` whose bound method ``attention`` is, for the
    stack's prefill and decode."""

    owner = getattr(attention, "__self__", None)
    return owner if isinstance(owner, PagedAttention) else None
