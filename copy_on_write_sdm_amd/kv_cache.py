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
from weakref import ref

import torch

from . import _native as nat
from .attention import (CODES, MAX_REQUESTS, PAGE_TOKENS, PageTableStep, cache_width,
                        cached_attention, extend_page_tables, prompt_attention, write_kv_cache)
from .head_rotation import HeadRotation, rotate_heads
from .pages import (compact_page_tables, copy_pages, fork_page_tables, release_page_tables)

# Where nothing is shared, requests' pages return in one launch in place, 256
# requests at a time and a request's pages one after another in a thread: so
# many pages one after another.  A call and the wait for it, in place and by
# release_page_tables: 1 request of 4 pages 37 and 61 us, of 128 52 and 62, of
# 1,024 174 and 63; 64 of 40 44 and 68, of 128 64 and 69; 384 of 10 52 and 80;
# 4,096 of 4 194 and 210, of 16 273 and 213.
_IN_PLACE_REQUESTS, _IN_PLACE_PAGES = 256, 128


class PagedKVCache:
    """Requests' pages and every layer's keys and values in them.

    The requests are rows of ``page_tables`` and ``lengths``, in the order of
    the decode state's batch.  How many tokens each holds is known on the host
    as well, so that running out of pages or columns is refused before a
    launch, without reading the device.  Requests that ``fork`` makes share
    the whole pages of what they have in common; such pages are full, and a
    request's new tokens go to pages of its own.  Calls on one cache must be
    stream-ordered.

    ``fork``, ``trim_pages`` and ``grow_pages`` are refused while a step of a
    ``PagedAttention`` over this cache has layers left to run, or the stack is
    within one.  Who calls ``extend`` and ``write`` by hand writes every layer
    before them: a fork copies what has been written, and a trim makes a step's
    slots void."""

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
        self.page_shares = torch.zeros(pages, dtype=torch.int32, device=device)
        self._lengths: list[int] = []
        # the requests' first pages that have been shared, by numbers of the
        # host's own, and how many requests hold each
        self._shared: list[tuple[int, ...]] = []
        self._holders: dict[int, int] = {}
        self._named = 0
        self._released: set[int] = set()
        self._free = pages
        self._before: tuple | None = None       # what the last extend may be taken back to
        self._added: dict[tuple[int, ...], torch.Tensor] = {}
        self._blocks: list[ref[PagedAttention]] = []     # those that run on this cache

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
        self._shared = self._shared + [()] * requests
        self._before = None
        self._added.clear()
        return list(range(first, first + requests))

    def _now(self) -> tuple:
        """What ``extend`` and ``admit`` replace, none of it in place: a table's
        entries past the pages that its request holds are not read."""

        return (self.page_tables, self.lengths, self.free_count, self._lengths, self._free,
                self._shared)

    def _back_to(self, before: tuple) -> None:
        (self.page_tables, self.lengths, self.free_count, self._lengths, self._free,
         self._shared) = before
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

    def _no_open_step(self) -> None:
        """Refuses what would copy or move pages, or replace the pool, while a
        step's slots are yet to be written or it may yet be taken back."""

        for known in self._blocks:
            block = known()
            if block is not None:
                block._none_unfinished()
                if block._whole:
                    raise ValueError("the stack is within a step of the KV cache")

    def fork(self, requests: Sequence[int], tokens: int | Sequence[int] | None = None
             ) -> list[int]:
        """One more request for each named one, after the others: it holds its
        first ``tokens`` tokens (one number for all, or one each; all that it
        holds when None), in every layer.  A request may be named more than
        once.  Whole pages are shared; the page in which the tokens end is
        copied.  Returns the new requests' indices."""

        self._no_open_step()
        named = [int(r) for r in requests]
        if any(not 0 <= r < self.requests or r in self._released for r in named):
            raise ValueError("forked request is invalid or inactive")
        if tokens is None:
            counts = [self._lengths[r] for r in named]
        elif isinstance(tokens, int):
            counts = [tokens] * len(named)
        else:
            counts = [int(n) for n in tokens]
        if len(counts) != len(named) or any(not 0 <= n <= self._lengths[r]
                                            for r, n in zip(named, counts)):
            raise ValueError("forked tokens must be one count per request, at most what it holds")
        page = self.page_tokens
        need = sum(n % page > 0 for n in counts)
        if need > self._free:
            raise ValueError(f"KV cache pages are exhausted: {need} needed, {self._free} free")
        if self.requests + len(named) > MAX_REQUESTS:
            raise ValueError(f"page tables take at most {MAX_REQUESTS} requests")
        first = self.requests
        if not named:
            return []
        both = torch.tensor([named, counts], dtype=torch.int32, device=self.device)
        fork = fork_page_tables(self.lengths, self.page_tables, self.page_shares,
                                self.free_pages, self.free_count, both[0], both[1],
                                page_tokens=page)
        if need:
            copy_pages(self.key_pages, self.key_scales, self.value_pages, self.value_scales,
                       fork.sources, fork.targets)
        tables = torch.cat((self.page_tables, fork.page_tables))
        lengths = torch.cat((self.lengths, fork.lengths))
        self.page_tables, self.lengths = tables, lengths
        self.page_shares, self.free_count = fork.page_shares, fork.free_count
        shared = list(self._shared)
        for r, n in zip(named, counts):
            whole = n // page
            more = range(self._named, self._named + max(0, whole - len(shared[r])))
            self._named += len(more)
            self._holders.update((p, 1) for p in more)
            shared[r] = shared[r] + tuple(more)
            shared.append(shared[r][:whole])
            for p in shared[-1]:
                self._holders[p] += 1
        self._shared = shared
        self._lengths = self._lengths + counts
        self._free -= need
        self._before = None
        self._added.clear()
        return list(range(first, first + len(named)))

    def release(self, requests: Sequence[int]) -> int:
        """The pages of finished requests go back to the pool, but for those
        that other requests share; their rows stay until ``compact``.  Returns
        the pages freed."""

        named = [int(r) for r in requests]
        gone = set(named)
        if (len(gone) != len(named) or any(not 0 <= r < self.requests for r in named)
                or self._released & gone):
            raise ValueError("released sequence is invalid, duplicated, or inactive")
        if not named:
            return 0
        rows = torch.tensor(named, dtype=torch.int32, device=self.device)
        self._before = None         # the stack holds no more what a step has taken off it
        held = [self._pages(self._lengths[r]) for r in named]
        freed, rounds = sum(held), -(-len(named) // _IN_PLACE_REQUESTS)
        if not self._holders and rounds * max(held) <= _IN_PLACE_PAGES:
            nat.check(nat.lib().cowsdm_pages_release(
                self.lengths.data_ptr(), self.page_tables.data_ptr(), self.requests,
                self.page_tables.shape[1], rows.data_ptr(), len(named),
                self.free_pages.data_ptr(), self.free_pages.numel(), self.free_count.data_ptr(),
                self.page_tokens, nat.stream_handle(self.device)), "cowsdm_pages_release")
        else:
            at = rows.long()
            # a launch takes so many; the pages of what comes first lie lowest, above
            # the count until all have gone
            left = self.lengths, self.page_shares, self.free_count
            for part in rows.split(MAX_REQUESTS):
                lengths, shares, count = left
                left = release_page_tables(lengths, self.page_tables, shares, self.free_pages,
                                           count, part, page_tokens=self.page_tokens)
            self.lengths, self.page_shares, self.free_count = left
            self.page_tables.index_fill_(0, at, -1)
        if self._holders:
            for r in named:
                for page in self._shared[r]:
                    self._holders[page] -= 1
                    if self._holders[page]:
                        freed -= 1          # others hold it still
                    else:
                        del self._holders[page]
            self._shared = [() if r in gone else s for r, s in enumerate(self._shared)]
        for r in named:
            self._lengths[r] = 0
        self._released |= gone
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
            self._shared = [self._shared[r] for r in kept]
            self._released = set()
            self._added.clear()
        return kept

    def trim_pages(self, *, headroom_pages: int = 0) -> int:
        """The pool shrunk to the pages that requests hold plus headroom (one
        page at least): the pages in use move to its lowest numbers first, in
        every layer.  Returns the pages given up.  The pool's tensors are
        replaced, which takes room for both meanwhile."""

        if headroom_pages < 0:
            raise ValueError("KV cache headroom cannot be negative")
        self._no_open_step()
        pages = self.free_pages.numel()
        used = pages - self._free
        target = max(1, used + headroom_pages)
        if target >= pages:
            return 0
        moves = compact_page_tables(self.lengths, self.page_tables, self.page_shares,
                                    page_tokens=self.page_tokens)
        most = min(used, pages - used)
        copy_pages(self.key_pages, self.key_scales, self.value_pages, self.value_scales,
                   moves.sources[:most], moves.targets[:most])
        # copies: a slice of a pool of one layer is contiguous as it is, and
        # would keep all of that pool's memory
        kept = [t[:, :target].clone(memory_format=torch.contiguous_format)
                for t in (self.key_pages, self.key_scales, self.value_pages, self.value_scales)]
        tables, shares = moves.page_tables.clone(), moves.page_shares[:target].clone()
        # the stack's numbers fall from the pool's last one on
        stack = moves.free_pages[pages - target:].clone()
        count = torch.full_like(self.free_count, target - used)
        self.key_pages, self.key_scales, self.value_pages, self.value_scales = kept
        self.page_tables, self.page_shares = tables, shares
        self.free_pages, self.free_count = stack, count
        self._free = target - used
        self._before = None
        return pages - target

    def grow_pages(self, pages: int) -> None:
        """``pages`` more in the pool, which are taken after those that are
        free now.  The pool's tensors are replaced, which takes room for both
        meanwhile."""

        if pages < 0:
            raise ValueError("added KV cache pages cannot be negative")
        self._no_open_step()
        if not pages:
            return
        before = self.free_pages.numel()
        if (before + pages) * self.page_tokens >= 1 << 31:
            raise ValueError("KV cache pages hold fewer than 2^31 tokens")

        def grown(t: torch.Tensor, value: int) -> torch.Tensor:
            bits = t.view(torch.uint8) if t.dtype is CODES else t
            new = bits.new_full((t.shape[0], before + pages, *t.shape[2:]), value)
            new[:, :before] = bits
            return new.view(t.dtype)

        pool = [grown(self.key_pages, 0), grown(self.key_scales, 1),
                grown(self.value_pages, 0), grown(self.value_scales, 1)]
        shares = torch.cat((self.page_shares, self.page_shares.new_zeros(pages)))
        fresh = torch.arange(before + pages - 1, before - 1, -1, dtype=torch.int32,
                             device=self.device)
        stack, count = torch.cat((fresh, self.free_pages)), self.free_count + pages
        self.key_pages, self.key_scales, self.value_pages, self.value_scales = pool
        self.page_shares, self.free_pages, self.free_count = shares, stack, count
        self._free += pages
        self._before = None

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
            "kv_tables": 4 * (self.page_tables.numel() + self.lengths.numel() + 2 * pages + 1),
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

    ``AttentionProjections`` makes both of the layers' weights.  With
    ``rotation`` or ``head_norms`` (for each of the layers the query's and the
    key's norm weight, or None), queries and keys go from ``project`` through
    ``rotate_heads`` at the tokens' positions, with ``norm_eps``.

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
                 finish: Finish, *, scale: float | None = None,
                 rotation: HeadRotation | None = None,
                 head_norms: Sequence[tuple[torch.Tensor | None, torch.Tensor | None]] | None
                 = None, norm_eps: float = 1e-6):
        self.cache, self.layers = cache, tuple(layers)
        if not self.layers or len(self.layers) > cache.layers:
            raise ValueError("the cache needs a layer for every attention layer")
        if head_norms is not None and len(head_norms) != len(self.layers):
            raise ValueError("head norms must be one pair per attention layer")
        self.project, self.finish, self.scale = project, finish, scale
        self.rotation, self.head_norms, self.norm_eps = rotation, head_norms, norm_eps
        self._step: PageTableStep | None = None
        self._next = 0              # the layer of the step that runs next
        self._prompt = False
        self._whole = False         # within a step that the stack has opened
        self._before: tuple | None = None       # where the cache stood before the step
        cache._blocks = [known for known in cache._blocks if known() is not None] + [ref(self)]

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
        self._whole = True
        try:
            yield
            if self._unfinished():
                raise ValueError(f"attention layer {self.layers[self._next]} is not in the layout")
        except BaseException:
            self.abort()
            raise
        finally:
            self._whole = False

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

    def _projected(self, layer: int, index: int, rows: torch.Tensor, positions: torch.Tensor
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        query, key, value = self.project(layer, rows, positions)
        if self.rotation is not None or self.head_norms is not None:
            norms = (None, None) if self.head_norms is None else self.head_norms[index]
            query, key = rotate_heads(query, key, positions, self.rotation, query_norm=norms[0],
                                      key_norm=norms[1], eps=self.norm_eps)
        return query, key, value

    @torch.no_grad()
    def prefill(self, layer: int, tokens: torch.Tensor):
        """``attention_block``: tokens [B, T, width] of B new requests."""

        batch, time, width = tokens.shape
        index, step = self._enter(layer, True, self._begin_prefill, batch, time)
        try:
            rows = tokens.reshape(batch * time, width)
            query, key, value = self._projected(layer, index, rows, step.positions)
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
            query, key, value = self._projected(layer, index, rows, step.positions)
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
