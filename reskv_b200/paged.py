"""Paged KV cache in 4 bits for sequences of different lengths.

The compressed caches of this package hold one batch of equal lengths.  ``PagedInt4Cache`` is the cache of a server whose
sequences come, grow, fork and go: keys (after RoPE) and values as 4-bit codes in pages of 64 tokens out of one pool for all
layers, 144 bytes per token and KV head instead of 512.  The kernels are ``csrc/paged_store.cu`` and
``csrc/paged_attention.cu``; the layout of a page is described in ``csrc/paged_int4.cuh``.

A step of a model::

    step = cache.extend(sequences, counts)          # room for the new tokens; tables on the device
    for layer ...:
        cache.write(layer, step, key, value)        # [new tokens, KV heads, 128], packed
        out = cache.attend(layer, step, query)      # one query per sequence, or prompt_attention for whole prompts
"""

from __future__ import annotations

from collections import Counter

import numpy as np
import torch

from ._extension import device_index_of, host, require_device

PAGE_TOKENS = 64
MOST_GROUP = 8  # query heads per KV head
_PAGE_HEAD = (4, 2304)  # blocks of 16 tokens, bytes of a block
_TYPES = (torch.float16, torch.bfloat16)


class PagedStep:
    """Where the tokens of one step lie: made by ``PagedInt4Cache.extend`` and used for every layer of the step.

    ``counts[i]`` tokens of ``sequences[i]`` are new, ``lengths[i]`` is its length with them; ``total`` is their sum over the
    step.  ``cu_seqlens`` (int32, on the device) says which rows of the packed tensors belong to which sequence and serves
    ``prompt_attention`` as it is."""

    __slots__ = ("sequences", "counts", "lengths", "total", "cu_seqlens", "starts", "device_lengths", "table", "_tables", "_use", "_whole", "_epoch",
                 "_current")

    def _everything(self):
        """``(cu_seqlens, starts, tokens)`` of all tokens of the sequences, the earlier ones included."""
        if self._whole is None:
            _refuse_capture(self.table.device)
            ends = np.concatenate(([0], np.cumsum(self.lengths)))
            if ends[-1] > 2**31 - 1:
                raise ValueError("too many tokens for one call")
            self._whole = (_upload(ends.astype(np.int32), self.table.device), torch.zeros_like(self.starts), int(ends[-1]))
        return self._whole


class _Tables:
    """Tables on the device, and how many steps have had them: they are the last one's."""

    __slots__ = ("numbers", "book", "uses")

    def __init__(self, numbers, book):
        self.numbers, self.book, self.uses = numbers, book, 0


def _refuse_capture(device, what="a step's tables come from the host: make them", instead=" (extend(reuse=) fills those of a captured step)") -> None:
    with torch.cuda.device(device):
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError(f"{what} outside of the capture{instead}")


def _pinned(numbers: np.ndarray) -> torch.Tensor:
    pinned = torch.empty(numbers.size, dtype=torch.int32, pin_memory=True)
    pinned.numpy()[:] = numbers.reshape(-1)
    return pinned


def _upload(numbers: np.ndarray, device) -> torch.Tensor:
    """int32 numbers on the device, without waiting for the copy."""
    return _pinned(numbers).to(device, non_blocking=True)


class PagedInt4Cache:
    """4-bit cache of ``layers`` layers with ``kv_heads`` heads of 128 in a pool of ``pages`` pages of 64 tokens.

    Sequences are numbers given out by ``add`` and ``fork``.  A page that is full may be shared by forked sequences; a page
    that still takes tokens belongs to one.  The calls launch on the current stream of the cache's device and do not wait for it;
    a caller that uses several streams orders them itself.  The tables are the host's, so one thread at a time changes a cache.
    """

    def __init__(self, layers: int, kv_heads: int, pages: int, *, dtype: torch.dtype = torch.float16, device="cuda"):
        for name, value in (("layers", layers), ("kv_heads", kv_heads), ("pages", pages)):
            if type(value) is not int or value < 1:
                raise ValueError(f"{name} must be a positive integer")
        if dtype not in _TYPES:
            raise ValueError("dtype must be torch.float16 or torch.bfloat16")
        self.layers, self.kv_heads, self.capacity, self.dtype = layers, kv_heads, pages, dtype
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("a paged cache lives on a CUDA device")
        self.device = torch.device("cuda", device_index_of(self.device))
        require_device(self.device.index)
        self.pages = torch.empty((layers, pages, kv_heads, *_PAGE_HEAD), dtype=torch.uint8, device=self.device)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._book = PageBook(pages)

    # -- sequences -------------------------------------------------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._book.free)

    def add(self, count: int = 1) -> list[int]:
        """``count`` new, empty sequences."""
        return self._book.add(count)

    def length(self, sequence: int) -> int:
        return self._book.of(sequence).length

    def extend(self, sequences, counts, *, width: int = 0, reuse: PagedStep | None = None) -> PagedStep:
        """Room for ``counts[i]`` (or ``counts`` for each) more tokens of ``sequences[i]``, no sequence twice.  Earlier steps
        of these sequences may not be used any more.  RuntimeError, and nothing changed, when the pool has too few pages.

        For captured graphs: the page table is made at least ``width`` pages wide, and with ``reuse``, an earlier step of as many
        sequences, the tables are written to that step's tensors, whose addresses a graph holds; the step that had them last may
        not be used any more either.  ValueError, and nothing
        changed, when a sequence has more pages than that table is wide."""
        _refuse_capture(self.device)
        book = self._book
        sequences, counts = list(sequences), [counts] * len(sequences) if type(counts) is int else list(counts)
        if type(width) is not int or width < 0:
            raise ValueError("width must be a non-negative integer")
        if reuse is not None:
            if not isinstance(reuse, PagedStep) or reuse._tables.book is not book or reuse.table.shape[0] != len(sequences):
                raise ValueError("reuse must be a step of this cache with as many sequences")
            if type(counts) is list and all(type(c) is int for c in counts) and len(counts) == len(sequences):
                most = max((-(-(book.of(q).length + c) // PAGE_TOKENS) for q, c in zip(sequences, counts)), default=0)
                if most > reuse.table.shape[1]:
                    raise ValueError(f"{most} pages of a sequence do not fit a table of {reuse.table.shape[1]}")
            width = reuse.table.shape[1]
        entries = book.extend(sequences, counts)
        try:
            step = self._tables_of(entries, sequences, counts, width, reuse)
        except BaseException:  # no memory for the tables: the device has not heard of these tokens
            book.retract(entries, counts)
            raise
        for e in entries:
            e.supersede(step)
        return step

    def _tables_of(self, entries, sequences, counts, width, reuse) -> PagedStep:
        step = PagedStep()
        n, width = len(entries), max([width, *(len(e.pages) for e in entries)])
        step.sequences, step.counts, step.lengths = tuple(sequences), tuple(counts), tuple(e.length for e in entries)
        step.total = sum(counts)
        numbers = np.zeros(3 * n + 1 + n * width, np.int32)
        np.cumsum(counts, out=numbers[1:n + 1])
        numbers[2 * n + 1:3 * n + 1] = step.lengths
        numbers[n + 1:2 * n + 1] = numbers[2 * n + 1:3 * n + 1] - np.asarray(counts, np.int32)
        table = numbers[3 * n + 1:].reshape(n, width)
        for row, e in zip(table, entries):
            row[:len(e.pages)] = e.pages
        if reuse is None:
            step._tables = _Tables(_upload(numbers, self.device), self._book)
        else:
            step._tables = reuse._tables
            step._tables.numbers.copy_(_pinned(numbers), non_blocking=True)
        step._tables.uses += 1
        step._use, there = step._tables.uses, step._tables.numbers
        step.cu_seqlens, step.starts, step.device_lengths = there[:n + 1], there[n + 1:2 * n + 1], there[2 * n + 1:3 * n + 1]
        step.table = there[3 * n + 1:].view(n, width)
        step._whole, step._epoch, step._current = None, self._book.epoch, True
        return step

    def _retract(self, step: PagedStep) -> None:
        """Takes back the last step of its sequences, which failed on its way: its tokens do not count."""
        self._check(step)
        entries = [self._book.of(s) for s in step.sequences]
        self._book.retract(entries, step.counts)
        for e in entries:
            e.supersede()

    def fork(self, sequences) -> list[int]:
        """A new sequence with the tokens of each of ``sequences`` (one may be named several times).  Full pages are shared, a
        partly filled last page is copied; steps of the forked sequences may not be used any more."""
        self._refuse_capture()
        return self._book.fork(list(sequences), self._copy)[0]

    def _exchange(self, ending, sequences) -> list[int]:
        """``free(ending)`` and ``fork(sequences)`` in one, all or nothing: the copies may take the pages that become free."""
        self._refuse_capture()
        return self._book.fork(list(sequences), self._copy, list(ending))[0]

    def free(self, sequences) -> None:
        """Ends ``sequences``; pages that no other sequence shares go back to the pool."""
        self._book.release(list(sequences))

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool and returns their number.  No earlier step may be used any more."""
        self._refuse_capture()
        return self._book.compact(self._copy)[0]

    # -- device ----------------------------------------------------------------------------------------------------------------
    def _check(self, step: PagedStep) -> None:
        if not isinstance(step, PagedStep):
            raise TypeError(f"expected a PagedStep, got {type(step).__name__}")
        if not step._current or step._use != step._tables.uses or step._epoch is not self._book.epoch:
            raise ValueError("the step belongs to another cache, or its sequences have been extended, forked, freed or moved since")

    def write(self, layer: int, step: PagedStep, key: torch.Tensor, value: torch.Tensor) -> None:
        """Stores the step's new tokens: ``key`` (after RoPE) and ``value`` ``[step.total, KV heads, 128]`` of the cache's type."""
        self._check(step)
        if isinstance(key, torch.Tensor) and (key.dtype != self.dtype or key.shape[:1] != (step.total,)):
            raise ValueError(f"key and value must hold the step's {step.total} tokens in {self.dtype}")
        host().paged_write(self.pages, layer, self._status, key, value, step.cu_seqlens, step.starts, step.table)

    def read(self, layer: int, step: PagedStep, *, everything: bool = False):
        """``(key, value)`` as the cache holds them: of the step's new tokens, or of all tokens of its sequences
        (``everything``), packed ``[tokens, KV heads, 128]`` in the order of the step."""
        self._check(step)
        cu, starts, tokens = step._everything() if everything else (step.cu_seqlens, step.starts, step.total)
        return host().paged_read(self.pages, layer, self._status, self.dtype == torch.bfloat16, cu, starts, step.table, tokens)

    def attend(self, layer: int, step: PagedStep, query: torch.Tensor, *, scaling: float | None = None, return_lse: bool = False):
        """One query per sequence of the step, ``[sequences, H, 128]`` after RoPE, against all of its tokens; ``H`` is up to
        eight times the KV heads, ``scaling`` (positive) defaults to ``128**-0.5``.  Returns ``[sequences, H, 128]``, with
        ``return_lse`` also FP32 ``[sequences, H]``, the logarithm of the sum of exponentials.  A sequence without tokens gets
        zeros (and minus infinity).  In a BF16 cache keys up to ``2**111`` and values up to ``2**101`` in magnitude can be
        attended to (NaN beyond); scales of values below ``2**-60`` lose bits."""
        self._check(step)
        if isinstance(query, torch.Tensor) and query.dtype != self.dtype:
            raise ValueError(f"query must be {self.dtype}")
        return host().paged_attention(self.pages, layer, self._status, query, step.device_lengths, step.table, scaling, bool(return_lse))

    def copy_pages(self, src, dst) -> None:
        """Copies pages ``src[i]`` to ``dst[i]`` in all layers, all at once: no page may be a destination twice, or source and
        destination.  What ``fork`` and ``compact`` use; the caller of this one answers for whose pages they are."""
        host().copy_pages(self.pages, src, dst)

    def _refuse_capture(self) -> None:
        _refuse_capture(self.device, "pages are given out by the host: fork and compact", " (copy_pages may be captured)")

    def _copy(self, pairs) -> None:
        if pairs:
            host().copy_pages(self.pages, *zip(*pairs))

    @property
    def status(self) -> torch.Tensor:
        """What ``check`` reads, int32 on the device; ``prompt_attention(..., status=cache.status)`` reports there too."""
        return self._status

    def check(self) -> None:
        """Waits for the device and raises if a kernel met a token or page outside its tables, or a wait that ran out."""
        word = self._status.item()
        if word:
            raise RuntimeError(f"paged cache: device status 0x{word & 0xFFFFFFFF:x}")

    @property
    def nbytes(self) -> int:
        return self.pages.nbytes


class _Sequence:
    __slots__ = ("pages", "length", "step")

    def __init__(self, pages=(), length=0):
        self.pages, self.length, self.step = list(pages), length, None

    def supersede(self, step=None):
        if self.step is not None:
            self.step._current = False
        self.step = step


class PageBook:
    """Which sequence holds which pages, and how often a page is held.  Host only."""

    def __init__(self, pages: int):
        self.free = list(range(pages - 1, -1, -1))  # taken from the end: the lowest numbers first
        self.holders = [0] * pages
        self.sequences: dict[int, _Sequence] = {}
        self.epoch = object()  # steps made before the pages moved belong to another one
        self._next = 0

    def of(self, sequence: int) -> _Sequence:
        entry = self.sequences.get(sequence) if type(sequence) is int else None
        if entry is None:
            raise ValueError(f"no sequence {sequence!r} in this cache")
        return entry

    def _new(self, entry: _Sequence) -> int:
        self.sequences[self._next] = entry
        self._next += 1
        return self._next - 1

    def _take(self) -> int:
        page = self.free.pop()
        self.holders[page] = 1
        return page

    def _need(self, pages: int) -> None:
        if pages > len(self.free):
            raise RuntimeError(f"out of pages: {pages} needed, {len(self.free)} free")

    def add(self, count: int) -> list[int]:
        if type(count) is not int or count < 0:
            raise ValueError("count must be a non-negative integer")
        return [self._new(_Sequence()) for _ in range(count)]

    def extend(self, sequences, counts) -> list[_Sequence]:
        entries = [self.of(s) for s in sequences]
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence is named twice")
        if len(counts) != len(entries) or any(type(c) is not int or c < 0 for c in counts):
            raise ValueError("counts must be one non-negative integer per sequence")
        if sum(counts) > 2**31 - 1 or any(e.length + c > 2**31 - PAGE_TOKENS for e, c in zip(entries, counts)):
            raise ValueError("too many tokens")
        more = [-(-(e.length + c) // PAGE_TOKENS) - len(e.pages) for e, c in zip(entries, counts)]
        self._need(sum(more))
        for e, c, m in zip(entries, counts, more):
            e.pages.extend(self._take() for _ in range(m))
            e.length += c
        return entries

    def retract(self, entries, counts) -> None:
        """Takes the last ``extend`` back."""
        for e, c in zip(reversed(entries), reversed(counts)):
            e.length -= c
            while len(e.pages) > -(-e.length // PAGE_TOKENS):
                self.holders[e.pages[-1]] = 0
                self.free.append(e.pages.pop())

    def fork(self, sequences, copy=None, ending=()):
        """(new sequences, pages to copy).  ``copy`` is called with the pages before anything changes; what it raises leaves the book
        as it is.  The sequences ``ending`` end with it, and their pages serve the new ones."""
        entries, ends = [self.of(s) for s in sequences], [self.of(s) for s in ending]
        if len(set(ending)) != len(ends) or not set(ending).isdisjoint(sequences):
            raise ValueError("a sequence that ends is named twice")
        parted = [e for e in entries if e.length % PAGE_TOKENS]
        left = Counter(page for e in ends for page in e.pages)  # how many of a page's holders end
        freed = [page for page, n in left.items() if n == self.holders[page]]
        if len(parted) > len(self.free) + len(freed):
            raise RuntimeError(f"out of pages: {len(parted)} needed, {len(self.free) + len(freed)} free")
        stay = max(0, len(self.free) - len(parted))
        taken = (self.free[:stay - 1:-1] if stay else self.free[::-1]) + freed
        pairs = [(e.pages[-1], page) for e, page in zip(parted, taken)]
        if copy is not None:
            copy(pairs)
        del self.free[stay:]
        self.release(list(ending))
        given = {page for _, page in pairs}
        self.free[stay:] = [page for page in self.free[stay:] if page not in given]
        new, at = [], iter(taken)
        for e in entries:
            pages = list(e.pages)
            shared = pages
            if e.length % PAGE_TOKENS:
                shared = pages[:-1]
                pages[-1] = next(at)
                self.holders[pages[-1]] = 1
            for page in shared:
                self.holders[page] += 1
            e.supersede()
            new.append(self._new(_Sequence(pages, e.length)))
        return new, pairs

    def release(self, sequences) -> None:
        entries = [self.of(s) for s in sequences]
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence is named twice")
        for s, e in zip(sequences, entries):
            e.supersede()
            for page in reversed(e.pages):
                self.holders[page] -= 1
                if self.holders[page] == 0:
                    self.free.append(page)
            del self.sequences[s]

    def compact(self, copy=None):
        """(pages in use, pages to copy); ``copy`` as for ``fork``."""
        pages = len(self.holders)
        used = pages - len(self.free)
        behind = [p for p in range(used, pages) if self.holders[p]]
        room = [p for p in range(used) if not self.holders[p]]
        pairs = list(zip(behind, room))
        if copy is not None:
            copy(pairs)
        moved = dict(pairs)
        for a, b in pairs:
            self.holders[b], self.holders[a] = self.holders[a], 0
        for e in self.sequences.values():
            e.pages = [moved.get(p, p) for p in e.pages]
            e.supersede()
        self.free = list(range(pages - 1, used - 1, -1))
        self.epoch = object()
        return used, pairs
