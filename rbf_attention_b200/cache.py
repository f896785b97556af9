"""The paged 8-bit cache of a model: which pages its sequences have, on the host, around the operators that write, read and move
them (``ops.cache_append``, ``cache_attention``, ``cache_read``, ``cache_copy_pages``). The reference has no cache: its
generation runs the whole prefix again for every token (train_rbf_transformer.py:446-530).

A step of a model is ``begin(new)`` - pages for the new tokens, before anything runs - then ``append`` and ``attend`` in every
layer, then ``end()``. All calls belong on one stream: a page that one call frees may be another's in the next."""

from __future__ import annotations

import heapq

import torch

from . import ops

PAGE_TOKENS = 256


class PagedCache:
    """Keys and values of up to ``max_sequences`` sequences of up to ``max_length`` tokens in a pool of ``num_pages`` pages of 256
    tokens (default: enough for all of them), every layer with the same pages. Blocks of 16 tokens are held in 8 bits with a
    scale per block and head, the last few tokens of a sequence in ``dtype``.

    ``pages`` (layers, pages, heads, bytes), ``page_table`` (max_sequences, pages of a sequence) and ``lengths`` (max_sequences,)
    stay where they are: a CUDA graph of a step on all sequences can be replayed between ``begin`` and ``end`` (or ``abort``, which
    takes a cache whose ``append`` has been captured to have been written)."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, max_sequences: int, max_length: int,
                 num_pages: int | None = None, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"unsupported dtype {dtype} (bfloat16 or float16)")
        if min(num_layers, num_heads, max_sequences, max_length) < 1:
            raise ValueError("layers, heads, sequences and the length must be positive")
        self.head_dim, self.dtype, self.max_length = head_dim, dtype, max_length
        columns = -(-max_length // PAGE_TOKENS)
        num_pages = max_sequences * columns if num_pages is None else num_pages
        self.pages = torch.empty(num_layers, num_pages, num_heads, ops.cache_page_bytes(head_dim), dtype=torch.uint8, device=device)
        self.page_table = torch.full((max_sequences, columns), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_sequences, dtype=torch.int32, device=device)
        self._held = [[] for _ in range(max_sequences)]         # pages of each sequence, in order
        self._tokens = [0] * max_sequences
        self._users = [0] * num_pages                           # sequences that have the page
        self._free = list(range(num_pages))                     # a heap: low pages first
        self._step = None
        self._captured = False                                  # a graph may append: nothing is seen of its replays

    # -- what there is ---------------------------------------------------------------------------
    @property
    def max_sequences(self) -> int:
        return len(self._tokens)

    @property
    def num_pages(self) -> int:
        return self.pages.shape[1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        """Tokens of a sequence."""
        return self._tokens[self._slot(sequence)]

    def _slot(self, sequence: int) -> int:
        if not 0 <= sequence < self.max_sequences:
            raise ValueError(f"sequence {sequence} is not in [0, {self.max_sequences})")
        return sequence

    def _between_steps(self, what: str) -> None:
        if self._step is not None:
            raise RuntimeError(f"{what} between begin() and end()")

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._users[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            heapq.heappush(self._free, page)

    def _write_rows(self, sequences) -> None:
        """The table's rows of these sequences, and their lengths, on the device."""
        sequences = sorted(set(sequences))
        if not sequences:
            return
        rows = torch.full((len(sequences), self.page_table.shape[1]), -1, dtype=torch.int32)
        for i, s in enumerate(sequences):
            rows[i, :len(self._held[s])] = torch.tensor(self._held[s], dtype=torch.int32)
        at = torch.tensor(sequences, device=self.page_table.device)
        self.page_table.index_copy_(0, at, rows.to(self.page_table.device))
        lengths = torch.tensor([self._tokens[s] for s in sequences], dtype=torch.int32)
        self.lengths.index_copy_(0, at, lengths.to(self.lengths.device))

    # -- a step ----------------------------------------------------------------------------------
    def begin(self, new, sequences=None) -> None:
        """Pages for ``new`` tokens (a number, or one for each) of all sequences, or of the listed ones, which are the batch
        of the following calls, in this order. A page that a sequence shares with others and would write into is copied first.
        Raises without any change if there are not enough pages or a sequence would get longer than ``max_length``."""
        self._between_steps("begin()")
        batch = list(range(self.max_sequences)) if sequences is None else [self._slot(s) for s in sequences]
        if len(set(batch)) != len(batch):
            raise ValueError("a sequence is in the batch twice")
        counts = [new] * len(batch) if isinstance(new, int) else [int(n) for n in new]
        if len(counts) != len(batch) or min(counts, default=0) < 0:
            raise ValueError(f"new tokens for {len(batch)} sequences, got {counts}")
        for s, n in zip(batch, counts):
            if self._tokens[s] + n > self.max_length:
                raise ValueError(f"sequence {s} would have {self._tokens[s] + n} tokens, the cache holds {self.max_length}")
        # the last user of a shared page writes into it, the others into copies
        copied, users = [], dict()
        wanted = 0
        for s, n in zip(batch, counts):
            if n == 0:
                continue
            wanted += -(-(self._tokens[s] + n) // PAGE_TOKENS) - len(self._held[s])
            if self._tokens[s] % PAGE_TOKENS:
                page = self._held[s][-1]
                left = users.get(page, self._users[page])
                if left > 1:
                    copied.append(s)
                    wanted += 1
                users[page] = left - 1
        if wanted > len(self._free):
            raise RuntimeError(f"the cache is full: {wanted} pages are needed, {len(self._free)} of {self.num_pages} are free")
        changed, src, dst = list(copied), [], []
        for s in copied:
            src.append(self._held[s][-1])
            dst.append(self._take())
            self._users[src[-1]] -= 1
            self._held[s][-1] = dst[-1]
        for s, n in zip(batch, counts):
            more = -(-(self._tokens[s] + n) // PAGE_TOKENS) - len(self._held[s]) if n else 0
            if more > 0:
                self._held[s] += [self._take() for _ in range(more)]
                changed.append(s)
        if src:
            ops.cache_copy_pages(self.pages, src, dst)
        self._write_rows(changed)
        uniform = len(set(counts)) <= 1
        device = self.lengths.device
        fresh = None if uniform else torch.tensor(counts, dtype=torch.int32).to(device)
        if sequences is None:
            at, table, lengths = None, self.page_table, self.lengths
        else:
            at = torch.tensor(batch, dtype=torch.int64).to(device)
            table, lengths = self.page_table.index_select(0, at), self.lengths.index_select(0, at)
        self._step, self._written = (batch, counts, at, table, lengths, fresh), False

    def _current(self, what: str):
        if self._step is None:
            raise RuntimeError(f"{what} outside of begin() and end()")
        return self._step

    @property
    def positions(self) -> torch.Tensor:
        """Tokens that each sequence of the step's batch had before it (int32, on the device)."""
        return self._current("positions")[4]

    @property
    def counts(self) -> list[int]:
        """New tokens of each sequence of the step's batch."""
        return list(self._current("counts")[1])

    def _layer(self, layer: int) -> torch.Tensor:
        if not 0 <= layer < self.pages.shape[0]:
            raise ValueError(f"layer {layer} is not in [0, {self.pages.shape[0]})")
        return self.pages[layer]

    def _check_rows(self, name: str, x: torch.Tensor, counts) -> None:
        if x.dtype != self.dtype or x.shape[-1] != self.head_dim:
            raise ValueError(f"{name} must be {self.dtype} with head dim {self.head_dim}, got {x.dtype} {tuple(x.shape)}")
        if x.dim() == 4 and x.shape[2] < max(counts, default=0):
            raise ValueError(f"{name} has {x.shape[2]} tokens, the step {max(counts)}")

    def _fresh(self, x, counts, fresh):
        """What the operators get as new lengths: nothing where all of the tokens are new ones."""
        if fresh is None and counts and x.shape[2] != counts[0]:
            fresh = torch.full((len(counts),), counts[0], dtype=torch.int32, device=self.lengths.device)
        return fresh

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's tokens of one layer: k, v (batch, heads, T, head_dim), padded to T tokens behind the new ones."""
        _batch, counts, _at, table, lengths, fresh = self._current("append()")
        self._check_rows("k", k, counts)
        self._check_rows("v", v, counts)
        self._written = True
        self._captured = self._captured or ops.capturing(self.pages.device)
        ops.cache_append(self._layer(layer), table, lengths, k, v, self._fresh(k, counts, fresh))

    def attend(self, layer: int, q: torch.Tensor, softmax: bool = True) -> torch.Tensor:
        """RBF attention of the step's tokens, which have been appended, to all that their sequences hold: q (batch, query
        heads, T, head_dim) -> the same shape."""
        _batch, counts, _at, table, lengths, fresh = self._current("attend()")
        self._check_rows("q", q, counts)
        return ops.cache_attention(q, self._layer(layer), table, lengths, self._fresh(q, counts, fresh), softmax=softmax)

    def end(self) -> None:
        """The step's tokens belong to their sequences."""
        batch, counts, at, _table, _lengths, fresh = self._current("end()")
        for s, n in zip(batch, counts):
            self._tokens[s] += n
        more = fresh if fresh is not None else counts[0] if counts else 0
        if at is None:
            self.lengths += more
        elif fresh is not None:
            self.lengths.index_add_(0, at, fresh)
        else:
            self.lengths.index_add_(0, at, torch.full_like(at, more, dtype=torch.int32))
        self._step = None

    def abort(self, written: bool | None = None) -> None:
        """Leaves the step without its tokens. If any layer has been written, the step's sequences are freed: tokens that fill a
        block up take the place of the ones that were held in 16 bits until then. Otherwise the pages for them are free again.
        ``written``: whether one has been. Without it, if ``append`` was called in the step, or ever while a graph was captured, which
        may have been replayed in it; operators that were called on ``pages`` directly are the caller's to tell."""
        batch, counts, *_ = self._current("abort()")
        self._step = None
        if self._written or self._captured if written is None else written:
            self.free([s for s, n in zip(batch, counts) if n])
            return
        for s in batch:
            kept = -(-self._tokens[s] // PAGE_TOKENS)
            for page in self._held[s][kept:]:
                self._drop(page)
            self._held[s] = self._held[s][:kept]
        self._write_rows(batch)

    def read(self, layer: int, sequences=None, count: int | None = None, first=None):
        """(k, v) (batch, heads, count, head_dim) as the cache holds them, from token ``first`` (one for each, default 0) on,
        zeros behind a sequence's last token; ``count``: by default as many as the longest one has."""
        batch = list(range(self.max_sequences)) if sequences is None else [self._slot(s) for s in sequences]
        if count is None:
            count = max((self._tokens[s] for s in batch), default=0)
        at = torch.tensor(batch, dtype=torch.int64).to(self.lengths.device)
        if first is not None:
            first = torch.tensor(list(first), dtype=torch.int32).to(self.lengths.device)
        return ops.cache_read(self._layer(layer), self.page_table.index_select(0, at), self.lengths.index_select(0, at),
                              self.head_dim, self.dtype, count, first=first)

    # -- pages -----------------------------------------------------------------------------------
    def fork(self, source: int, sequences) -> None:
        """The empty ``sequences`` become copies of ``source``, on the same pages: only a last page that is not full is copied,
        when a sequence that shares it gets its next token."""
        self._between_steps("fork()")
        self._slot(source)
        targets = [self._slot(s) for s in sequences]
        if len(set(targets)) != len(targets) or any(self._tokens[s] or s == source for s in targets):
            raise ValueError(f"sequences {targets} must be different, empty and not {source}")
        for s in targets:
            self._held[s] = list(self._held[source])
            self._tokens[s] = self._tokens[source]
            for page in self._held[s]:
                self._users[page] += 1
        self._write_rows(targets)

    def free(self, sequences) -> None:
        """The sequences are empty; pages that no other sequence has are free."""
        self._between_steps("free()")
        batch = {self._slot(s) for s in sequences}
        for s in batch:
            for page in self._held[s]:
                self._drop(page)
            self._held[s], self._tokens[s] = [], 0
        self._write_rows(batch)

    def compact(self) -> int:
        """Moves pages so that the used ones are the first of the pool, in all layers with one launch; returns how many."""
        self._between_steps("compact()")
        used = [p for p, n in enumerate(self._users) if n]
        move = dict(zip([p for p in used if p >= len(used)], [p for p in range(len(used)) if not self._users[p]]))
        if move:
            ops.cache_copy_pages(self.pages, list(move), list(move.values()))
            for src, dst in move.items():
                self._users[dst], self._users[src] = self._users[src], 0
            self._held = [[move.get(p, p) for p in pages] for pages in self._held]
            self._free = [p for p, n in enumerate(self._users) if not n]
            heapq.heapify(self._free)
            self._write_rows(s for s, pages in enumerate(self._held) if pages)
        return len(move)

    def resize(self, num_pages: int) -> None:
        """Another pool of ``num_pages`` pages, after ``compact``; fewer than are used are refused. ``pages`` is a new tensor."""
        used = sum(1 for n in self._users if n)
        if num_pages < used:
            raise ValueError(f"{used} pages are used, {num_pages} are too few")
        self.compact()
        pages = self.pages.new_empty(self.pages.shape[0], num_pages, *self.pages.shape[2:])
        pages[:, :used] = self.pages[:, :used]
        self.pages = pages
        self._users = self._users[:used] + [0] * (num_pages - used)
        self._free = list(range(used, num_pages))
