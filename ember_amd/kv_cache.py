"""A key/value cache in 4 bits (no counterpart in the reference, which has no
attention).

``KVCache`` holds the keys and values of several sequences in pages of a
common pool, 17/32 byte per element (``include/ember_amd.h`` describes the
format: 32 neighbours of a head row share a power of two and are rounded to
0, 0.5, 1, 1.5, 2, 3, 4 or 6 times it).  ``write`` appends rows, ``attention``
is the causal attention of the rows last appended over all that their
sequences hold, ``read`` gives the values back.  Lengths and the page table
are kept on the host and, for the kernels, on the device; a step uploads the
table where a sequence gets a new page, and its counts where they are given.
"""

from __future__ import annotations

from collections.abc import Sequence

import numpy as np

from ember_amd import _core as C
from ember_amd.tensor import Tensor, _need_tensor, _scale

GROUP = 32


def upload_ints(a) -> C._Tensor:
    """int32 values in device memory, an element of the buffer each."""
    return C._from_numpy(np.ascontiguousarray(a, np.int32).reshape(-1).view(np.float32))


def _bytes(n: int) -> C._Tensor:
    return C._Tensor((n + 3) // 4)


class KVCache:
    """Room for ``sequences`` sequences of up to ``tokens`` tokens each, of
    ``heads`` heads of ``head_dim`` (32, 64 or 128) elements, on ``pages`` pages
    of ``page_size`` tokens (a power of two from 16 on).  Without ``pages``
    there are enough for all sequences to be full; with fewer, ``write``
    raises ValueError when none is free."""

    def __init__(self, sequences: int, heads: int, head_dim: int, tokens: int, page_size: int = 64,
                 pages: int | None = None):
        if head_dim not in (32, 64, 128):
            raise ValueError(f"head_dim must be 32, 64 or 128, not {head_dim}")
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 65536, not {page_size}")
        if not 1 <= sequences <= 65535 or not 1 <= heads <= 65535 or tokens < 1:
            raise ValueError(f"sequences, heads and tokens must be positive (65535 at most for the first two), "
                             f"got {sequences}, {heads}, {tokens}")
        self.places = -(-tokens // page_size)
        if self.places * page_size > 2 ** 31 - 2 ** 16:
            raise ValueError(f"{tokens} tokens to a sequence are more than the cache can number")
        self.pages = sequences * self.places if pages is None else pages
        if not 1 <= self.pages < 2 ** 31:
            raise ValueError(f"pages must be from 1 to 2^31 - 1, not {self.pages}")
        self.sequences, self.heads, self.head_dim, self.tokens, self.page_size = sequences, heads, head_dim, tokens, page_size
        rows = self.pages * heads * page_size
        self._arrays = [_bytes(rows * head_dim // n) for n in (2, GROUP, 2, GROUP)]
        self.reset()

    def reset(self, sequence: int | None = None) -> None:
        """Empties the cache, or one sequence of it; its pages are free again."""
        if sequence is None:
            self._lengths = np.zeros(self.sequences, np.int32)
            self._table = np.full((self.sequences, self.places), -1, np.int32)
            self._free = list(range(self.pages - 1, -1, -1))
        else:
            row = self._table[self._index(sequence)]
            self._free += [int(p) for p in row[row >= 0][::-1]]
            row[:] = -1
            self._lengths[sequence] = 0
        self._device_table = self._device_lengths = None
        self._last = None

    def _index(self, sequence: int) -> int:
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"sequence {sequence} is out of range for a cache of {self.sequences}")
        return sequence

    @property
    def lengths(self) -> list[int]:
        """Tokens that each sequence holds."""
        return self._lengths.tolist()

    @property
    def nbytes(self) -> int:
        """Device memory of the codes and scales."""
        return sum(4 * a.size for a in self._arrays)

    def _view(self) -> tuple:
        if self._device_table is None:
            self._device_table = upload_ints(self._table)
        return (*self._arrays, self._device_table, self.pages, self.heads, self.page_size, self.head_dim,
                self.sequences, self.places)

    def _counts(self, T: int, count) -> np.ndarray:
        if count is None:
            return np.full(self.sequences, T, np.int32)
        n = np.asarray(count)
        if n.shape != (self.sequences,) or n.dtype.kind not in "iu" or (n < 0).any() or (n > T).any():
            raise ValueError(f"count must be {self.sequences} integers from 0 to {T}, got {count!r}")
        return n.astype(np.int32)

    def _append(self, k, k_at: int, v, v_at: int, T: int, strides: tuple[int, int, int], count) -> None:
        """Writes T rows per sequence from cores k and v, from their elements
        k_at and v_at on."""
        n = self._counts(T, count)
        after = self._lengths.astype(np.int64) + n
        if (after > self.tokens).any():
            b = int(np.argmax(after > self.tokens))
            raise ValueError(f"sequence {b} would hold {after[b]} tokens, and has room for {self.tokens}")
        have = -(-self._lengths.astype(np.int64) // self.page_size)
        need = -(-after // self.page_size) - have
        if need.sum() > len(self._free):
            raise ValueError(f"{int(need.sum())} new pages are needed, and {len(self._free)} are free")
        taken = [(b, i) for b in np.nonzero(need)[0] for i in range(have[b], have[b] + need[b])]
        for place in taken:
            self._table[place] = self._free.pop()
        if taken:
            self._device_table = None
        try:
            if self._device_lengths is None:
                self._device_lengths = upload_ints(self._lengths)
            start, counts = self._device_lengths, None if count is None else upload_ints(n)
            behind = C._Tensor(self.sequences)
            C._kv_cache_write(self._view(), k, k_at, v, v_at, T, *strides, start, counts, behind)
        except Exception:
            for place in reversed(taken):
                self._free.append(int(self._table[place]))
                self._table[place] = -1
            self._device_table = None
            raise
        self._device_lengths, self._lengths = behind, after.astype(np.int32)
        self._last = (T, start, counts)

    def write(self, k: Tensor, v: Tensor, count: Sequence[int] | None = None) -> None:
        """Appends the rows k and v, (sequences, T, heads, head_dim); of sequence
        b the first ``count[b]`` (all without count: pad a ragged batch behind)."""
        for name, t in (("k", k), ("v", v)):
            _need_tensor(t, f"KVCache.write() {name}")
        if len(k.shape) != 4 or k.shape != v.shape or k.shape[0] != self.sequences or k.shape[2:] != (self.heads, self.head_dim):
            raise ValueError(f"k and v must be ({self.sequences}, T, {self.heads}, {self.head_dim}), got {k.shape} and {v.shape}")
        T = k.shape[1]
        self._append(k._core, 0, v._core, 0, T, (T * self.heads * self.head_dim, self.head_dim, self.heads * self.head_dim), count)

    def _attend(self, q, q_at: int, T: int, q_heads: int, strides: tuple[int, int, int], causal: bool, scale: float | None):
        if self._last is None:
            raise RuntimeError("write() must run before attention()")
        if T != self._last[0]:
            raise ValueError(f"q has {T} rows to a sequence, and the last write had {self._last[0]}")
        if q_heads % self.heads:
            raise ValueError(f"{q_heads} query heads are no multiple of the cache's {self.heads}")
        _, start, counts = self._last
        return C._kv_cache_attention(self._view(), q, q_at, T, q_heads, _scale(self.head_dim, scale), causal, *strides, start, counts)

    def attention(self, q: Tensor, causal: bool = True, scale: float | None = None) -> tuple[Tensor, Tensor]:
        """(O, LSE) of the rows last written: q (sequences, T, query heads,
        head_dim) with T as in that ``write``, O like q, LSE (sequences, query
        heads, T).  Query head h reads cache head h // (query heads / heads).
        Row t of sequence b sees the tokens up to its own (all that the sequence
        holds where not ``causal``); rows past ``count`` get 0 and -infinity."""
        _need_tensor(q, "KVCache.attention() q")
        if len(q.shape) != 4 or q.shape[0] != self.sequences or q.shape[3] != self.head_dim or q.shape[2] < 1:
            raise ValueError(f"q must be ({self.sequences}, T, query heads, {self.head_dim}), got {q.shape}")
        _, T, H, D = q.shape
        o, lse = self._attend(q._core, 0, T, H, (T * H * D, D, H * D), causal, scale)
        return Tensor._from_core(o, q.shape), Tensor._from_core(lse, (self.sequences, H, T))

    def read(self) -> tuple[Tensor, Tensor]:
        """The keys and values held, (sequences, longest length, heads,
        head_dim), with zeros past a sequence's length."""
        T = int(self._lengths.max())
        k, v = C._kv_cache_read(self._view(), T, upload_ints(np.zeros(self.sequences)), upload_ints(self._lengths))
        shape = (self.sequences, T, self.heads, self.head_dim)
        return Tensor._from_core(k, shape), Tensor._from_core(v, shape)


__all__ = ["KVCache"]
