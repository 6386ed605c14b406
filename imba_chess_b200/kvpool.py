"""Paged, device-resident KV pool and the token sequences that live in it.

One pool per model per device: a ``[num_pages, page_elems]`` tensor in the
model dtype whose page layout is ``[layer][K: H x 16 x d_qk | V: H x 16 x
d_v]`` (include/imba_b200.h).  A ``KVSequence`` is an append-only list of
pages plus a token count; token ``t`` lives at physical slot
``pages[t // 16] * 16 + t % 16``.

The reference keeps two kinds of KV stores (src/imba_chess/eval/
actor_server.py:206-344):

* a game's growing root prefix (``_GameState``), re-built by ``torch.cat``
  on every incremental extension, and
* a turn's decode-node arena (``_KVArena``), a ``[L, H, capacity, d]`` tensor
  grown by doubling, whose rows are minted consecutively in wave order.

Both map onto ``KVSequence``: appending never moves existing tokens, so a
turn's snapshot of a game prefix (a sequence plus the length it had) stays
valid while the game grows, and arena row ``r`` of a turn is token ``r`` of
that turn's arena sequence - the same row ids the reference mints.
Sequences are reference-counted; pages return to the pool when the last
holder releases them.

A pool can also hold its tokens in 8 bits (``dtype=torch.float8_e4m3fn``, half
of bf16): e4m3 codes with one power-of-two scale for each block of a page's 16
tokens, head, and K or V.  ``data`` then holds the codes (V's tokens lie in
pairs, ``[H][8][d_v][2]``) and ``scales`` the scales' exponents, one byte per
block (0: an empty block).  A block's scale grows with its tokens and never
shrinks, so pages start afresh when they are handed out: ``alloc`` notes them
and ``begin_pages`` clears their scales on the stream of the next call that
writes to the pool.  Those pages may be another stream's, before and after, so
that clearing waits for what the pool's other streams have enqueued, and their
next calls wait for it.  ``imba_chess_b200.paged`` has the operators on a pool.
"""

from __future__ import annotations

from itertools import chain

import numpy as np
import torch

from . import _native

PAGE = _native.PAGE_TOKENS


class KVPoolExhausted(RuntimeError):
    """The pool has fewer free pages than a request needs."""


def to_device(host: torch.Tensor, device: torch.device) -> torch.Tensor:
    """A host tensor's copy on ``device``, enqueued on its current stream: the
    host goes on at once, through pinned memory that is not handed out again
    before the copy is done."""
    if device.type != "cuda" or host.numel() == 0:
        return host.to(device)
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("host data cannot be copied in a capture (its replays would copy it again): "
                               "put it on the device before")
        pinned = torch.empty(host.shape, dtype=host.dtype, device="cpu", pin_memory=True)
        return pinned.copy_(host).to(device, non_blocking=True)


class KVPool:
    def __init__(self, *, num_layers: int, num_heads: int, attention_dim: int, linear_dim: int,
                 num_pages: int, dtype: torch.dtype, device: torch.device) -> None:
        if num_pages <= 0:
            raise ValueError("num_pages must be positive")
        self.num_layers, self.num_heads = int(num_layers), int(num_heads)
        self.attention_dim, self.linear_dim = int(attention_dim), int(linear_dim)
        self.page_elems = num_layers * num_heads * PAGE * (attention_dim + linear_dim)
        self.num_pages = int(num_pages)
        self.dtype = dtype
        self.device = device
        self.scales: torch.Tensor | None = None
        with torch.inference_mode(False):  # (pages are emptied in place, in that mode and outside of it)
            self._make(num_layers, num_heads, attention_dim, linear_dim)
        self._free = np.arange(self.num_pages - 1, -1, -1, dtype=np.int64).tolist()
        self._fresh: list[int] = []  # pages in 8 bits handed out since begin_pages()
        self._streams: dict[int, torch.cuda.Stream] = {}  # that calls on a pool in 8 bits ran on, by handle
        self._ordered: set[int] = set()  # of them, those behind the last begin_pages()
        self._begun_on: torch.cuda.Stream | None = None  # where that one, or at first the making of the pool, ran
        if self.scales is not None and self.data.is_cuda:
            self._began(torch.cuda.current_stream(self.data.device))
        self.desc = _native.PoolDesc(self.data.data_ptr(), self.num_pages)

    def _began(self, stream: torch.cuda.Stream) -> None:
        self._streams[stream.cuda_stream] = self._begun_on = stream
        self._ordered = {stream.cuda_stream}

    def _make(self, num_layers: int, num_heads: int, attention_dim: int, linear_dim: int) -> None:
        dtype, device = self.dtype, self.device
        if dtype == torch.float8_e4m3fn:
            dims = (32, 64, 96, 128)
            if attention_dim not in dims or linear_dim not in dims or (
                    attention_dim != linear_dim and max(attention_dim, linear_dim) > 64):
                raise ValueError(f"a pool in 8 bits takes head dimensions of {dims} (equal ones above 64), "
                                 f"got {attention_dim} / {linear_dim}")
            codes = self.num_pages * self.page_elems
            memory = torch.zeros(codes + self.num_pages * num_layers * 2 * num_heads, dtype=torch.uint8, device=device)
            self.data = memory[:codes].view(torch.float8_e4m3fn).view(self.num_pages, self.page_elems)
            self.scales = memory[codes:].view(self.num_pages, num_layers, 2, num_heads)
        else:
            self.data = torch.zeros((self.num_pages, self.page_elems), dtype=dtype, device=device)
        # what the operators on the pool report to (made here: in a capture, each replay would clear it)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def page_bytes(self) -> int:
        scales = 0 if self.scales is None else 2 * self.num_layers * self.num_heads
        return self.page_elems * self.data.element_size() + scales

    def alloc(self, n: int) -> list[int]:
        if n > len(self._free):
            raise KVPoolExhausted(
                f"KV pool exhausted: need {n} pages, {len(self._free)} of {self.num_pages} free"
            )
        if n <= 0:
            return []
        out = self._free[-n:]
        del self._free[-n:]
        out.reverse()
        if self.scales is not None:
            self._fresh.extend(out)
        return out

    def begin_pages(self, pages=None) -> None:
        """Empty the blocks of ``pages`` (default: the pages handed out since
        the last call) of a pool in 8 bits, on the current stream.  The
        operators and the model's steps call this; a caller that recycles
        pages without ``alloc``, or captures a CUDA graph after one, does.
        Behind all that the pool's other streams, which have to live as long
        as it does, have enqueued (a graph's replays are not known here: order
        them yourself)."""
        if self.scales is None or (pages is None and not self._fresh):
            return
        if self.data.is_cuda:
            with torch.cuda.device(self.data.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("pages are not emptied in a capture: call pool.begin_pages() before the capture")
        if pages is None:
            pages, self._fresh = self._fresh, []
        ids = torch.as_tensor(pages, dtype=torch.int64, device="cpu")
        if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= self.num_pages):
            raise ValueError("begin_pages: page id outside the pool")
        if self.data.is_cuda:
            stream = torch.cuda.current_stream(self.data.device)
            for other in self._streams.values():
                if other.cuda_stream != stream.cuda_stream:
                    stream.wait_stream(other)
            self._began(stream)
        self.scales.index_fill_(0, to_device(ids, self.data.device), 0)

    def join_stream(self) -> None:
        """The current stream is one that works on this pool in 8 bits: its
        next work comes after the last ``begin_pages`` (at first, after the
        making of the pool), and the next ``begin_pages`` after its work."""
        stream = torch.cuda.current_stream(self.data.device)
        with torch.cuda.device(self.data.device):
            if torch.cuda.is_current_stream_capturing():
                return  # (a capture cannot wait for work outside of it)
        if self._begun_on is not None:
            stream.wait_stream(self._begun_on)
        self._streams[stream.cuda_stream] = stream
        self._ordered.add(stream.cuda_stream)

    def release_pages(self, pages: list[int]) -> None:
        self._free.extend(reversed(pages))


class KVSequence:
    """Append-only token sequence in a ``KVPool`` (reference-counted)."""

    __slots__ = ("pool", "pages", "length", "refs")

    def __init__(self, pool: KVPool) -> None:
        self.pool = pool
        self.pages: list[int] = []
        self.length = 0
        self.refs = 1

    def retain(self) -> "KVSequence":
        if self.refs <= 0:
            raise RuntimeError("retain() on a released KV sequence")
        self.refs += 1
        return self

    def release(self) -> None:
        if self.refs <= 0:
            return
        self.refs -= 1
        if self.refs == 0:
            self.pool.release_pages(self.pages)
            self.pages = []
            self.length = 0

    def reserve(self, n: int) -> np.ndarray:
        """Append ``n`` token slots; returns their physical slots (int64)."""
        start = self.length
        need_pages = -(-(start + n) // PAGE) - len(self.pages)
        if need_pages > 0:
            self.pages.extend(self.pool.alloc(need_pages))
        self.length = start + n
        return self.slots(start, start + n)

    @staticmethod
    def reserve_many(seqs: "list[KVSequence]", counts) -> np.ndarray:
        """``seqs[i].reserve(counts[i])`` for every i, in order; returns all
        the new slots concatenated (int64), computed in one pass over the
        sequences' page lists instead of one small array per sequence."""
        n = len(seqs)
        starts = np.empty(n, dtype=np.int64)
        for i, (s, c) in enumerate(zip(seqs, counts)):
            start = s.length
            need = -(-(start + int(c)) // PAGE) - len(s.pages)
            if need > 0:
                s.pages.extend(s.pool.alloc(need))
            s.length = start + int(c)
            starts[i] = start
        cnt = np.asarray(counts, dtype=np.int64).reshape(n)
        total = int(cnt.sum())
        if total == 0:
            return np.zeros(0, dtype=np.int64)
        npg = np.fromiter((len(s.pages) for s in seqs), dtype=np.int64, count=n)
        pbase = np.zeros(n, dtype=np.int64)
        np.cumsum(npg[:-1], out=pbase[1:])
        cat = np.fromiter(chain.from_iterable(s.pages for s in seqs), dtype=np.int64, count=int(npg.sum()))
        rbase = np.zeros(n, dtype=np.int64)
        np.cumsum(cnt[:-1], out=rbase[1:])
        t = np.repeat(starts, cnt) + np.arange(total, dtype=np.int64) - np.repeat(rbase, cnt)
        return cat[np.repeat(pbase, cnt) + t // PAGE] * PAGE + t % PAGE

    def truncate(self, length: int, num_pages: int) -> None:
        """Undo reservations: back to ``length`` tokens on the first
        ``num_pages`` pages (values recorded before the reservations); the
        pages past them return to the pool."""
        if num_pages < len(self.pages):
            self.pool.release_pages(self.pages[num_pages:])
            del self.pages[num_pages:]
        self.length = min(self.length, int(length))

    def slots(self, start: int, stop: int) -> np.ndarray:
        t = np.arange(start, stop, dtype=np.int64)
        pages = np.asarray(self.pages, dtype=np.int64)
        return pages[t // PAGE] * PAGE + t % PAGE

    def slots_of(self, tokens) -> np.ndarray:
        t = np.asarray(tokens, dtype=np.int64)
        pages = np.asarray(self.pages, dtype=np.int64)
        return pages[t // PAGE] * PAGE + t % PAGE

    def page_array(self, length: int | None = None) -> np.ndarray:
        n = self.length if length is None else length
        return np.asarray(self.pages[: -(-n // PAGE)], dtype=np.int32)
