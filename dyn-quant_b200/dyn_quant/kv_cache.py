"""Paged 4-bit KV cache of one attention layer: append, attend, evict.

Keys and values are kept in the INT4 row format of the weights (one group of
head_dim values per token and KV head, FP16 scale and zero-point, quantized
bit for bit as dyn_quant.quantize does it): 4.25 bits a number at head_dim 128
(4.5 at 64) instead of 16.  Attention reads the codes directly; a running
attention weight per slot can be kept and the cache cut to the slots that have
received the most.  No counterpart in the reference, whose scope is the linear
layers on either side of the attention; dyn_quant.attention.Int4Attention joins
them.

A decode step issues kernel launches only (lengths live on the device), so it
can be captured in a CUDA graph; what does not fit the pages is reported in the
device error word (Int4KVCache.check); calls on one cache must be stream-ordered.  Pages
may be shared by sequences with a common beginning, but only to be read: append,
evict and accumulated weights need pages that one sequence owns.  There are no
gradients.
"""
from __future__ import annotations

import math
from typing import Sequence

import torch

import dyn_quant

UNIT_TOKENS = 16  # slots of one unit

# Bits 16 .. 18 (append, evict) and 20 .. 22 (attend) of the device error word
_ERRORS = ("a page outside the pool", "a length, count or start outside the sequence's pages",
           "a wait for the kernel's own copies or products gave up")


def unit_bytes(head_dim: int) -> int:
    """Bytes of 16 slots of one KV head: K codes, V codes, scales and zeros."""
    return UNIT_TOKENS * head_dim + 8 * UNIT_TOKENS


class Int4KVCache:
    """The 4-bit KV cache of one layer for a fixed set of sequence slots.

    Args:
        n_seqs:     sequences (batch slots); at most 1024.
        n_pages:    pages of the pool, shared out to the sequences by `page_table`.
        n_kv_heads: KV heads.
        head_dim:   64 or 128.
        page_size:  token slots of a page, a multiple of 16.
        max_pages:  pages a sequence may have (default: n_pages).
        units, meta, page_table: existing buffers to use instead of new ones.

    Buffers (all on the device, all plain tensors that may be read and copied):
        units       uint8 [n_pages, n_kv_heads, page_size / 16, unit_bytes]; the
                    layout is dq_kv_cache_t's in include/dq_abi.h.
        mass        float32 [n_pages, n_kv_heads, page_size], a slot's accumulated
                    attention weight; pos int32, the position of its token.
        lengths     int32 [n_seqs], slots in use; evicted int32 [n_seqs], tokens
                    evicted so far (the next position is lengths + evicted).
        page_table  int32 [n_seqs, max_pages], -1 where there is no page.
        meta        one int32 buffer behind mass, pos, lengths and evicted.

    Pages hold 16-slot units, so new pages need no clearing: nothing behind
    `lengths` is read into a result (append with `at` above a length moves it past
    slots that then are).
    """

    def __init__(self, n_seqs: int, n_pages: int, n_kv_heads: int, head_dim: int = 128, page_size: int = 64,
                 max_pages: int | None = None, device: torch.device | str | None = None, *,
                 units: torch.Tensor | None = None, meta: torch.Tensor | None = None,
                 page_table: torch.Tensor | None = None) -> None:
        if head_dim not in (64, 128):
            raise RuntimeError(f"head_dim must be 64 or 128, got {head_dim}")
        if page_size <= 0 or page_size % UNIT_TOKENS != 0:
            raise RuntimeError(f"page_size must be a positive multiple of {UNIT_TOKENS}, got {page_size}")
        if n_seqs < 1 or n_pages < 1 or n_kv_heads < 1:
            raise RuntimeError("n_seqs, n_pages and n_kv_heads must be positive")
        if max_pages is None:
            max_pages = n_pages
        if max_pages < 1:
            raise RuntimeError("max_pages must be positive")
        dyn_quant._require_extension()
        dev = torch.device(device if device is not None else "cuda")
        if dev.type != "cuda":
            raise RuntimeError("the KV cache lives on a CUDA device")
        self.n_seqs, self.n_pages, self.n_kv_heads = n_seqs, n_pages, n_kv_heads
        self.head_dim, self.page_size, self.max_pages = head_dim, page_size, max_pages
        shape = (n_pages, n_kv_heads, page_size // UNIT_TOKENS, unit_bytes(head_dim))
        self.units = units if units is not None else torch.empty(shape, dtype=torch.uint8, device=dev)
        if tuple(self.units.shape) != shape:
            raise RuntimeError(f"units must have shape {shape}, got {tuple(self.units.shape)}")
        slots = n_pages * n_kv_heads * page_size
        self.meta = meta if meta is not None else torch.zeros(2 * slots + 2 * n_seqs, dtype=torch.int32, device=dev)
        if self.meta.dtype != torch.int32 or tuple(self.meta.shape) != (2 * slots + 2 * n_seqs,) \
                or not self.meta.is_contiguous():
            raise RuntimeError(f"meta must be a contiguous int32 tensor of {2 * slots + 2 * n_seqs} values")
        self.mass = self.meta[:slots].view(torch.float32).view(n_pages, n_kv_heads, page_size)
        self.pos = self.meta[slots:2 * slots].view(n_pages, n_kv_heads, page_size)
        self.lengths = self.meta[2 * slots:2 * slots + n_seqs]
        self.evicted = self.meta[2 * slots + n_seqs:]
        self.page_table = page_table if page_table is not None else \
            torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=dev)
        if tuple(self.page_table.shape) != (n_seqs, max_pages):
            raise RuntimeError(f"page_table must have shape {(n_seqs, max_pages)}, got {tuple(self.page_table.shape)}")
        self._arrivals = torch.zeros(n_seqs * (1 + n_kv_heads), dtype=torch.int32,
                                     device=self.units.device)
        self._h = dyn_quant._C.KVCache(self.units, self.mass, self.pos, self.lengths, self.evicted, self.page_table,
                                       self._arrivals)

    def assign(self, seq: int, pages: Sequence[int]) -> None:
        """Give sequence `seq` these pages, in slot order (a copy from the host)."""
        pages = [int(p) for p in pages]
        if not 0 <= seq < self.n_seqs:
            raise RuntimeError(f"sequence {seq} out of range")
        if len(pages) > self.max_pages:
            raise RuntimeError(f"{len(pages)} pages for a sequence, at most {self.max_pages}")
        if any(not 0 <= p < self.n_pages for p in pages):
            raise RuntimeError("page index outside the pool")
        if len(set(pages)) != len(pages):
            raise RuntimeError("a sequence cannot have a page twice")
        row = torch.full((self.max_pages,), -1, dtype=torch.int32)
        row[:len(pages)] = torch.tensor(pages, dtype=torch.int32)
        self.page_table[seq].copy_(row)

    def reset(self, seq: int | None = None) -> None:
        """Empty one sequence, or all of them (pages stay assigned)."""
        at = slice(None) if seq is None else seq
        if seq is None:
            self._arrivals.zero_()  # non-zero only after a call that reported a device error
        self.lengths[at] = 0
        self.evicted[at] = 0

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None,
               at: torch.Tensor | None = None, values: bool = False):
        """Quantize new keys and values into the cache (one kernel).

        Args:
            k, v:   [n_seqs, T, n_kv_heads, head_dim] float16, or [n_seqs,
                    n_kv_heads, head_dim] for one token each; slices of a fused
                    projection's output are read in place.
            counts: int32 [n_seqs], new tokens of each sequence (default: T each;
                    0 leaves a sequence as it is, unless `at` moves its end).
            at:     int32 [n_seqs], the slot of each sequence's first new token
                    (default: its length).  The length becomes at + counts, also
                    for 0 tokens.  Below the length it rewinds the sequence, e.g.
                    past rejected draft tokens; not below what an eviction has
                    rearranged.  Above the length the slots between count as in
                    use and must hold rows already, e.g. a prefix copied into
                    `units`, `mass` and `pos`.
            values: return (k, v) as the cache now holds them, float16, zero for
                    padding tokens.
        """
        return self._h.append(k, v, counts, at, values)

    def attend(self, q: torch.Tensor, scale: float | None = None, counts: torch.Tensor | None = None,
               accumulate: bool = False, out: torch.Tensor | None = None, return_lse: bool = False):
        """Attention of the newest tokens over the cache (append them first).

        Args:
            q:          [n_seqs, T, q_heads, head_dim] float16 or [n_seqs, q_heads,
                        head_dim]; q_heads a multiple of n_kv_heads.  The T query
                        tokens are the last T of the sequence, each seeing the
                        slots up to its own.
            scale:      of the scores (default 1 / sqrt(head_dim)).
            counts:     int32 [n_seqs], query tokens of each sequence (default: T);
                        the rows of the others are zero, their lse -inf.
            accumulate: add each slot's attention weight, summed over query tokens
                        and the KV head's query heads, to `mass` (with scores of
                        the whole pool, up to 1 GiB, in a temporary buffer).
            out:        tensor to write into, of q's shape, not among q's memory.
            return_lse: also return log(sum(exp(scores))), float32, without head_dim.

        Returns:
            out, or (out, lse).  Rows without any key are zero with lse -inf.
        """
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim)
        return self._h.attend(q, scale, counts, accumulate, out, return_lse)

    def evict(self, keep: int, recent: int = 0, sink: int = 0) -> None:
        """Cut every sequence of more than `keep` slots to `keep`, head by head:
        the last `recent` and the first `sink` positions stay, and of the other
        slots those with the largest `mass` (equal ones: lowest slot first).
        Kept slots beyond `keep` move into the freed ones below.  One kernel, two
        when min(keep, capacity - keep) is above 256, with lists that grow with
        it; the capacity is max_pages * page_size, so a max_pages close to what a
        sequence needs keeps a step at the cache's bound in one kernel.  A
        sequence with a page missing is left as it is (see check)."""
        self._h.evict(keep, recent, sink)

    def check(self) -> None:
        """Raise RuntimeError if a call on this device has reported an error since the last check: slots in a page
        outside the pool (not written, not read), a length, count or `at` outside a sequence's pages (tokens that do
        not fit are dropped), a wait that gave up.  The calls themselves only launch kernels and never raise for
        these.  Synchronises; clears the device error word, which all kernels of the library share."""
        with torch.cuda.device(self.units.device):
            torch.cuda.synchronize()
            word = dyn_quant._C.read_device_error(True)
        if word:
            what = [f"{call}: {text}" for shift, call in ((16, "append or evict"), (20, "attend"))
                    for bit, text in enumerate(_ERRORS) if word >> (shift + bit) & 1]
            raise RuntimeError(f"device error word {word:#x} ({'; '.join(what) or 'not of a KV cache call'})")

    def read(self, seq: int):
        """(k, v) of one sequence as the cache holds them, float16 [length,
        n_kv_heads, head_dim] each, in slot order (for inspection; synchronises)."""
        n, d, size = int(self.lengths[seq]), self.head_dim, self.page_size
        if not 0 <= n <= self.max_pages * size:
            raise RuntimeError(f"sequence {seq} has a length of {n}, outside its pages")
        pages = self.page_table[seq, :-(-n // size)].long()
        if bool(((pages < 0) | (pages >= self.n_pages)).any()):
            raise RuntimeError(f"sequence {seq} has slots in a page outside the pool")
        u = self.units[pages].transpose(0, 1).reshape(self.n_kv_heads, -1, unit_bytes(d))
        par = u[..., 16 * d:].contiguous().view(torch.float16).view(self.n_kv_heads, -1, 4).float()
        rows = (u[..., :8 * d].reshape(self.n_kv_heads, -1, d // 2),
                u[..., 8 * d:16 * d].reshape(self.n_kv_heads, -1, 8, d // 4, 2, 2).transpose(3, 4)
                .reshape(self.n_kv_heads, -1, d // 2))
        got = []
        for i, r in enumerate(rows):
            codes = torch.stack([r & 15, r >> 4], dim=-1).flatten(-2).float()
            val = (par[..., 2 * i:2 * i + 1] * (codes - par[..., 2 * i + 1:2 * i + 2])).half()
            got.append(val[:, :n].transpose(0, 1).contiguous())
        return got[0], got[1]
