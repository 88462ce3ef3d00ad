"""Keys and values held in 4 or 8 bits.

``PackedKV`` is one layer's packed pages (csrc/packed_kv.cuh has the format) and what is done with them: tokens are rotated
and quantised as they are written, read back as plain keys and values, and attended to where they lie.  Pages, slots and
block tables are the cache manager's, as of an unpacked layer.  The reference engine has no counterpart.
"""
from __future__ import annotations

import os
from typing import Optional, Sequence

import torch

from ..csrc import ops

# as in parts/attention.py, which says what they do and what was measured
ATTN_POLICY = os.environ.get("GOLLMGO_B200_ATTN", "auto")
SHORT_PROMPT_KEYS = int(os.environ.get("GOLLMGO_B200_ATTN_SHORT_KEYS", "256"))
SCRATCH_TOKENS = 65536         # tokens that prefill() reads back at a time (one sequence may be longer)
MOST_SEQUENCES = 1024          # ... of so many sequences


def long_tiles(options: bool, tiles128: int, num_heads: int, window: int, longest: int, num_sms: int) -> bool:
    """Whether the prompt kernels on tcgen05 take portions that make ``tiles128`` tiles of 128 rows, the longest with ``longest`` keys: the line
    of the attention layer, for plain scores (Attention._few_short_tiles) and for ones with ``options`` (Attention.long_tiles)."""
    reach = (window or 1 << 30) if options else 1 << 30
    if options and (reach < 128 or longest <= 144):
        return False
    return tiles128 * ((num_heads + 1) // 2) * 2 > num_sms or min(longest, reach) > SHORT_PROMPT_KEYS


class PackedKV:
    """``pages``: uint8 [pages, kv heads, bytes of a page and head] (``PackedKV.empty`` makes them).

    All calls run on the current stream of the device that holds the pages, which must be the current one.  Activations are
    bfloat16 or float32; with float32 ones the whole path computes in 32 bits or more."""

    def __init__(self, pages: torch.Tensor, head_dim: int, page_size: int, bits: int):
        need = ops.packed_page_bytes(bits, head_dim, page_size)
        if pages.dtype != torch.uint8 or pages.dim() != 3 or pages.shape[2] != need or not pages.is_contiguous() or not pages.is_cuda:
            raise ops.KernelError(f"packed pages are contiguous uint8 [pages, kv heads, {need}] on a CUDA device, "
                                  f"got {pages.dtype} {tuple(pages.shape)} on {pages.device}")
        self.pages, self.head_dim, self.page_size, self.bits = pages, head_dim, page_size, bits
        self.kv_heads = pages.shape[1]
        self._sms = 148

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int, bits: int, device="cuda") -> "PackedKV":
        size = ops.packed_page_bytes(bits, head_dim, page_size)
        return cls(torch.zeros(num_pages, kv_heads, size, dtype=torch.uint8, device=device), head_dim, page_size, bits)

    # ------------------------------------------------------------------ store and read back
    def write(self, qkv: torch.Tensor, positions: Optional[torch.Tensor], slots: Optional[torch.Tensor], num_heads: int,
              inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False, magnitude: float = 1.0,
              q_out: Optional[torch.Tensor] = None, early: bool = False) -> torch.Tensor:
        """Rows of qkv [T, (num_heads + 2 kv heads) * head size]: q and k are rotated by ``positions`` (``inv_freq`` float64
        [width / 2]; None: they are not), k and v quantised into their pages at ``slots`` (page * page_size + place; below
        0: not stored; none twice; None: nothing is stored).  Returns the rotated q [T, num_heads, head size], in ``q_out``
        where given (which may be the q columns of qkv).  ``early``: no kernel that may still run on the stream writes positions, slots or inv_freq
        (they came by a copy, or before an event that the stream has waited for), and they may be read while kernels ahead run."""
        if q_out is None:
            q_out = qkv.new_empty((qkv.shape[0], num_heads, self.head_dim))
        ops.packed_write(qkv, positions, slots, inv_freq, magnitude, self.pages, q_out, num_heads, self.kv_heads, self.head_dim,
                         self.page_size, self.bits, interleaved, early)
        return q_out

    def read(self, tables: torch.Tensor, lens: torch.Tensor, first_page: torch.Tensor, num_pages: int, dtype=torch.bfloat16,
             out=None):
        """Plain keys and values of whole sequences: page j of sequence b (``tables`` [B, width]) becomes page
        first_page[b] + j of the two results [num_pages, kv heads, page_size, head size], for the pages of its first
        lens[b] tokens; what lies behind the last token is zero.  Other pages of the results are not written."""
        if out is None:
            out = self.pages.new_empty((2, num_pages, self.kv_heads, self.page_size, self.head_dim), dtype=dtype).unbind(0)
        ops.packed_read(self.pages, tables, lens, first_page, out[0], out[1], tables.shape[1], self.kv_heads, self.head_dim,
                        self.page_size, self.bits)
        return out

    # ------------------------------------------------------------------ attention
    def _out(self, what: str, q: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
        shape = q.shape
        if len(shape) != 3 or shape[2] != self.head_dim or shape[1] == 0 or shape[1] % self.kv_heads:
            raise ops.KernelError(f"{what}: q is [tokens, heads in multiples of {self.kv_heads}, {self.head_dim}], got {tuple(shape)}")
        return q.new_empty(shape) if out is None else out

    def _on_tensor_cores(self, q: torch.Tensor, out: torch.Tensor) -> bool:
        return ops.packed_decode_mma_ok(q.dtype, self.head_dim, self.page_size) and q.data_ptr() % 16 == 0 \
            and q.stride(0) * q.element_size() % 16 == 0 and out.data_ptr() % 16 == 0

    def decode(self, q: torch.Tensor, tables: torch.Tensor, context_lens: torch.Tensor, max_context: int, scale: float, *,
               window: int = 0, softcap: float = 0.0, sink=None, slopes=None, temperature=None, cu_q_lens=None, seqs=None,
               out: Optional[torch.Tensor] = None, early: bool = False) -> torch.Tensor:
        """Attention of single tokens, each the last of its sequence's context_lens[b] stored ones: q [n, heads, head size]
        (row i of sequence i; with ``seqs`` token i belongs to sequence seqs[i], none of the tables': padding, and with ``cu_q_lens``
        its row is cu_q_lens[sequence]).  ``max_context``: no context is expected to be longer (the work is spread by it).
        The options are those of the attention layer; a token with no key in sight gives zeros.  ``early``: no kernel that may still run on
        the stream writes block tables or index lists (they came by a copy, or before an event that the stream has waited for), and they may be
        read while kernels ahead run."""
        out = self._out("decode", q, out)
        nh, d = q.shape[1], self.head_dim
        n = seqs.numel() if seqs is not None else q.shape[0]
        more = (window, scale, softcap, sink, slopes, temperature)
        if self._on_tensor_cores(q, out):
            shape = (nh, self.kv_heads, d, self.page_size, self.bits)
            most = ops.packed_decode_tokens(nh, tables.shape[-1], self.page_size)
            size = ops.packed_launches_scratch(q.dtype, n, most, nh, self.kv_heads, d, self.bits, max_context, window)
            scratch = q.new_empty((size,), dtype=torch.float32)
            if n <= most:
                ops.packed_decode_mma(q, self.pages, tables, cu_q_lens, context_lens, seqs, n, max_context, scratch, out, *shape, *more, early)
                return out
            if seqs is None and cu_q_lens is None:      # more tokens than a launch takes: rows of q go with their sequences
                for lo in range(0, n, most):
                    hi = min(n, lo + most)
                    ops.packed_decode_mma(q[lo:hi], self.pages, tables[lo:hi], None, context_lens[lo:hi], None, hi - lo, max_context, scratch,
                                          out[lo:hi], *shape, *more, early)
                return out
            if seqs is None:
                seqs, early = torch.arange(n, dtype=torch.int32, device=q.device), False       # (a list that the kernel ahead writes)
            for lo in range(0, n, most):
                part = seqs[lo:lo + most]
                ops.packed_decode_mma(q, self.pages, tables, cu_q_lens, context_lens, part, part.numel(), max_context, scratch, out, *shape, *more, early)
            return out
        splits = self._splits(n, self.kv_heads, max_context, window)
        rows = n * nh * splits
        part = torch.empty(rows * (d + 2), dtype=torch.float32, device=q.device)
        ops.packed_decode(q, self.pages, tables, cu_q_lens, context_lens, seqs, n, splits, part[:rows * d], part[rows * d:], out, nh,
                          self.kv_heads, d, self.page_size, self.bits, *more)
        return out

    @staticmethod
    def _splits(n: int, kv_heads: int, max_context: int, window: int) -> int:
        """The general kernel: slices of the context until every multiprocessor has four blocks."""
        reach = min(max_context, window) if window else max_context
        return max(1, min(64, -(-reach // 64), 592 // max(1, n * kv_heads)))

    @staticmethod
    def decode_spread(dtype: torch.dtype, n: int, num_heads: int, kv_heads: int, head_dim: int, page_size: int, bits: int, max_context: int,
                      window: int = 0) -> tuple:
        """How decode() spreads n tokens: two values of ``max_context`` for which this is the same launch the same (a call captured with one
        of them serves contexts up to the other as well)."""
        if not ops.packed_decode_mma_ok(dtype, head_dim, page_size):
            return (PackedKV._splits(n, kv_heads, max_context, window),)
        most = ops.PACKED_DECODE_TOKENS
        sizes = sorted({min(n, most), n % most or min(n, most)})
        return tuple(ops.packed_decode_shape(dtype, m, num_heads, kv_heads, head_dim, bits, max_context, window) for m in sizes if m)

    def prefill(self, q: torch.Tensor, tables: torch.Tensor, cu_q_lens: torch.Tensor, context_lens: torch.Tensor,
                q_lens: Sequence[int], contexts: Sequence[int], scale: float, *, window: int = 0, softcap: float = 0.0, sink=None,
                slopes=None, temperature=None, least: int = 1, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of prompt portions: sequence b brings rows cu_q_lens[b] .. cu_q_lens[b + 1] of q [T, heads, head
        size], the last q_lens[b] of its context_lens[b] stored tokens.  ``q_lens`` and ``contexts`` say on the host what
        the two device lists hold.  Sequences of fewer than ``least`` rows are left out (their rows of ``out`` stay as they are).

        bfloat16 rows, heads of 64 or 128: the pages of the portions are read back once, in half precision, and the prompt kernels run on them
        (0.17 % off 64 bits, as single tokens are); steps of many long portions go in runs of sequences, so that what is read back at a time
        stays within ``SCRATCH_TOKENS`` (or the longest sequence).  float32 rows that the tensor cores take attend to the codes where they lie, as
        single tokens do; other rows too, on the general kernel."""
        out = self._out("prefill", q, out)
        B, P = len(q_lens), self.page_size
        if len(contexts) != B or tables.shape[0] < B:
            raise ops.KernelError(f"prefill: {B} portions, {len(contexts)} contexts and block tables of {tables.shape[0]} sequences")
        if sum(a for a in q_lens if a > 0) > q.shape[0]:
            raise ops.KernelError(f"prefill: portions of {sum(a for a in q_lens if a > 0)} rows in q of {q.shape[0]}")
        lo = hi = pages = most = longest = items = 0           # (a run of sequences: from its first portion to behind its last)
        exact = q.dtype == torch.float32 and self._on_tensor_cores(q, out)
        fold = ops.packed_prompt_fold(q.shape[1], self.kv_heads) if exact else 1
        counts = [0, 0, 0]

        def run():
            self._portions(q, out, tables, cu_q_lens, context_lens, lo, hi, pages, most, counts, longest, scale, window, softcap, sink, slopes,
                           temperature, least)
        for b in range(B):
            a, c = q_lens[b], contexts[b]
            if a < least or a <= 0:
                continue
            if a > c or c > tables.shape[1] * P:
                raise ops.KernelError(f"prefill: sequence {b} brings {a} of {c} tokens, its block table holds {tables.shape[1] * P}")
            if exact:
                items += -(-a // fold)
                longest = max(longest, c)
                continue
            n = -(-c // P)
            seen = n - (max(0, c - a - window + 1) // P if window else 0)
            if pages and ((pages + seen) * P > SCRATCH_TOKENS or b - lo >= MOST_SEQUENCES):
                run()
                pages, most, longest, counts = 0, 0, 0, [0, 0, 0]
            if not pages:
                lo = b
            hi = b + 1
            pages += seen
            most = max(most, n)
            longest = max(longest, c)
            for i, h in enumerate((16, 64, 128)):
                counts[i] += -(-a // h)
        if items:
            if tables.shape[0] != B:
                tables, context_lens, cu_q_lens = tables[:B], context_lens[:B], cu_q_lens[:B + 1]
            size = ops.packed_launches_scratch(q.dtype, items, ops.packed_decode_tokens(q.shape[1], tables.shape[1], P), q.shape[1], self.kv_heads,
                                               self.head_dim, self.bits, longest, window)
            ops.packed_prompt_f32(q, self.pages, tables, cu_q_lens, context_lens, least, items, q.new_empty((2 * items,), dtype=torch.int32),
                                  longest, q.new_empty((size,)), out, q.shape[1], self.kv_heads, self.head_dim, self.page_size, self.bits,
                                  window, scale, softcap, sink, slopes, temperature)
        if pages:
            run()
        return out

    def _portions(self, q, out, tables, cu_q_lens, context_lens, lo, hi, pages, most, counts, longest, scale, window, softcap, sink, slopes,
                  temperature, least):
        """prefill() of sequences lo .. hi, whose portions see ``pages`` pages and make counts[i] tiles of 16, 64 and 128 rows."""
        nh, d, P = q.shape[1], self.head_dim, self.page_size
        ops.packed_prefill_rows(q, out, self.pages, nh, d, sink, slopes)
        if hi - lo != tables.shape[0]:
            tables, context_lens, cu_q_lens = tables[lo:hi], context_lens[lo:hi], cu_q_lens[lo:hi + 1]
        # (the plain tcgen05 kernel takes the largest product for the largest score)
        options = softcap > 0 or sink is not None or slopes is not None or temperature is not None or not scale > 0
        fast = q.dtype == torch.bfloat16 and d in (64, 128) and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 0 \
            and ATTN_POLICY != "general" and self.kv_heads <= 1024
        if not fast:                               # on the codes where they lie, in float32 arithmetic
            n = counts[0]
            ints = torch.empty(2 * n, dtype=torch.int32, device=q.device)
            ops.packed_unfold(self.pages, tables, cu_q_lens, context_lens, None, None, 0, None, [(16, n, ints[:n], ints[n:])], self.kv_heads, d, P,
                              self.bits, window, least)
            ops.packed_prefill(q, self.pages, tables, cu_q_lens, context_lens, ints[:n], ints[n:], n, out, nh, self.kv_heads, d, P, self.bits,
                               window, scale, softcap, sink, slopes, temperature)
            return
        lists = [(64, counts[1])]
        if ATTN_POLICY == "auto" and long_tiles(options, counts[2], nh, window, longest, self._sms):
            lists.append((128, counts[2]))
        (B, width), new = tables.shape, q.new_empty
        k, v = new((2, pages, self.kv_heads, P, d), dtype=torch.float16).unbind(0)
        floats = new((ops.packed_unfold_floats(self.kv_heads),), dtype=torch.float32)
        ints = new((B * width + 2 * sum(n for _, n in lists),), dtype=torch.int32)
        at, tiles = B * width, []
        for _, n in lists:
            tiles.append((ints[at:at + n], ints[at + n:at + 2 * n], n))
            at += 2 * n
        plain = ints[:B * width]
        ops.packed_unfold(self.pages, tables, cu_q_lens, context_lens, k, v, most, plain, [(h, n, *t[:2]) for (h, n), t in zip(lists, tiles)],
                          self.kv_heads, d, P, self.bits, window, least, floats)
        ops.attn_prefill_half(q, k, v, floats, plain, width, cu_q_lens, context_lens, tiles[0], tiles[1] if len(tiles) > 1 else None, out, nh,
                              self.kv_heads, d, P, window, scale, options, softcap, sink, slopes, temperature)

    @staticmethod
    def scratch_bytes(needs, max_context: int, dtype) -> int:
        """Most bytes that prefill() reads back at a time for any packed need among ``needs``."""
        def flat(need):
            return [n for sub in need for n in flat(sub)] if isinstance(need, (tuple, list)) else [need]
        width = max((n.n_kv_heads * n.head_dim for n in flat(list(needs)) if getattr(n, "bits", None)), default=0)
        return max(max_context, SCRATCH_TOKENS) * width * 2 * torch.empty((), dtype=dtype).element_size()
