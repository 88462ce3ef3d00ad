"""Keys and values held in 4 or 8 bits.

``PackedKV`` is one layer's packed pages (csrc/packed_kv.cuh has the format) and what is done with them: tokens are rotated
and quantised as they are written, read back as plain keys and values, and attended to where they lie.  Pages, slots and
block tables are the cache manager's, as of an unpacked layer.  The reference engine has no counterpart.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from ..csrc import ops

SHORT_PROMPT_KEYS = 256


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
        where given (which may be the q columns of qkv).  ``early``: positions, slots and inv_freq are not the output of the kernel
        ahead on the stream, and may be read while it runs."""
        if q_out is None:
            q_out = torch.empty(qkv.shape[0], num_heads, self.head_dim, dtype=qkv.dtype, device=qkv.device)
        ops.packed_write(qkv, positions, slots, inv_freq, magnitude, self.pages, q_out, num_heads, self.kv_heads, self.head_dim,
                         self.page_size, self.bits, interleaved, early)
        return q_out

    def read(self, tables: torch.Tensor, lens: torch.Tensor, first_page: torch.Tensor, num_pages: int, dtype=torch.bfloat16,
             out=None):
        """Plain keys and values of whole sequences: page j of sequence b (``tables`` [B, width]) becomes page
        first_page[b] + j of the two results [num_pages, kv heads, page_size, head size], for the pages of its first
        lens[b] tokens; what lies behind the last token is zero.  Other pages of the results are not written."""
        if out is None:
            shape = (num_pages, self.kv_heads, self.page_size, self.head_dim)
            out = (torch.empty(shape, dtype=dtype, device=self.pages.device), torch.empty(shape, dtype=dtype, device=self.pages.device))
        ops.packed_read(self.pages, tables, lens, first_page, out[0], out[1], tables.shape[1], self.kv_heads, self.head_dim,
                        self.page_size, self.bits)
        return out

    # ------------------------------------------------------------------ attention
    def decode(self, q: torch.Tensor, tables: torch.Tensor, context_lens: torch.Tensor, max_context: int, scale: float, *,
               window: int = 0, softcap: float = 0.0, sink=None, slopes=None, temperature=None, cu_q_lens=None, seqs=None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of single tokens, each the last of its sequence's context_lens[b] stored ones: q [n, heads, head size]
        (row i of sequence i; with ``seqs`` token i belongs to sequence seqs[i], below 0: padding, and with ``cu_q_lens``
        its row is cu_q_lens[sequence]).  ``max_context``: none of the contexts is longer (what the split of the work is
        chosen from).  The options are those of the attention layer; a token with no key in sight gives zeros."""
        nh, d = q.shape[1], self.head_dim
        if q.dim() != 3 or q.shape[2] != d or nh % self.kv_heads:
            raise ops.KernelError(f"decode: q is [tokens, heads in multiples of {self.kv_heads}, {d}], got {tuple(q.shape)}")
        n = seqs.numel() if seqs is not None else q.shape[0]
        if out is None:
            out = torch.empty(q.shape[0], nh, d, dtype=q.dtype, device=q.device)
        more = (window, scale, softcap, sink, slopes, temperature)
        if ops.packed_decode_mma_ok(q.dtype, d, self.page_size) and q.data_ptr() % 16 == 0 and q.stride(0) % 8 == 0 \
                and n <= ops.PACKED_DECODE_TOKENS:
            size = ops.packed_decode_scratch(n, nh, self.kv_heads, d, self.bits, max_context, window)
            scratch = torch.empty(size, dtype=torch.float32, device=q.device)
            ops.packed_decode_mma(q, self.pages, tables, cu_q_lens, context_lens, seqs, n, max_context, scratch, out, nh, self.kv_heads,
                                  d, self.page_size, self.bits, *more)
            return out
        reach = min(max_context, window) if window else max_context
        splits = max(1, min(64, -(-reach // 64), 592 // max(1, n * self.kv_heads)))
        part = torch.empty(n * nh * splits * (d + 2), dtype=torch.float32, device=q.device)
        ops.packed_decode(q, self.pages, tables, cu_q_lens, context_lens, seqs, n, splits, part[:n * nh * splits * d],
                          part[n * nh * splits * d:], out, nh, self.kv_heads, d, self.page_size, self.bits, *more)
        return out

    def prefill(self, q: torch.Tensor, tables: torch.Tensor, cu_q_lens: torch.Tensor, context_lens: torch.Tensor,
                q_lens: Sequence[int], contexts: Sequence[int], scale: float, *, window: int = 0, softcap: float = 0.0, sink=None,
                slopes=None, temperature=None, least: int = 1, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of prompt portions: sequence b brings rows cu_q_lens[b] .. cu_q_lens[b + 1] of q [T, heads, head
        size], the last q_lens[b] of its context_lens[b] stored tokens.  ``q_lens`` and ``contexts`` say on the host what
        the two device lists hold.  Sequences of fewer than ``least`` rows are left out (their rows of ``out`` stay as they are)."""
        nh, d = q.shape[1], self.head_dim
        if q.dim() != 3 or q.shape[2] != d or nh % self.kv_heads:
            raise ops.KernelError(f"prefill: q is [tokens, heads in multiples of {self.kv_heads}, {d}], got {tuple(q.shape)}")
        if out is None:
            out = torch.empty(q.shape[0], nh, d, dtype=q.dtype, device=q.device)
        P, dev, i32 = self.page_size, q.device, torch.int32
        pages = most = tiles16 = tiles64 = tiles128 = 0
        long = 0
        for a, c in zip(q_lens, contexts):
            if a >= least:
                n = -(-c // P)
                most = max(most, n)
                pages += n - (max(0, c - a - window + 1) // P if window else 0)
                tiles16 += -(-a // 16)
                tiles64 += -(-a // 64)
                tiles128 += -(-a // 128)
                long = max(long, c)
        if not pages:
            return out
        B, width = tables.shape
        fast = q.dtype == torch.bfloat16 and d in (64, 128) and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0
        keep = torch.empty(2, pages, self.kv_heads, P, d, dtype=q.dtype, device=dev)
        lists = [(64, tiles64)] if fast else [(16, tiles16)]
        if fast and (tiles128 * ((nh + 1) // 2) * 2 > self._sms or min(long, window or long) > SHORT_PROMPT_KEYS):
            lists.append((128, tiles128))
        ints = torch.empty(B * width + 2 * sum(n for _, n in lists), dtype=i32, device=dev)
        at, full = B * width, []
        for h, n in lists:
            full.append((h, n, ints[at:at + n], ints[at + n:at + 2 * n]))
            at += 2 * n
        plain_tables = ints[:B * width].view(B, width)
        ops.packed_unfold(self.pages, tables, cu_q_lens, context_lens, keep[0], keep[1], most, plain_tables, full, self.kv_heads, d, P,
                          self.bits, window, least)
        t = {h: dict(seq=s, q0=r, n=n) for h, n, s, r in full}
        t16, t64, t128 = (t.get(h) or dict(seq=None, q0=None, n=0) for h in (16, 64, 128))
        more = {}
        if t128["n"]:
            more = dict(tile128_seq=t128["seq"], tile128_q0=t128["q0"], num_tiles128=t128["n"])
        if softcap > 0 or sink is not None or slopes is not None or temperature is not None:
            ops.attn_prefill_x(q, q.stride(0), keep[0], keep[1], plain_tables, width, cu_q_lens, context_lens, t16["seq"], t16["q0"], t16["n"],
                               out, nh, self.kv_heads, d, d, 1, P, window, scale, softcap, t64["seq"], t64["q0"], t64["n"],
                               allow_mma=fast, sink=sink, slopes=slopes, temperature=temperature, **more)
        else:
            ops.attn_prefill(q, q.stride(0), keep[0], keep[1], plain_tables, width, cu_q_lens, context_lens, t16["seq"], t16["q0"], t16["n"],
                             out, nh, self.kv_heads, d, P, window, scale, t64["seq"], t64["q0"], t64["n"], allow_mma=fast,
                             allow_tc=bool(more), **more)
        return out
