"""Paged 8-bit key/value cache of a serving loop: sequences that come, branch and go.

The packed state (``tq_adaptive_backend.py``) compresses one growing sequence per batch row to a mix of widths; the
reference has nothing else (kvquant/tq_adaptive_backend.py:245-541).  This cache stands beside it for what a server
does around that: it keeps every token at 8 bits, admits and ends sequences in the middle of a batch, and lets the
beams of a search share their past.  ``include/odmkv_b200.h`` describes the layout; the kernels are behind the
``block8_*``, ``pages_*`` and ``beam_select`` functions of ``ops.py``.

One step::

    cache.begin(1)                                  # or a [N] int32 tensor: tokens per sequence in this step
    for layer in range(L):
        cache.append(layer, k, v)                   # [N, H, T, 128]
        out = cache.attention(layer, q)             # [N, Hq, T, 128]
    scores, parents, tokens = ops.beam_select(logits, scores)
    cache.fork(parents)                             # a beam search's reordering

Nothing in a step reads the device from the host, so a step can be captured into a CUDA graph; ``check()`` reads the
status word and raises if a step was refused.  Calls on one cache belong on one stream (or are ordered by events).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import ops
from ._lib import (APPEND_SHORT, ATTN_EXPIRED, BLOCK_MAX_SEQS, CODE_E4M3, CODE_INT8, HEAD_DIM, PAGES_BAD_PARENT, PAGES_EXHAUSTED, PAGES_POOL_SMALL,
                   PAGES_TABLE_FULL, BlockCache, OdmkvError, dtype_code, require_cuda)

__all__ = ["BlockKVCache"]

CODE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_FORMATS = {torch.float8_e4m3fn: CODE_E4M3, torch.int8: CODE_INT8}
_REFUSALS = ((PAGES_EXHAUSTED, "no free page was left for a sequence"),
             (PAGES_TABLE_FULL, "a sequence outgrew its table row"),
             (PAGES_BAD_PARENT, "a fork named a parent outside its search"),
             (PAGES_POOL_SMALL, "the new pool holds fewer pages than are in use"),
             (APPEND_SHORT, "a layer's keys and values held fewer tokens than a sequence's step"),
             (ATTN_EXPIRED, "a bounded wait of an attention kernel expired; its results are invalid"))


class BlockKVCache:
    """The tensors of one cache (all on one CUDA device, contiguous, 16-byte aligned):

    ``k_codes``, ``v_codes`` [L, pages, H, page, 128] float8_e4m3fn or int8; ``k_scale``, ``v_scale`` [L, pages, H] fp32 powers
    of two;
    ``k_tail``, ``v_tail`` [L, N, H, page, 128] fp16 or bf16; ``table`` [N, width], ``lens`` [N], ``new_lens`` [N] and
    ``refs`` [pages] int32; ``status`` [1] int32 (made here when absent).  ``allocate`` makes an empty cache."""

    def __init__(self, k_codes, v_codes, k_scale, v_scale, k_tail, v_tail, table, lens, new_lens, refs, status=None):
        if k_codes.dim() != 5 or k_codes.shape[-1] != HEAD_DIM:
            raise ValueError(f"expected codes [L, pages, H, page, {HEAD_DIM}], got {tuple(k_codes.shape)}")
        L, pages, H, page, _ = k_codes.shape
        if page not in (16, 32, 64, 128):
            raise ValueError(f"page must be 16, 32, 64 or 128 tokens, got {page}")
        if table.dim() != 2:
            raise ValueError(f"expected table [N, width], got {tuple(table.shape)}")
        N, width = table.shape
        if k_codes.dtype not in _FORMATS:
            raise ValueError(f"codes must be float8_e4m3fn or int8, got {k_codes.dtype}")
        if k_tail.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"tails must be fp16 or bf16, got {k_tail.dtype}")
        if min(L, pages, H, N, width) < 1 or N > BLOCK_MAX_SEQS:
            raise ValueError(f"a cache needs at least one layer, page, head and sequence, and at most {BLOCK_MAX_SEQS} sequences")
        if max((width + 1) * page, N * width) > 0x7fffffff:
            raise ValueError(f"positions and table entries are counted in 32 bits, got a table {(N, width)} of pages of {page} tokens")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=k_codes.device)
        i32 = torch.int32
        want = dict(k_codes=(k_codes, (L, pages, H, page, HEAD_DIM), k_codes.dtype), v_codes=(v_codes, (L, pages, H, page, HEAD_DIM), k_codes.dtype),
                    k_scale=(k_scale, (L, pages, H), torch.float32), v_scale=(v_scale, (L, pages, H), torch.float32),
                    k_tail=(k_tail, (L, N, H, page, HEAD_DIM), k_tail.dtype), v_tail=(v_tail, (L, N, H, page, HEAD_DIM), k_tail.dtype),
                    table=(table, (N, width), i32), lens=(lens, (N,), i32), new_lens=(new_lens, (N,), i32), refs=(refs, (pages,), i32),
                    status=(status, (1,), i32))
        struct = BlockCache()
        for name, (t, shape, dtype) in want.items():
            require_cuda(t, name)
            if tuple(t.shape) != shape or t.dtype != dtype:
                raise ValueError(f"expected {name} {shape} {dtype}, got {tuple(t.shape)} {t.dtype}")
            if t.device != k_codes.device:
                raise ValueError(f"{name} is on {t.device}, the codes are on {k_codes.device}")
            if not t.is_contiguous() or (t.dim() == 5 and t.data_ptr() % 16):
                raise ValueError(f"{name} must be contiguous and 16-byte aligned")
            setattr(self, name, t)
            setattr(struct, name, t.data_ptr())
        self.num_layers, self.num_pages, self.num_heads, self.page = L, pages, H, page
        self.num_seqs, self.width = N, width
        self.dtype, self.device = k_tail.dtype, k_codes.device
        struct.L, struct.N, struct.H, struct.page, struct.pages, struct.width = L, N, H, page, pages, width
        struct.code_format, struct.tail_dtype = _FORMATS[k_codes.dtype], dtype_code(k_tail.dtype)
        self._struct = struct
        self._ref = ctypes.byref(struct)

    def __deepcopy__(self, memo):
        import copy
        names = [f[0] for f in BlockCache._fields_[:11]]
        new = type(self)(**{x: copy.deepcopy(getattr(self, x), memo) for x in names})
        memo[id(self)] = new
        return new

    @classmethod
    def allocate(cls, num_layers: int, num_seqs: int, num_heads: int, num_pages: int, max_tokens: int, page: int = 64,
                 dtype: torch.dtype = torch.bfloat16, fmt: str = "e4m3", device="cuda") -> "BlockKVCache":
        """An empty cache for ``num_seqs`` sequences of up to ``max_tokens`` tokens that share ``num_pages`` pages."""
        if fmt not in CODE_DTYPES:
            raise ValueError(f"fmt must be one of {sorted(CODE_DTYPES)}, got {fmt!r}")
        if page not in (16, 32, 64, 128):
            raise ValueError(f"page must be 16, 32, 64 or 128 tokens, got {page}")
        width = max(1, -(-int(max_tokens) // page))
        codes = (num_layers, num_pages, num_heads, page, HEAD_DIM)
        tails = (num_layers, num_seqs, num_heads, page, HEAD_DIM)

        def zeros(shape, dt):
            if dt == torch.float8_e4m3fn:
                return torch.zeros(shape, dtype=torch.uint8, device=device).view(dt)
            return torch.zeros(shape, dtype=dt, device=device)

        i32 = torch.int32
        return cls(zeros(codes, CODE_DTYPES[fmt]), zeros(codes, CODE_DTYPES[fmt]), torch.ones(codes[:3], device=device),
                   torch.ones(codes[:3], device=device), zeros(tails, dtype), zeros(tails, dtype),
                   torch.full((num_seqs, width), -1, dtype=i32, device=device), zeros((num_seqs,), i32), zeros((num_seqs,), i32),
                   zeros((num_pages,), i32))

    # ------------------------------------------------------------------ a step
    def begin(self, new_lens: Union[int, torch.Tensor]) -> None:
        """Finish the running step and take the pages of the next: ``new_lens`` tokens per sequence (an int for all, or
        int32 [N]).  A sequence whose pages cannot be had gets 0 tokens and sets the status."""
        ops.pages_begin(self, new_lens)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Store the running tokens of a layer, once a step: [N, H, T, 128], T no less than any ``new_lens[n]``, the number of
        tokens that sequence n takes."""
        ops.block8_append(self, layer, k, v)

    def attention(self, layer: int, q: torch.Tensor, scale: Optional[float] = None, softcap: float = 0.0,
                  slopes: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Causal attention of the running tokens [N, Hq, T, 128] over everything stored, themselves included."""
        return ops.block8_attn(self, layer, q, scale=scale, softcap=softcap, slopes=slopes, return_lse=return_lse)

    # ------------------------------------------------------------------ sequences and pages
    def fork(self, parents: torch.Tensor) -> None:
        """Reorder the beams of searches: parents [N / W, W] int64, indices inside a search of W neighbouring sequences.  Not
        between ``begin`` and the last layer's ``append``."""
        ops.pages_fork(self, parents)

    def free(self, leave: torch.Tensor) -> None:
        """End the sequences where ``leave`` [N] bool is set."""
        ops.pages_free(self, leave)

    def compact_into(self, other: "BlockKVCache") -> None:
        """Move everything into another pool, pages side by side (see ``ops.pages_compact``)."""
        ops.pages_compact(self, other)

    def compact(self, num_pages: Optional[int] = None) -> "BlockKVCache":
        """A new cache over a pool of ``num_pages`` pages (by default as many as are in use), holding the same sequences;
        tails and status are shared with this one, which should not be used any more.  Reads the host."""
        live = int((self.refs > 0).sum())
        num_pages = max(1, live) if num_pages is None else int(num_pages)
        if num_pages < live:
            raise ValueError(f"{live} pages are in use, the new pool would hold {num_pages}")
        codes = (self.num_layers, num_pages, self.num_heads, self.page, HEAD_DIM)
        new = [torch.zeros(codes, dtype=torch.uint8, device=self.device).view(self.k_codes.dtype) for _ in range(2)]
        scales = [torch.ones(codes[:3], device=self.device) for _ in range(2)]
        out = BlockKVCache(*new, *scales, self.k_tail, self.v_tail, torch.empty_like(self.table), torch.empty_like(self.lens),
                           torch.empty_like(self.new_lens), torch.empty(num_pages, dtype=torch.int32, device=self.device), self.status)
        ops.pages_compact(self, out)
        return out

    # ------------------------------------------------------------------ reads
    def check(self) -> None:
        """Raise if any call since the cache was made refused its work (synchronises)."""
        bits = int(self.status.item())
        if bits:
            raise OdmkvError("; ".join(text for bit, text in _REFUSALS if bits & bit))

    def free_pages(self) -> int:
        """Pages that nobody holds (synchronises)."""
        return int((self.refs == 0).sum())

    def materialize(self, layer: int, seq: int):
        """What the cache stands for: keys and values [H, tokens, 128] fp32 of one sequence (synchronises)."""
        total = int(self.lens[seq]) + int(self.new_lens[seq])
        full, rest = divmod(total, self.page)
        at = self.table[seq, :full].long()
        out = []
        for codes, scale, tail in ((self.k_codes, self.k_scale, self.k_tail), (self.v_codes, self.v_scale, self.v_tail)):
            pages = codes[layer].view(torch.uint8)[at].view(codes.dtype).float() * scale[layer][at][..., None, None]
            out.append(torch.cat([pages.transpose(0, 1).reshape(self.num_heads, full * self.page, HEAD_DIM),
                                  tail[layer, seq, :, :rest].float()], dim=1))
        return out[0], out[1]
