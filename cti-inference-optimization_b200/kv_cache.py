"""The 4-bit key/value cache: its storage, and the host-side book-keeping of
which sequence holds which pages.

The reference keeps no cache: it runs every token of every user's sequence
again in each forward (``baseline/infer.py:388-409``).  The operators are
``ops.kv4_append``, ``ops.kv4_read`` and ``ops.kv4_attention``; the format is
described in ``include/cti_b200.h``.
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import _lib
from ._lib import lib

PAGE_TOKENS = _lib.KV4_PAGE_TOKENS


class KV4Cache:
    """The pages of one layer: ``pages`` uint8 [num_pages, kv_heads, bytes] on
    ``device``, 64 tokens of every KV head per page, for keys and values of
    ``dtype`` (bfloat16 or float16) with ``head_dim`` 32, 64 or 128.  A token
    takes 1.25 * head_dim bytes per KV head, against 4 * head_dim in 16 bits.
    Each 32 head dims of a token share a scale and a base of ``dtype``; such a
    group is NaN as a whole where one value is not finite, or where the base does
    not fit: from magnitudes of 20,900 in float16 and 1e38 in bfloat16 on."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
        if num_pages <= 0:
            raise ValueError("num_pages must be positive")
        page_bytes = lib.cti_kv4_page_bytes(int(kv_heads), int(head_dim))
        if page_bytes == 0:
            raise RuntimeError(
                f"KV4Cache: unsupported shape (kv_heads {kv_heads}, head_dim {head_dim})")
        self.kv_heads = int(kv_heads)
        self.head_dim = int(head_dim)
        self.dtype = dtype
        self.dtype_code = _lib.DTYPE_CODES[dtype]
        self.pages = torch.zeros((int(num_pages), self.kv_heads, page_bytes // self.kv_heads),
                                 dtype=torch.uint8, device=device)
        self.device = self.pages.device
        self.index = self.pages.get_device()  # -1 on the CPU

    @property
    def num_pages(self) -> int:
        return self.pages.shape[0]


class SequenceCache:
    """Keys and values of up to ``max_seqs`` sequences in every layer of a
    model, in 4 bits: one ``KV4Cache`` per layer over common page numbers, a
    page table, and the pages that are free.

    ``extend`` makes room for new tokens of some sequences and returns what
    ``TransformerEncoder.forward`` takes as its ``extension``: the forward of
    those tokens appends their keys and values and attends to the sequences'
    histories.  ``undo`` takes an extension back whose forward did not run.
    ``release`` gives a sequence's pages back.  The book-keeping is on the host;
    ``extend`` copies three small tensors to the device and does not wait for it.
    Use one stream for the forwards of one cache, or order them: a page that was
    given back may go to the next sequence at once."""

    def __init__(self, num_layers: int, max_seqs: int, num_pages: int, kv_heads: int,
                 head_dim: int, max_tokens: int, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda"):
        if num_layers <= 0 or max_seqs <= 0 or max_tokens <= 0:
            raise ValueError("num_layers, max_seqs and max_tokens must be positive")
        self.layers = [KV4Cache(num_pages, kv_heads, head_dim, dtype, device)
                       for _ in range(num_layers)]
        self.max_seqs = int(max_seqs)
        self.max_tokens = int(max_tokens)
        self._pages: list[list[int]] = [[] for _ in range(self.max_seqs)]
        self._lens = [0] * self.max_seqs
        self._last = [0] * self.max_seqs  # the last change of each sequence
        self._changes = 0
        self._free = list(range(int(num_pages) - 1, -1, -1))

    @property
    def device(self) -> torch.device:
        return self.layers[0].device

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        """Tokens of sequence ``seq`` so far."""
        return self._lens[seq]

    def _check(self, seqs: Sequence[int]) -> list[int]:
        seqs = [int(s) for s in seqs]
        if any(s < 0 or s >= self.max_seqs for s in seqs):
            raise IndexError(f"sequences must be in [0, {self.max_seqs})")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may be named once")
        return seqs

    def extend(self, seqs: Sequence[int], new: Sequence[int]) -> dict:
        """Makes room for ``new[i]`` tokens at the end of sequence ``seqs[i]``.
        Raises, and changes nothing, where the pages do not suffice or a
        sequence would pass ``max_tokens``."""
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("extend cannot be captured into a graph: extend first, then capture "
                               "the forward of what it returned")
        seqs, new = self._check(seqs), [int(n) for n in new]
        if len(new) != len(seqs) or any(n < 0 for n in new):
            raise ValueError("new must hold a count for each sequence")
        totals = [self._lens[s] + n for s, n in zip(seqs, new)]
        if any(t > self.max_tokens for t in totals):
            raise ValueError(f"a sequence would pass max_tokens = {self.max_tokens}")
        need = [-(-t // PAGE_TOKENS) - len(self._pages[s]) for s, t in zip(seqs, totals)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages are needed, {len(self._free)} are free")
        before = [(s, self._lens[s], len(self._pages[s]), self._last[s]) for s in seqs]
        self._changes += 1
        for s, t, n in zip(seqs, totals, need):
            self._pages[s] += [self._free.pop() for _ in range(n)]
            self._lens[s] = t
            self._last[s] = self._changes
        cols = max([len(self._pages[s]) for s in seqs], default=0)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        # One copy: offsets, lengths, and the table's rows.
        rows = [self._pages[s] + [-1] * (cols - len(self._pages[s])) for s in seqs]
        flat = torch.tensor(cu + totals + [p for r in rows for p in r], dtype=torch.int32)
        if self.device.type == "cuda":
            flat = flat.pin_memory().to(self.device, non_blocking=True)
        n = len(seqs)
        return {"cache": self, "cu_seqlens": flat[:n + 1], "kv_lens": flat[n + 1:2 * n + 1],
                "page_table": flat[2 * n + 1:].view(n, cols), "max_seqlen": max(new, default=0),
                "max_kv_len": max(totals, default=0), "tokens": cu[-1],
                "undo": (self._changes, before)}

    def undo(self, extension: dict) -> None:
        """Takes back what ``extend`` returned as ``extension``: its sequences have
        the lengths and pages that they had before.  For a forward that raised;
        raises ValueError, and changes nothing, where one of the sequences was
        extended or released since, or the extension taken back."""
        if extension["cache"] is not self:
            raise ValueError("the extension is of another cache")
        change, before = extension["undo"]
        if any(self._last[s] != change for s, *_ in before):
            raise ValueError("the extension is not the last change of its sequences")
        for s, length, pages, last in reversed(before):
            while len(self._pages[s]) > pages:
                self._free.append(self._pages[s].pop())
            self._lens[s], self._last[s] = length, last

    def release(self, seqs: Sequence[int]) -> None:
        """Forgets the sequences and frees their pages."""
        self._changes += 1
        for s in self._check(seqs):
            self._free += reversed(self._pages[s])
            self._pages[s] = []
            self._lens[s] = 0
            self._last[s] = self._changes
