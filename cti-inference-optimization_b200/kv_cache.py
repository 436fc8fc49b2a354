"""The 4-bit key/value cache: its storage, and the host-side book-keeping of
which sequence holds which pages.

The reference keeps no cache: it runs every token of every user's sequence
again in each forward (``baseline/infer.py:388-409``).  The operators are
``ops.kv4_append``, ``ops.kv4_read`` and ``ops.kv4_attention``; the format is
described in ``include/cti_b200.h``.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import lib

PAGE_TOKENS = _lib.KV4_PAGE_TOKENS


class KV4Cache:
    """The pages of one layer: ``pages`` uint8 [num_pages, kv_heads, bytes] on
    ``device``, 64 tokens of every KV head per page, for keys and values of
    ``dtype`` (bfloat16 or float16) with ``head_dim`` 32, 64 or 128.  A token
    takes 1.25 * head_dim bytes per KV head, against 4 * head_dim in 16 bits."""

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
