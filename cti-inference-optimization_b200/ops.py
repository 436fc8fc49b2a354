"""Tensor-level wrappers of the five hot-path stages.

Each function validates its tensors, passes raw device pointers and the
current CUDA stream to one ``libcti_b200.so`` entry point, and returns torch
tensors.  They are the building blocks of :class:`SMoE` and
:class:`RepEncoder`, and what the parity tests drive stage by stage.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from ._lib import check, lib, ptr, require_cuda, stream_handle, status_word
from .kv_cache import PAGE_TOKENS, KV4Cache


@dataclass
class RouterOut:
    idx2: torch.Tensor  # [T, 2] int32 expert ids (top-1, top-2)
    gate2: torch.Tensor  # [T, 2] fp32 gate weights
    route_rank: torch.Tensor  # [T, 2] int32 rank inside the 128-token router block
    block_hist: torch.Tensor  # [ceil(T/128), E] int32 per-block expert counts


@dataclass
class DispatchOut:
    offsets: torch.Tensor  # [E+1] int32 expert segment starts
    perm_inv: torch.Tensor  # [T, 2] int32 sorted position of each route
    sorted_token: torch.Tensor  # [2T] int32 token of each sorted row
    xperm: torch.Tensor | None  # [2T, D] bf16 rows in expert order


def router(x: torch.Tensor, wg: torch.Tensor, bg: torch.Tensor, renorm: bool = True) -> RouterOut:
    """Stage 1: fp32 Top-2 router (see cti_moe_router)."""
    require_cuda(x, "x", torch.bfloat16)
    require_cuda(wg, "wg", torch.float32)
    require_cuda(bg, "bg", torch.float32)
    T, D = x.shape
    E = wg.shape[0]
    dev = x.device
    nblk = (T + _lib.ROUTER_BLOCK_TOKENS - 1) // _lib.ROUTER_BLOCK_TOKENS
    idx2 = torch.empty((T, 2), dtype=torch.int32, device=dev)
    gate2 = torch.empty((T, 2), dtype=torch.float32, device=dev)
    rank = torch.empty((T, 2), dtype=torch.int32, device=dev)
    hist = torch.empty((max(nblk, 1), E), dtype=torch.int32, device=dev)
    check(
        lib.cti_moe_router(
            ptr(x), ptr(wg), ptr(bg), T, D, E, int(renorm), ptr(idx2), ptr(gate2), ptr(rank),
            ptr(hist), ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_moe_router",
    )
    return RouterOut(idx2, gate2, rank, hist)


def dispatch(x: torch.Tensor, r: RouterOut, num_experts: int, permute: bool = True) -> DispatchOut:
    """Stage 2: offsets + stable permutation of rows into expert order.

    Consumes ``r.block_hist`` (rewritten in place into per-block bases)."""
    require_cuda(x, "x", torch.bfloat16)
    T, D = x.shape
    dev = x.device
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    perm_inv = torch.empty((T, 2), dtype=torch.int32, device=dev)
    sorted_token = torch.empty(2 * T, dtype=torch.int32, device=dev)
    xperm = torch.empty((2 * T, D), dtype=torch.bfloat16, device=dev) if permute else None
    check(
        lib.cti_moe_dispatch(
            ptr(x), ptr(r.idx2), ptr(r.route_rank), ptr(r.block_hist), T, D, num_experts,
            ptr(offsets), ptr(perm_inv), ptr(sorted_token), ptr(xperm),
            ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_moe_dispatch",
    )
    return DispatchOut(offsets, perm_inv, sorted_token, xperm)


def grouped_gemm(
    a: torch.Tensor,
    w: torch.Tensor,
    bias: torch.Tensor | None,
    group_offsets: torch.Tensor,
    act: str = "none",
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Stage 3: C = act(A[group rows] @ W[g % Gw]^T + bias[g % Gw]).

    a [rows, K] bf16; w [Gw, N, K] bf16; bias [Gw, N] fp32 or None;
    group_offsets [G+1] int32 on the device."""
    require_cuda(a, "A", torch.bfloat16)
    require_cuda(w, "W", torch.bfloat16)
    require_cuda(group_offsets, "group_offsets", torch.int32)
    if bias is not None:
        require_cuda(bias, "bias", torch.float32)
    rows, K = a.shape
    Gw, N, K2 = w.shape
    if K2 != K:
        raise ValueError(f"K mismatch: A has {K}, W has {K2}")
    G = group_offsets.numel() - 1
    dev = a.device
    if out is None:
        out = torch.empty((rows, N), dtype=torch.bfloat16, device=dev)
    check(
        lib.cti_moe_grouped_gemm(
            ptr(a), ptr(w), ptr(bias), ptr(group_offsets), G, Gw, rows, N, K,
            _lib.ACTIVATIONS[act], ptr(out), ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_moe_grouped_gemm",
    )
    return out


def expert_ffn_fused(
    xp: torch.Tensor,
    w1: torch.Tensor,
    b1: torch.Tensor,
    w2: torch.Tensor,
    b2: torch.Tensor,
    group_offsets: torch.Tensor,
    act: str = "gelu",
    out: torch.Tensor | None = None,
    pair: bool = False,
) -> torch.Tensor:
    """Stage 3, fused: Y = act(Xp @ W1[e]^T + b1[e]) @ W2[e]^T + b2[e] per group.
    ``pair``: the CTA-pair kernel (cti_moe_expert_ffn_fused_pair, d_model 256)."""
    require_cuda(xp, "Xp", torch.bfloat16)
    require_cuda(w1, "W1", torch.bfloat16)
    require_cuda(w2, "W2", torch.bfloat16)
    require_cuda(b1, "b1", torch.float32)
    require_cuda(b2, "b2", torch.float32)
    rows, D = xp.shape
    Gw, F, _ = w1.shape
    G = group_offsets.numel() - 1
    dev = xp.device
    if out is None:
        out = torch.empty((rows, D), dtype=torch.bfloat16, device=dev)
    fn = lib.cti_moe_expert_ffn_fused_pair if pair else lib.cti_moe_expert_ffn_fused
    check(
        fn(
            ptr(xp), ptr(w1), ptr(b1), ptr(w2), ptr(b2), ptr(group_offsets), G, Gw, rows, D, F,
            _lib.ACTIVATIONS[act], ptr(out), ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_moe_expert_ffn_fused_pair" if pair else "cti_moe_expert_ffn_fused",
    )
    return out


def expert_ffn_fused_gather(
    x: torch.Tensor,
    sorted_token: torch.Tensor,
    w1: torch.Tensor,
    b1: torch.Tensor,
    w2: torch.Tensor,
    b2: torch.Tensor,
    group_offsets: torch.Tensor,
    act: str = "gelu",
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Stage 3, fused, rows gathered in the kernel: row r is x[sorted_token[r]]
    (no dispatched copy of the rows).  Equals expert_ffn_fused on the
    dispatched rows bit for bit."""
    require_cuda(x, "x", torch.bfloat16)
    require_cuda(sorted_token, "sorted_token", torch.int32)
    require_cuda(w1, "W1", torch.bfloat16)
    require_cuda(w2, "W2", torch.bfloat16)
    require_cuda(b1, "b1", torch.float32)
    require_cuda(b2, "b2", torch.float32)
    T, D = x.shape
    rows = sorted_token.numel()
    Gw, F, _ = w1.shape
    G = group_offsets.numel() - 1
    dev = x.device
    if out is None:
        out = torch.empty((rows, D), dtype=torch.bfloat16, device=dev)
    check(
        lib.cti_moe_expert_ffn_fused_gather(
            ptr(x), T, ptr(sorted_token), ptr(w1), ptr(b1), ptr(w2), ptr(b2), ptr(group_offsets),
            G, Gw, rows, D, F, _lib.ACTIVATIONS[act], ptr(out), ptr(status_word(dev)),
            stream_handle(dev),
        ),
        "cti_moe_expert_ffn_fused_gather",
    )
    return out


def combine(y: torch.Tensor, perm_inv: torch.Tensor, gate2: torch.Tensor,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """Stage 4: out[t] = g0*Y[perm_inv[t,0]] + g1*Y[perm_inv[t,1]] (fp32 math, bf16 out)."""
    require_cuda(y, "Y", torch.bfloat16)
    require_cuda(perm_inv, "perm_inv", torch.int32)
    require_cuda(gate2, "gate2", torch.float32)
    T = perm_inv.shape[0]
    D = y.shape[1]
    dev = y.device
    if out is None:
        out = torch.empty((T, D), dtype=torch.bfloat16, device=dev)
    check(
        lib.cti_moe_combine(
            ptr(y), y.shape[0], ptr(perm_inv), ptr(gate2), T, D, ptr(out),
            ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_moe_combine",
    )
    return out


def embedding_bag_sum(
    values: torch.Tensor,
    row_offsets: torch.Tensor,
    val_offsets: torch.Tensor,
    table: torch.Tensor,
    table_row_base: torch.Tensor,
    vocab: torch.Tensor,
    num_features: int,
    out_dtype: torch.dtype = torch.float32,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Stage 5: pooled[b, f*dim:(f+1)*dim] = sum of clamped table rows of bag (b, f).

    The reference's flat layout: values int64 [N]; row_offsets int64
    [F*(B+1)] per-feature offsets; val_offsets int64 [F]."""
    for name, t in (("values", values), ("row_offsets", row_offsets),
                    ("val_offsets", val_offsets), ("table_row_base", table_row_base),
                    ("vocab", vocab)):
        require_cuda(t, name, torch.int64)
    require_cuda(table, "table", torch.float16)
    F = num_features
    if row_offsets.numel() % F != 0:
        raise ValueError("row_offsets length must be a multiple of the feature count")
    B = row_offsets.numel() // F - 1
    dim = table.shape[1]
    dev = table.device
    if out is None:
        out = torch.empty((B, F * dim), dtype=out_dtype, device=dev)
    check(
        lib.cti_embbag_sum(
            ptr(values), values.numel(), ptr(row_offsets), ptr(val_offsets),
            ptr(table_row_base), ptr(vocab), ptr(table), table.shape[0], B, F, dim, ptr(out),
            _lib.DTYPE_CODES[out.dtype], ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_embbag_sum",
    )
    return out


def rep_encoder_fused(values: torch.Tensor, row_offsets: torch.Tensor, val_offsets: torch.Tensor,
                      table: torch.Tensor, table_row_base: torch.Tensor, vocab: torch.Tensor,
                      num_features: int, wg: torch.Tensor, r1: torch.Tensor, c: torch.Tensor,
                      eps: float = 1e-5, out: torch.Tensor | None = None) -> torch.Tensor:
    """The RepEncoder in one launch (cti_rep_encoder_fused): the embedding-bag
    pooling of ``embedding_bag_sum`` (64-wide fp16 rows), LayerNorm over the
    pooled row and the Linear, with the LayerNorm folded into the weights:
    ``wg`` bf16 [N, F*64] = W * gamma, ``r1`` fp32 [N] = wg.float().sum(1),
    ``c`` fp32 [N] = W beta + b.  Returns bf16 [B, N]; N in {128, 256}."""
    for name, t in (("values", values), ("row_offsets", row_offsets),
                    ("val_offsets", val_offsets), ("table_row_base", table_row_base),
                    ("vocab", vocab)):
        require_cuda(t, name, torch.int64)
    require_cuda(table, "table", torch.float16)
    require_cuda(wg, "wg", torch.bfloat16)
    require_cuda(r1, "r1", torch.float32)
    require_cuda(c, "c", torch.float32)
    F = num_features
    if row_offsets.numel() % F != 0:
        raise ValueError("row_offsets length must be a multiple of the feature count")
    B = row_offsets.numel() // F - 1
    dim = table.shape[1]
    N = wg.shape[0]
    if wg.shape[1] != F * dim or r1.numel() != N or c.numel() != N:
        raise ValueError("wg must be [N, F*dim] with r1, c of length N")
    dev = table.device
    if out is None:
        out = torch.empty((B, N), dtype=torch.bfloat16, device=dev)
    check(
        lib.cti_rep_encoder_fused(
            ptr(values), values.numel(), ptr(row_offsets), ptr(val_offsets),
            ptr(table_row_base), ptr(vocab), ptr(table), table.shape[0], B, F, dim, ptr(wg),
            ptr(r1), ptr(c), N, float(eps), ptr(out), ptr(status_word(dev)), stream_handle(dev),
        ),
        "cti_rep_encoder_fused",
    )
    return out


def add_layernorm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                  bias: torch.Tensor, eps: float = 1e-5, write_sum: bool = True):
    """The CTR model's residual add + LayerNorm: s = x + residual (bf16), out =
    LayerNorm(s).  Returns (s, out); s is x itself when residual is None.
    x, residual [rows, cols] bf16; weight, bias [cols] bf16."""
    require_cuda(x, "x", torch.bfloat16)
    if residual is not None:
        require_cuda(residual, "residual", torch.bfloat16)
        if residual.shape != x.shape:
            raise ValueError("x and residual must have the same shape")
    require_cuda(weight, "weight", torch.bfloat16)
    require_cuda(bias, "bias", torch.bfloat16)
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    dev = x.device
    out = torch.empty_like(x)
    s = torch.empty_like(x) if (residual is not None and write_sum) else None
    check(
        lib.cti_add_layernorm(ptr(x), ptr(residual), ptr(weight), ptr(bias), rows, cols,
                              float(eps), ptr(s), ptr(out), stream_handle(dev)),
        "cti_add_layernorm",
    )
    return (x if residual is None else s), out


def varlen_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     cu_seqlens: torch.Tensor, max_seqlen: int) -> torch.Tensor:
    """Causal attention inside packed sequences.  q, k, v [T, H, 32] bf16
    views whose last two dims are contiguous (any token stride, e.g. the
    thirds of one qkv projection); cu_seqlens int32 [N+1].  Returns a new
    contiguous [T, H, 32] bf16 tensor."""
    T, H, hd = q.shape
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda or t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be a bf16 CUDA tensor")
        if t.shape != q.shape or t.stride(2) != 1 or t.stride(1) != hd:
            raise ValueError(f"{name} must be [T, H, head_dim] with contiguous heads")
    require_cuda(cu_seqlens, "cu_seqlens", torch.int32)
    out = torch.empty((T, H, hd), dtype=torch.bfloat16, device=q.device)
    check(
        lib.cti_varlen_attention(ptr(q), ptr(k), ptr(v), q.stride(0), k.stride(0), v.stride(0),
                                 ptr(cu_seqlens), cu_seqlens.numel() - 1, int(max_seqlen), T, H,
                                 hd, ptr(out), ptr(status_word(q.device)),
                                 stream_handle(q.device)),
        "cti_varlen_attention",
    )
    return out


def ctr_head(h: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, w2: torch.Tensor,
             b2: torch.Tensor, limit: float = 15.0, want_logits: bool = True,
             want_probs: bool = True):
    """The CTR head in one launch (cti_ctr_head): logits = clamp(w2 .
    relu(W1 h + b1) + b2, +-limit) and probs = sigmoid(logits), fp32 [T].
    h [T, D] bf16; w1 [Hd, D] bf16; b1 [Hd], w2 [Hd], b2 [1] fp32.  Returns
    (logits or None, probs or None)."""
    require_cuda(h, "h", torch.bfloat16)
    require_cuda(w1, "W1", torch.bfloat16)
    for name, t in (("b1", b1), ("w2", w2), ("b2", b2)):
        require_cuda(t, name, torch.float32)
    T, D = h.shape
    Hd = w1.shape[0]
    dev = h.device
    logits = torch.empty(T, dtype=torch.float32, device=dev) if want_logits else None
    probs = torch.empty(T, dtype=torch.float32, device=dev) if want_probs else None
    check(
        lib.cti_ctr_head(ptr(h), ptr(w1), ptr(b1), ptr(w2), ptr(b2), T, D, Hd, float(limit),
                         ptr(logits), ptr(probs), ptr(status_word(dev)), stream_handle(dev)),
        "cti_ctr_head",
    )
    return logits, probs


_INT32 = torch.int32


def _kv4_run(cache: KV4Cache, fn, what: str, args: tuple) -> None:
    """Calls a kv4 entry point on the cache's device and its current stream."""
    index = cache.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, status_word(cache.device).data_ptr(), stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, status_word(cache.device).data_ptr(), stream)
    if rc:
        check(rc, what)


def _kv4_rows(t: torch.Tensor, name: str, cache: KV4Cache, heads: int) -> tuple[int, int]:
    """(tokens, token stride) of a [tokens, heads, head_dim] view with contiguous heads in the
    cache's type."""
    hd = cache.head_dim
    if t.dtype is not cache.dtype or not t.is_cuda:
        raise TypeError(f"{name} must be a {cache.dtype} CUDA tensor")
    if t.get_device() != cache.index:
        raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != hd:
        raise ValueError(f"{name} must be [tokens, {heads}, {hd}], got {tuple(shape)}")
    n, stride = shape[0], t.stride()
    if n and (stride[2] != 1 or (heads > 1 and stride[1] != hd)):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] with contiguous heads")
    return n, stride[0] if n > 1 else heads * hd  # a single token has any stride


def _kv4_index(cache: KV4Cache, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
               page_table: torch.Tensor) -> tuple:
    """Checks the index tensors; the arguments that every kv4 entry point takes of them, up to the
    number of sequences."""
    index, shape = cache.index, page_table.shape
    n = kv_lens.numel()
    if (index >= 0 and cu_seqlens.dtype is _INT32 and kv_lens.dtype is _INT32
            and page_table.dtype is _INT32 and cu_seqlens.get_device() == index
            and kv_lens.get_device() == index and page_table.get_device() == index
            and kv_lens.dim() == 1 and cu_seqlens.dim() == 1 and cu_seqlens.numel() == n + 1
            and len(shape) == 2 and shape[0] == n and kv_lens.is_contiguous()
            and cu_seqlens.is_contiguous()):
        cols, stride = shape[1], page_table.stride()
        if not n or cols <= 1 or stride[1] == 1:
            return (cu_seqlens.data_ptr(), kv_lens.data_ptr(), page_table.data_ptr(),
                    stride[0] if n > 1 else cols, cols, n)
    raise _kv4_index_error(cache, cu_seqlens, kv_lens, page_table)


def _kv4_index_error(cache, cu_seqlens, kv_lens, page_table) -> Exception:
    """What is wrong with the index tensors."""
    if cache.index < 0:
        return RuntimeError("the cache must be on a CUDA device (this library has no CPU path)")
    for name, t, dims in (("cu_seqlens", cu_seqlens, 1), ("kv_lens", kv_lens, 1),
                          ("page_table", page_table, 2)):
        if t.dtype is not _INT32 or not t.is_cuda:
            return TypeError(f"{name} must be an int32 CUDA tensor, got {t.dtype} on {t.device}")
        if t.get_device() != cache.index:
            return ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
        if t.dim() != dims or (dims == 1 and not t.is_contiguous()):
            return ValueError(f"{name} must have {dims} contiguous dimension(s), got "
                              f"{tuple(t.shape)}")
    return ValueError("kv_lens must be [N], cu_seqlens [N + 1] and page_table [N, pages] with "
                      f"contiguous rows, got {tuple(kv_lens.shape)}, {tuple(cu_seqlens.shape)} "
                      f"and {tuple(page_table.shape)}")


@lru_cache(maxsize=256)
def _kv4_workspace_bytes(*sizes: int) -> int:
    return lib.cti_kv4_attention_workspace_bytes(*sizes)


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
               kv_lens: torch.Tensor, page_table: torch.Tensor) -> None:
    """Quantises keys and values into the 4-bit cache (see cti_kv4_append).
    k, v [tokens, kv_heads, head_dim] views of the cache's dtype (any token
    stride); cu_seqlens int32 [N+1] packs them by sequence; kv_lens int32 [N]
    are the sequences' lengths with these tokens, which are their last;
    page_table int32 [N, pages].  A position past the table or a page outside
    the cache is skipped and reported in the device status word.  A group of 32
    head dims with a value that is not finite, or with magnitudes of 20,900
    (float16) or 1e38 (bfloat16) and more, is held as NaN."""
    seqs = _kv4_index(cache, cu_seqlens, kv_lens, page_table)
    H = cache.kv_heads
    tokens, k_stride = _kv4_rows(k, "k", cache, H)
    v_tokens, v_stride = _kv4_rows(v, "v", cache, H)
    if v_tokens != tokens:
        raise ValueError("k and v must have the same number of tokens")
    pages = cache.pages
    _kv4_run(cache, lib.cti_kv4_append, "cti_kv4_append",
             (k.data_ptr(), v.data_ptr(), k_stride, v_stride, cache.dtype_code, *seqs, tokens, H,
              cache.head_dim, pages.data_ptr(), pages.size(0)))


def kv4_read(cache: KV4Cache, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
             page_table: torch.Tensor, tokens: int,
             out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """What the cache holds for the last cu_seqlens[i+1] - cu_seqlens[i] tokens
    of every sequence (see cti_kv4_read): (k, v), each [tokens, kv_heads,
    head_dim] in the cache's dtype.  ``tokens`` is cu_seqlens[-1]; with
    cu_seqlens the offsets of kv_lens, whole sequences are read.  ``out``: the
    two tensors to write (rows of no sequence keep their contents)."""
    seqs = _kv4_index(cache, cu_seqlens, kv_lens, page_table)
    H, hd = cache.kv_heads, cache.head_dim
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    if out is None:
        k = torch.empty((tokens, H, hd), dtype=cache.dtype, device=cache.device)
        v = torch.empty_like(k)
        k_stride = v_stride = H * hd
    else:
        k, v = out
        k_tokens, k_stride = _kv4_rows(k, "out[0]", cache, H)
        v_tokens, v_stride = _kv4_rows(v, "out[1]", cache, H)
        if k_tokens != tokens or v_tokens != tokens:
            raise ValueError(f"out must hold {tokens} tokens")
    pages = cache.pages
    _kv4_run(cache, lib.cti_kv4_read, "cti_kv4_read",
             (pages.data_ptr(), pages.size(0), cache.dtype_code, *seqs, tokens, H, hd,
              k.data_ptr(), v.data_ptr(), k_stride, v_stride))
    return k, v


def kv4_attention(q: torch.Tensor, cache: KV4Cache, cu_seqlens: torch.Tensor,
                  kv_lens: torch.Tensor, page_table: torch.Tensor, max_new: int | None = None,
                  causal: bool = True, scale: float | None = None,
                  max_kv_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over the 4-bit cache, which holds their own keys
    and values already (see cti_kv4_attention).  q [tokens, heads, head_dim]
    view of the cache's dtype, heads a multiple of the cache's kv_heads (query
    head h reads KV head h // (heads // kv_heads)); the other arguments as in
    kv4_append.  causal: a token sees the keys up to its own position, else all
    of its sequence's.  scale: of the scores, 1 / sqrt(head_dim) by default.
    max_new, max_kv_len: bounds of the new tokens of a sequence and of kv_lens
    (defaults: from the token count and the table's width); the work is split
    by them, results hold for any.  Returns a contiguous [tokens, heads,
    head_dim]; a token that sees no key is zero, and rows of no sequence are
    not written.  Relative error of a row: 0.0022 in bfloat16 and 0.0003 in
    float16 for few tokens, 0.0017 and 0.0003 where they are taken in tiles of
    128 rows."""
    seqs = _kv4_index(cache, cu_seqlens, kv_lens, page_table)
    hd, Hkv = cache.head_dim, cache.kv_heads
    H = q.shape[1] if q.dim() == 3 else 0
    if H <= 0 or H % Hkv:
        raise ValueError(f"q must be [tokens, heads, head_dim] with heads a multiple of {Hkv}, "
                         f"got {tuple(q.shape)}")
    T, q_stride = _kv4_rows(q, "q", cache, H)
    cols, n = seqs[4], seqs[5]
    if max_new is None:
        max_new = 1 if T <= n else T
    if max_kv_len is None:
        max_kv_len = cols * PAGE_TOKENS
    if scale is None:
        scale = hd ** -0.5
    if out is None:
        out = q.new_empty((T, H, hd))
    else:
        _kv4_rows(out, "out", cache, H)
        if out.size(0) != T or not out.is_contiguous():
            raise ValueError("out must be contiguous, of q's shape")
    # Bounds may be as large as one likes: the C entry point takes 32 and 64 bits.
    max_new, max_kv_len = min(int(max_new), T), min(int(max_kv_len), 2 ** 62)
    need = _kv4_workspace_bytes(n, T, max_new, max_kv_len, H, Hkv, hd)
    ws = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    pages = cache.pages
    _kv4_run(cache, lib.cti_kv4_attention, "cti_kv4_attention",
             (q.data_ptr(), q_stride, cache.dtype_code, *seqs, T, max_new, max_kv_len, H, Hkv, hd,
              float(scale), 1 if causal else 0, pages.data_ptr(), pages.size(0), out.data_ptr(),
              ptr(ws), need))
    return out
