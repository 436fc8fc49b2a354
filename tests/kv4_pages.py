"""Values that name their page (test only): dim p % head_dim of a token in page p is 1, the others 0,
and with a scale of zero every key that a row sees counts alike.  A page that is left out, counted
twice, or counted for another row shows in full in its dim."""
import torch

import kv4_ref as ref


def values(total, heads, head_dim, dtype):
    v = torch.zeros(sum(total), heads, head_dim, dtype=dtype)
    at = 0
    for L in total:
        t = torch.arange(L)
        v[at + t, :, t // ref.PAGE % head_dim] = 1
        at += L
    return v


def expected(v, heads, new, total, causal, dropped=None):
    """(out, tol) in float64 for `heads` query heads.  dropped: (sequence, page) that is left out (what
    the test must notice).  With a scale of zero weights and their sum are whole numbers times a
    power of two, exact in every type that they pass through.  With e the type's half step: each
    value is rounded to the type, or to fp16, whose half step is no larger, 2 e A at most with
    the scale's and base's, A = the mean of |v|; the output, once: e |out|; fp32 sums of up to
    2^13 terms: 2^-11 A; and fp16's smallest step for small values."""
    held = ref.held(v)
    group = heads // v.shape[1]
    D = v.shape[2]
    out = torch.zeros(sum(new), heads, D, dtype=torch.float64)
    A = torch.zeros_like(out)
    n0 = t0 = 0
    for i, (n, L) in enumerate(zip(new, total)):
        x = held[t0:t0 + L].repeat_interleave(group, 1)
        pos = L - n + torch.arange(n) if causal else torch.full((n,), L - 1)
        sees = (torch.arange(L)[None, :] <= pos[:, None]).double()
        if dropped is not None and dropped[0] == i:
            sees[:, ref.PAGE * dropped[1]:ref.PAGE * (dropped[1] + 1)] = 0
        w = sees / sees.sum(-1, keepdim=True).clamp(min=1)
        out[n0:n0 + n] = torch.einsum("nl,lhd->nhd", w, x)
        A[n0:n0 + n] = torch.einsum("nl,lhd->nhd", w, x.abs())
        n0, t0 = n0 + n, t0 + L
    e = ref.rounding(v.dtype)
    return out, e * out.abs() + (2 * e + 2.0 ** -11) * A + 2.0 ** -24


# Sequences' new tokens and lengths: few and long (split over blocks), one whose last page holds one
# token, tiles of 128 rows, many rows of short sequences.
CALLS = [([1], [64 * 129 + 1]), ([1, 1], [3000, 5]), ([5, 40], [4100, 2500]),
         ([3, 1, 2], [700, 1, 64 * 20]), ([150], [4000]), ([257, 1, 300], [900, 1000, 300]),
         ([90, 100, 70], [2049, 640, 70])]
