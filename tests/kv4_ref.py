"""Plain 64-bit forms of the 4-bit cache's operators (test only): no pages, one
sequence at a time, every formula written out.  All tensors are on the CPU."""
import torch

GROUP = 32
PAGE = 64


def quantise(x):
    """(codes, scale, base) of x [..., head_dim] in float64, groups last but one."""
    y = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).to(x.dtype).double()
    b = (lo - 16 * s).to(x.dtype).double()
    n = torch.round((y - b) / torch.where(s > 0, s, 1.0)) - 16
    n = torch.where(s > 0, n.clamp(0, 15), 0.0)
    bad = ~torch.isfinite(b) | ~torch.isfinite(s)
    nan = torch.full_like(s, float("nan"))
    return torch.where(bad, 0.0, n), torch.where(bad, nan, s), torch.where(bad, nan, b)


def held(x):
    """What x [..., head_dim] is held as, in float64."""
    n, s, b = quantise(x)
    return ((16 + n) * s + b).flatten(-2)


def rounding(dtype):
    """Relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, new, total, causal, scale):
    """float64 attention of the last new[i] tokens of every sequence over its total[i]; q packs the
    new tokens, k and v (what the cache holds) all of them.  Returns (out, tol): tol bounds the
    error of an implementation that keeps scores, maxima, sums and outputs in fp32, rounds the
    weights p and the values once each to the tensors' type, may round the keys to 11 bits, and
    rounds the output.

    With e = eps / 2 of the type, u = 2^-24 of fp32, A = sum p |v|:
      p's and v's rounding: 2 e A; the output's: e |out|;
      p below the type's normals, or those of fp16 (the type may be bf16 and p, v held in fp16):
      half the smallest step, 2^-25, for each key, over a sum l >= 1;
      v's scale below fp16's normals: 31 2^-25 < 2^-20, or, after a common factor that takes a bound
      of 8 max |v| to 2^14 at least, 31 2^-25 8 2^-14 max |v| < 2^-31 max |v|;
      a score is off by at most d, so a weight by a factor of exp(+-2 d) with its sum: expm1(2 d) A.
    d, for a score q . k with k = (16 + n) s + b:
      - q (16 + n) s and q b may be summed apart, in fp32, over up to head_dim + 8 terms.  In a
        group with largest magnitude kmax, s <= 2 kmax / 15 and |b| <= kmax + 16 s, so 31 s + |b| <
        8 kmax: below 16 sum |q| kmax (head_dim + 8) u;
      - the sum of q over a group may be split into two numbers of the type, short by e^2 of
        itself, twice (for s and b): below 2 e^2 16 sum |q| kmax;
      - keys rounded to 11 bits: 2^-12 sum |q| |k|, and as for v 2^-20 max(1, 2^-11 max |k|) sum |q|."""
    dtype = q.dtype
    e, u = rounding(dtype), 2.0 ** -24
    tiny = 2.0 ** -25
    H, D = q.shape[1], q.shape[2]
    group = H // k.shape[1]

    def most(x):
        return float(torch.nan_to_num(x).abs().max()) if x.numel() else 0.0

    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    n0 = t0 = 0
    for n, L in zip(new, total):
        qs = q[n0:n0 + n].double()
        ks = k[t0:t0 + L].repeat_interleave(group, 1)
        vs = v[t0:t0 + L].repeat_interleave(group, 1)
        s = torch.einsum("nhd,lhd->hnl", qs, ks) * scale
        kmax = ks.abs().unflatten(-1, (-1, GROUP)).amax(-1, keepdim=True).expand(
            -1, -1, -1, GROUP).flatten(-2)
        d = torch.einsum("nhd,lhd->hnl", qs.abs(), kmax) * abs(scale) * 16 * (
            (D + 8) * u + 2 * e * e)
        d = d + abs(scale) * (2.0 ** -12 * torch.einsum("nhd,lhd->hnl", qs.abs(), ks.abs()) +
                              2.0 ** -20 * max(1.0, 2.0 ** -11 * most(ks)) *
                              qs.abs().sum(-1).T[:, :, None])
        if causal:
            pos = L - n + torch.arange(n)
            s = s.masked_fill(torch.arange(L)[None, :] > pos[:, None], float("-inf"))
        seen = torch.isfinite(s) | torch.isnan(s)
        some = seen.any(-1)
        p = torch.softmax(s, -1)
        p = torch.where(some[..., None], p, 0.0)
        # 0 * NaN of a key that is not seen counts as 0.
        vz = torch.nan_to_num(vs, nan=0.0)
        o = torch.einsum("hnl,lhd->nhd", torch.nan_to_num(p), vz)
        vnan = torch.isnan(vs).any(-1).T  # [h, l]
        bad = torch.isnan(p).any(-1) | (seen & vnan[:, None, :]).any(-1)  # [h, n]
        o[bad.T] = float("nan")
        A = torch.einsum("hnl,lhd->nhd", torch.nan_to_num(p), vz.abs())
        dmax = torch.where(seen, torch.nan_to_num(d), 0.0).amax(-1) if L else torch.zeros(H, n)
        few = torch.einsum("hnl,lhd->nhd", seen.double(), vz.abs())
        out[n0:n0 + n] = o
        tol[n0:n0 + n] = (e * o.abs() + 2 * e * A + torch.expm1(2 * dmax.T[..., None]) * A + 2.0 ** -20 * A +
                          tiny * few + 2.0 ** -20 * max(1.0, 2.0 ** -11 * most(vs))) * 1.01
        n0, t0 = n0 + n, t0 + L
    return out, tol


def page_table(total, pages, seed=0, extra=0):
    """A table of distinct random pages for sequences of total[i] tokens; entries past a sequence's
    last page are -1."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    need = [-(-t // PAGE) for t in total]
    assert sum(need) <= pages
    table = torch.full((len(total), max(need + [0]) + extra), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def offsets(lens):
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int64), 0).to(torch.int32)
    return cu
