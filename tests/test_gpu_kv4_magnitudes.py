"""Attention over the 4-bit cache, for values, keys, queries and scales of all magnitudes: the error
of each row's output as a vector, against the 64-bit form on what the cache holds.

The tolerance.  With e the tensors' type's half step (finfo.eps / 2) and f = 2^-11 fp16's:
  - up to 96 rows of a KV head (warps): the values and the output are rounded to the type;
  - from 97 rows on (tiles): the output is rounded to the type, keys, values and weights to fp16.
Each rounding moves a term of sum_j p_j v_j by at most its half step relative to the term, one
term's error is independent of the next one's, and so is the terms' own sign: errors of both
kinds add up as the roots of sums of squares, and the ratio of the two is sqrt(2) e for warps and
sqrt(e^2 + 3 f^2) for tiles.  (A key's rounding moves a score by its half step times the root of the
sum of q_d^2 k_d^2 scale^2, about the scores' standard deviation, which these tests keep near 1, and
a weight as much.)  The rounding errors' mean square is a third of the half step's or less, which
leaves a factor of sqrt(3) for rows whose terms happen to cancel more than others': 1.5 is used."""
import math

import pytest
import torch

import kv4_pages as pages
import kv4_ref as ref
from test_gpu_kv4 import TYPES, Setup

pytestmark = pytest.mark.gpu

SHAPES = [(2, 2, 32), (4, 2, 64), (2, 1, 128)]
# New tokens of the sequence: one row, a few, and tiles of 128 rows for all SHAPES.
TOKENS = [1, 12, 100, 150]


def _tolerance(dtype, tiles):
    e, f = ref.rounding(dtype), 2.0 ** -11
    return 1.5 * math.sqrt(e * e + 3 * f * f if tiles else 2 * e * e)


def _check(s, dtype, tiles, scale=None, causal=True, held=ref.held, **kw):
    """The largest error of a row, relative to the row."""
    from cti_b200 import _lib, ops

    D = s.q.shape[2]
    out = ops.kv4_attention(s.q.to(s.dev), s.cache, s.cu, s.lens, s.table, causal=causal,
                            scale=scale, **kw)
    _lib.raise_on_status(s.dev)
    want, _ = ref.attention(s.q, held(s.k), held(s.v), s.new, s.total, causal,
                            D ** -0.5 if scale is None else scale)
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    off = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max()
    assert off <= _tolerance(dtype, tiles), float(off)


def _setup(dev, n, total, H, Hkv, D, dtype, size_k=1.0, size_v=1.0, size_q=1.0):
    """size_k, size_v: of the keys and values, a number or one for each token."""
    g = torch.Generator().manual_seed(n + total + D)
    size_k, size_v = (torch.as_tensor(x, dtype=torch.float64).reshape(-1, 1, 1)
                      for x in (size_k, size_v))
    k = (torch.randn(total, Hkv, D, generator=g) * size_k).to(dtype)
    v = (torch.randn(total, Hkv, D, generator=g) * size_v).to(dtype)
    s = Setup(dev, [n], [total], H, Hkv, D, dtype, k=k, v=v)
    s.q = (s.q.double() * size_q).to(dtype)
    return s


def _by_page(total, sizes):
    return torch.tensor(sizes, dtype=torch.float64)[torch.arange(total) // 64 % len(sizes)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("total", [400, 2500])
def test_small_values_beside_a_larger_page_and_a_sink(cuda_device, dtype, H, Hkv, D, n, total):
    """Values of 0.003, twice that in the first page, and a key whose value is next to nothing and
    whose score is 6 above the others': the output is what the small weights give."""
    s = _setup(cuda_device, n, total, H, Hkv, D, dtype,
               size_v=torch.where(torch.arange(total) < 64, 0.006, 0.003))
    s.k[3], s.v[3] = 6 / D ** 0.5, 1e-4
    s.q = (s.q.float() + 1.0).to(dtype)
    t = Setup(cuda_device, [n], [total], H, Hkv, D, dtype, k=s.k, v=s.v)
    t.q = s.q
    _check(t, dtype, n >= 100, max_new=n)
    _check(t, dtype, n >= 100, max_new=n, causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("sizes", [[0.002, 0.008], [0.008, 0.002], [700.0, 2800.0],
                                   [0.02, 50.0, 0.5, 0.02]])
def test_pages_of_different_magnitudes(cuda_device, dtype, H, Hkv, D, n, sizes):
    """One range of pages (a sequence of 7) and several (of 40)."""
    for total in (400, 2500):
        s = _setup(cuda_device, n, total, H, Hkv, D, dtype, size_v=_by_page(total, sizes))
        _check(s, dtype, n >= 100, max_new=n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("last", [1, 2, 3])
def test_small_values_and_a_last_page_of_a_few_tokens(cuda_device, dtype, H, Hkv, D, last):
    for n in (1, 100, 150):
        s = _setup(cuda_device, n, 384 + last, H, Hkv, D, dtype, size_v=0.004)
        _check(s, dtype, n >= 100, max_new=n)


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("total", [400, 2500])
def test_values_at_the_ends_of_the_range(cuda_device, H, Hkv, D, n, total):
    """Of bf16: values of 1e37, all of one sign, so that their weighted sum before it is divided
    passes fp32's range; of 1e36 of both signs; and of 1e-34."""
    for size, mean in ((1e36, 1e37), (1e36, 0.0), (1e-34, 0.0)):
        s = _setup(cuda_device, n, total, H, Hkv, D, torch.bfloat16, size_v=size)
        s = Setup(cuda_device, [n], [total], H, Hkv, D, torch.bfloat16, k=s.k,
                  v=(s.v.double() + mean).bfloat16())
        _check(s, torch.bfloat16, n >= 100, max_new=n)


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("size_q,size_k", [(1e34, 1e-34), (2e37, 1e-33), (1e-34, 1e34)])
def test_queries_at_the_ends_of_the_range(cuda_device, H, Hkv, D, n, size_q, size_k):
    """Of bf16, whose scores are ordinary."""
    s = _setup(cuda_device, n, 400, H, Hkv, D, torch.bfloat16, size_k=size_k, size_q=size_q)
    _check(s, torch.bfloat16, n >= 100, scale=D ** -0.5 / (size_q * size_k), max_new=n)


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
def test_scale_of_zero_and_next_to_it(cuda_device, H, Hkv, D, n):
    """A scale of zero weighs all keys alike, whatever their size; one of 1e-36 belongs to keys, or
    queries, of 1e36, and one of 1e-42, below fp32's normal numbers, to both."""
    for size_q, size_k, scale in ((1e10, 1e30, 0.0), (1.0, 1e36, 1e-36), (3e30, 3e5, 1e-36),
                                  (1e20, 1e22, 1e-42), (1e-20, 1e30, -1e-10)):
        s = _setup(cuda_device, n, 400, H, Hkv, D, torch.bfloat16, size_k=size_k, size_q=size_q)
        scale *= D ** -0.5
        # fp32's numbers below 1e-38 have few bits: the scale that the call is given
        scale = float(torch.tensor(scale, dtype=torch.float32))
        _check(s, torch.bfloat16, n >= 100, scale=scale, max_new=n)
        _check(s, torch.bfloat16, n >= 100, scale=scale, max_new=n, causal=False)


@pytest.mark.parametrize("dtype,lo", [(torch.float16, 2161.632), (torch.bfloat16, 1.26258875e37)])
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_a_group_whose_top_code_passes_the_type(cuda_device, dtype, lo, H, Hkv, D):
    """Values up to the type's largest: the scale's rounding can take the group's top past it.  Such
    a group is NaN as a whole, and reaches only the rows that see its token."""
    from cti_b200 import _lib, ops

    total = 200
    hi = torch.finfo(dtype).max
    ramp = (lo + (hi - lo) * torch.linspace(0, 1, 32, dtype=torch.float64)).to(dtype)
    _, s, b = ref.quantise(ramp)
    top = (31 * s + b).to(dtype)
    assert torch.isfinite(ramp).all() and torch.isfinite(b) and torch.isinf(top)
    below = (ramp.double() * 0.98).to(dtype)  # held: its top is within the type
    _, s, b = ref.quantise(below)
    assert torch.isfinite((31 * s + b).to(dtype))
    for n in (12, 150):
        t = _setup(cuda_device, n, total, H, Hkv, D, dtype)
        t.v[total - 1, 0, :32], t.k[0, 0, :32], t.v[total - n - 1, Hkv - 1, -32:] = ramp, 0, below
        t = Setup(cuda_device, [n], [total], H, Hkv, D, dtype, k=t.k, v=t.v)
        cu = torch.tensor([0, total], dtype=torch.int32, device=cuda_device)
        _, v = ops.kv4_read(t.cache, cu, t.lens, t.table, total)
        assert torch.isnan(v[total - 1, 0, :32]).all() and int(torch.isnan(v).sum()) == 32
        assert not torch.isinf(v).any()
        out = ops.kv4_attention(t.q.to(cuda_device), t.cache, t.cu, t.lens, t.table, max_new=n)
        _lib.raise_on_status(cuda_device)
        out = out.cpu()
        assert torch.isfinite(out[:n - 1]).all()
        assert torch.isnan(out[n - 1, :H // Hkv, :32]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("sink", [0, 2400])
def test_many_small_weights_beside_one_large(cuda_device, dtype, H, Hkv, D, n, sink):
    """A key of no value has a score 13 above the others' mean, at the sequence's start or near its
    end: the output comes from 2,500 weights of about 2^-18.8.  fp16 holds 11 bits of a number down
    to 2^-14, so they are rounded to 11 bits where they are formed 2^4.8 larger, or more.  The
    queries' first 32 dims are 1, and the key has no others, so its score is the same for all rows;
    values of 64 keep the output, of about 64 sqrt(2500) 2^-18.8 = 0.007, in fp16's normal range."""
    total = 2500
    s = _setup(cuda_device, n, total, H, Hkv, D, dtype, size_k=0.5, size_v=64.0)
    s.k[sink], s.v[sink] = 0.0, 0.0
    s.k[sink, :, :32] = 13.0 * D ** 0.5 / 32
    s.q[..., :32] = 1.0
    t = Setup(cuda_device, [n], [total], H, Hkv, D, dtype, k=s.k, v=s.v)
    t.q = s.q
    _check(t, dtype, n >= 100, max_new=n, causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 32), (6, 3, 64), (8, 2, 128)])
@pytest.mark.parametrize("new,total", pages.CALLS)
def test_ordinary_values(cuda_device, dtype, H, Hkv, D, new, total):
    """Numbers near 1, long and short, few rows and many, for every bound of the work."""
    g = torch.Generator().manual_seed(sum(total) + D)
    k, v = (torch.randn(sum(total), Hkv, D, generator=g).to(dtype) for _ in range(2))
    s = Setup(cuda_device, new, total, H, Hkv, D, dtype, k=k, v=v)
    for max_new in (max(new), 1, 200):
        # Tiles may be taken from 65 rows on or from 97: the larger of both kernels' bounds.
        tiles = dtype == torch.float16 and max_new * H // Hkv >= 65
        _check(s, dtype, tiles, max_new=max_new)
        _check(s, dtype, tiles, max_new=max_new, causal=False)


@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("n", TOKENS)
def test_groups_of_different_magnitudes(cuda_device, H, Hkv, D, n):
    """Values of 1e-5 in one group of dims beside values near 1: their own part of the output is as
    good as the others'.  So are scores that come from keys of 1e-5 where the queries' dims are
    1e5, beside keys near 1."""
    from cti_b200 import _lib, ops

    total = 700
    size = torch.ones(D, dtype=torch.float64)
    size[32:64] = 1e-5
    g = torch.Generator().manual_seed(n + D)
    k, v = ((torch.randn(total, Hkv, D, generator=g) * size).bfloat16() for _ in range(2))
    s = Setup(cuda_device, [n], [total], H, Hkv, D, torch.bfloat16, k=k, v=v)
    s.q = (s.q.double() / size * 0.7).bfloat16()
    out = ops.kv4_attention(s.q.to(cuda_device), s.cache, s.cu, s.lens, s.table, n)
    _lib.raise_on_status(cuda_device)
    want, _ = ref.attention(s.q, ref.held(k), ref.held(v), [n], [total], True, D ** -0.5)
    off = (out.double().cpu() - want).unflatten(-1, (-1, 32)).norm(dim=-1)
    off = (off / want.unflatten(-1, (-1, 32)).norm(dim=-1)).max()
    assert off <= _tolerance(torch.bfloat16, n >= 100), float(off)


@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (16, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("n", [16, 110, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_fp16_is_rounded_twice_whatever_the_rows(cuda_device, H, Hkv, D, n, causal):
    """Keys with channels of their own size and offset, as projections give them.  Two roundings to
    fp16 count, whichever kernel runs: the output's and one of values and weights.  A rounding's
    mean square is a third of the half step's at most, so over all rows of a head the error is
    below sqrt(2 / 3) 2^-11 of the output."""
    from cti_b200 import _lib, ops

    total = 1500
    g = torch.Generator().manual_seed(n + D)
    k = torch.randn(total, Hkv, D, generator=g) * torch.exp(0.5 * torch.randn(Hkv, D, generator=g))
    k = (k + 0.7 * torch.randn(Hkv, D, generator=g)).half()
    v = torch.randn(total, Hkv, D, generator=g).half()
    s = Setup(cuda_device, [n], [total], H, Hkv, D, torch.float16, k=k, v=v)
    out = ops.kv4_attention(s.q.to(cuda_device), s.cache, s.cu, s.lens, s.table, n, causal=causal)
    _lib.raise_on_status(cuda_device)
    want, _ = ref.attention(s.q, ref.held(k), ref.held(v), [n], [total], causal, D ** -0.5)
    off = (out.double().cpu() - want).norm(dim=(0, 2)) / want.norm(dim=(0, 2))
    assert off.max() <= math.sqrt(2 / 3) * 2.0 ** -11, off.tolist()


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", TOKENS)
@pytest.mark.parametrize("where", [0, 3, 6])
@pytest.mark.parametrize("size", [1e15, 1e-15])
def test_a_page_of_other_magnitude_and_no_weight(cuda_device, H, Hkv, D, n, where, size):
    """One page's values are 1e15, or all others' are, and its keys' scores lie 150 below the
    others': it takes part in no output, and must not take the others' bits, whether it comes
    first, in between or last."""
    total = 448
    mine = torch.arange(total) // 64 == where
    s = _setup(cuda_device, n, total, H, Hkv, D, torch.bfloat16, size_k=0.7,
               size_v=torch.where(mine, size, 1.0) if size > 1 else torch.where(mine, 1.0, 1e15))
    s.k[mine] = 0.0
    s.k[mine, :, :32] = -150.0 * D ** 0.5 / 32
    s.q[..., :32] = 1.0
    t = Setup(cuda_device, [n], [total], H, Hkv, D, torch.bfloat16, k=s.k, v=s.v)
    t.q = s.q
    _check(t, torch.bfloat16, n >= 100, max_new=n, causal=False)
