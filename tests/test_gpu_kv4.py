"""The 4-bit key/value cache on the GPU against plain 64-bit forms (kv4_ref).

Reading back: the kernel forms (16 + n) s + b by one fp32 fused multiply-add and rounds it to the
type, so a value is off by at most e |value| (1 + 2^-23) + 2^-24 |value| with e the type's half
step, half the smallest step for subnormals; a wrong code is off by a whole step s, far more.
Attention: the bound is derived in kv4_ref.attention."""
import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _values(T, H, D, dtype, seed, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g) * torch.exp(spread * torch.randn(H, D, generator=g))
    return (x + 0.5 * torch.randn(H, D, generator=g)).to(dtype)


def _read_tolerance(want, dtype):
    fi = torch.finfo(dtype)
    return want.abs() * (fi.eps / 2 + 2.0 ** -23) + fi.smallest_normal * fi.eps / 2


def _check_read(got, x):
    want = ref.held(x)
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs() - _read_tolerance(want, x.dtype)
    assert not (off > 0).any(), float(off.nan_to_num().max())


class Setup:
    """Sequences of total[i] tokens, the last new[i] of them new, all appended."""

    def __init__(self, dev, new, total, H, Hkv, D, dtype, seed=0, k=None, v=None, extra=0):
        import cti_b200
        from cti_b200 import ops

        self.new, self.total, self.dev = new, total, dev
        T = sum(total)
        self.k = _values(T, Hkv, D, dtype, seed) if k is None else k
        self.v = _values(T, Hkv, D, dtype, seed + 1, 0.2) if v is None else v
        g = torch.Generator().manual_seed(seed + 2)
        self.q = torch.randn(sum(new), H, D, generator=g).to(dtype)
        pages = sum(-(-t // 64) for t in total) + 3
        self.cache = cti_b200.KV4Cache(pages, Hkv, D, dtype=dtype, device=dev)
        # What a page holds behind its sequence's end is never used.
        self.cache.pages.fill_(0xff)
        self.table = ref.page_table(total, pages, seed, extra).to(dev)
        self.lens = torch.tensor(total, dtype=torch.int32, device=dev)
        self.cu = ref.offsets(new).to(dev)
        ops.kv4_append(self.cache, self.k.to(dev), self.v.to(dev), ref.offsets(total).to(dev),
                       self.lens, self.table)

    def check(self, causal=True, scale=None, **kw):
        from cti_b200 import _lib, ops

        q = self.q.to(self.dev)
        out = ops.kv4_attention(q, self.cache, self.cu, self.lens, self.table, causal=causal,
                                scale=scale, **kw)
        _lib.raise_on_status(self.dev)
        self.compare(out, causal, scale)
        return out

    def compare(self, out, causal=True, scale=None):
        D = self.q.shape[2]
        want, tol = ref.attention(self.q, ref.held(self.k), ref.held(self.v), self.new, self.total,
                                  causal, D ** -0.5 if scale is None else scale)
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        got = out.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        off = (got - want).abs() - tol
        assert not (off > 0).any(), (float(off.nan_to_num().max()), float((off / tol).nan_to_num().max()))


# ---------------------------------------------------------------------------
# Writing and reading back.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,D", [(8, 32), (1, 32), (4, 64), (3, 64), (2, 128), (5, 128)])
def test_append_then_read(cuda_device, dtype, H, D):
    from cti_b200 import _lib, ops

    lens = [1, 63, 0, 64, 65, 200, 3, 128]
    s = Setup(cuda_device, lens, lens, H, H, D, dtype, seed=D + H)
    k, v = ops.kv4_read(s.cache, s.cu, s.lens, s.table, sum(lens))
    _lib.raise_on_status(cuda_device)
    _check_read(k, s.k)
    _check_read(v, s.v)


@pytest.mark.parametrize("dtype", TYPES)
def test_pieces_of_any_size_fill_the_cache_as_one_call_does(cuda_device, dtype):
    """Histories written a few tokens at a time, from strided views, leave the same bytes."""
    import cti_b200
    from cti_b200 import ops

    dev, H, D = cuda_device, 4, 64
    lens = [130, 64, 7, 1, 191]
    s = Setup(dev, lens, lens, H, H, D, dtype, seed=5)
    other = cti_b200.KV4Cache(s.cache.num_pages, H, D, dtype=dtype, device=dev)
    other.pages.fill_(0xff)
    ends = ref.offsets(lens).tolist()
    qkv = torch.zeros(sum(lens), 3, H, D, dtype=dtype)
    qkv[:, 1], qkv[:, 2] = s.k, s.v
    done = [0] * len(lens)
    g = torch.Generator().manual_seed(1)
    while done != lens:
        n = [min(int(torch.randint(0, 40, (), generator=g)), t - d) for t, d in zip(lens, done)]
        rows = [ends[i] + done[i] + j for i in range(len(lens)) for j in range(n[i])]
        part = qkv[rows].to(dev)
        done = [d + m for d, m in zip(done, n)]
        ops.kv4_append(other, part[:, 1], part[:, 2], ref.offsets(n).to(dev),
                       torch.tensor(done, dtype=torch.int32, device=dev), s.table)
    assert torch.equal(other.pages, s.cache.pages)


@pytest.mark.parametrize("H,D,tokens", [(9, 32, 77000), (9, 128, 19200), (3, 64, 3000),
                                        (1, 32, 5000), (2, 128, 1500)])
def test_many_sequences_of_any_lengths(cuda_device, H, D, tokens):
    """Calls large and small, with runs of empty sequences and of single tokens longer than a warp
    is wide; then the ends of the sequences alone, from odd tokens on."""
    from cti_b200 import _lib, ops

    g = torch.Generator().manual_seed(H + D)
    lens = [0] * 40 + [1] * 70 + [0] * 33 + [2, 0, 64, 129]
    while sum(lens) < tokens:
        lens.append(int(torch.randint(0, 200, (), generator=g)) if len(lens) % 5 else 0)
    lens += [0] * 35
    s = Setup(cuda_device, lens, lens, H, H, D, torch.bfloat16, seed=D)
    k, v = ops.kv4_read(s.cache, s.cu, s.lens, s.table, sum(lens))
    _check_read(k, s.k)
    _check_read(v, s.v)
    some = [n // 2 for n in lens]
    cu = ref.offsets(some)
    ends = torch.tensor(lens).cumsum(0).tolist()
    rows = torch.tensor([e - n + j for e, n in zip(ends, some) for j in range(n)])
    ks, vs = ops.kv4_read(s.cache, cu.to(cuda_device), s.lens, s.table, sum(some))
    _lib.raise_on_status(cuda_device)
    assert torch.equal(ks.cpu(), k.cpu()[rows]) and torch.equal(vs.cpu(), v.cpu()[rows])


@pytest.mark.parametrize("dtype", TYPES)
def test_values_on_and_next_to_the_borders_between_codes(cuda_device, dtype):
    """Groups whose values lie exactly on s (n + 1/2) + b (ties go to the even code) and one step of
    the type beside it, tiny values beside large ones, and groups with the smallest ranges."""
    from cti_b200 import ops

    rows = []
    for hi in (15.0, 7.5, 30.0, 0.9375, 240.0):
        x = torch.full((32,), 0.0)
        x[0], x[1] = 0.0, hi
        x[2:17] = hi / 15 * (torch.arange(15) + 0.5)
        rows.append(x)
        rows.append(-x)
        # a symmetric group: zero, and values next to it, lie near a border
        y = torch.zeros(32)
        y[0], y[1] = -hi, hi
        y[3:19] = torch.tensor([1.0, -1.0]).repeat(8) * 2.0 ** -torch.arange(0, 16).float() * 1e-2
        rows.append(y)
    x = torch.stack(rows).to(dtype)
    up = torch.nextafter(x, torch.full_like(x, float("inf"))) if dtype == torch.float32 else None
    assert up is None
    bits = x.view(torch.int16)
    near = torch.cat([x, (bits + 1).view(dtype), (bits - 1).view(dtype)])
    near = torch.where(torch.isfinite(near), near, torch.zeros_like(near))
    near[:, 0], near[:, 1] = x.repeat(3, 1)[:, 0], x.repeat(3, 1)[:, 1]
    const = torch.tensor([0.0, 1.0, -3.1415, 1e-4, 60.0]).to(dtype)[:, None].expand(5, 32)
    step = const.clone()
    step[:, 7] = (const[:, 7].contiguous().view(torch.int16) + 1).view(dtype)
    rnd = _values(400, 1, 32, dtype, 9).reshape(400, 32)
    k = torch.cat([near, const, step, rnd, rnd * 2.0 ** -12])[:, None, :]
    T = k.shape[0]
    s = Setup(cuda_device, [T], [T], 1, 1, 32, dtype, k=k, v=k.flip(0).contiguous())
    gk, gv = ops.kv4_read(s.cache, s.cu, s.lens, s.table, T)
    _check_read(gk, s.k)
    _check_read(gv, s.v)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_value_that_is_not_finite_spoils_its_group_alone(cuda_device, dtype):
    from cti_b200 import ops

    k, v = _values(70, 2, 64, dtype, 1), _values(70, 2, 64, dtype, 2)
    k[3, 0, 5], k[66, 1, 40], v[0, 1, 63] = float("nan"), float("inf"), float("-inf")
    s = Setup(cuda_device, [70], [70], 2, 2, 64, dtype, k=k, v=v)
    gk, gv = ops.kv4_read(s.cache, s.cu, s.lens, s.table, 70)
    _check_read(gk, s.k)
    _check_read(gv, s.v)
    assert int(torch.isnan(gk).sum()) == 64 and int(torch.isnan(gv).sum()) == 32


def test_positions_and_pages_outside_are_left_out_and_reported(cuda_device):
    import cti_b200
    from cti_b200 import _lib, ops

    dev, H, D = cuda_device, 2, 32
    c = cti_b200.KV4Cache(4, H, D, device=dev)
    before = c.pages.clone()
    x = _values(6, H, D, torch.bfloat16, 0).to(dev)
    one = torch.tensor([0, 6], dtype=torch.int32, device=dev)
    for table, length in (([[4, 1]], 6), ([[-1, 1]], 6), ([[0, 2]], 200), ([[0, 2]], 0)):
        t = torch.tensor(table, dtype=torch.int32, device=dev)
        lens = torch.tensor([length], dtype=torch.int32, device=dev)
        ops.kv4_append(c, x, x, one, lens, t)
        assert _lib.read_status(dev)[0] == _lib.CTI_ERR_BOUNDS
        assert torch.equal(c.pages, before)
        k, v = ops.kv4_read(c, one, lens, t, 6)
        assert _lib.read_status(dev)[0] == _lib.CTI_ERR_BOUNDS
        assert not k.any() and not v.any()
    # Only the last 4 of the 6 tokens have a position.
    t = torch.tensor([[3, 1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([4], dtype=torch.int32, device=dev)
    ops.kv4_append(c, x, x, one, lens, t)
    assert _lib.read_status(dev)[0] == _lib.CTI_ERR_BOUNDS
    k, _ = ops.kv4_read(c, torch.tensor([0, 4], dtype=torch.int32, device=dev), lens, t, 4)
    _lib.raise_on_status(dev)
    _check_read(k, x[2:].cpu())
    assert torch.equal(c.pages[:3], before[:3])


def test_rows_of_no_sequence_are_left_as_they_were(cuda_device):
    import cti_b200
    from cti_b200 import _lib, ops

    dev, H, D = cuda_device, 2, 64
    c = cti_b200.KV4Cache(4, H, D, device=dev)
    x = _values(40, H, D, torch.bfloat16, 0).to(dev)
    cu = torch.tensor([3, 10, 33], dtype=torch.int32, device=dev)
    lens = torch.tensor([7, 23], dtype=torch.int32, device=dev)
    t = torch.tensor([[2], [0]], dtype=torch.int32, device=dev)
    ops.kv4_append(c, x, x, cu, lens, t)
    k, v = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    ops.kv4_read(c, cu, lens, t, 40, out=(k, v))
    o = torch.full_like(x, 7.0)
    ops.kv4_attention(x, c, cu, lens, t, out=o)
    _lib.raise_on_status(dev)
    for y in (k, v, o):
        assert (y[:3] == 7.0).all() and (y[33:] == 7.0).all() and not (y[3:33] == 7.0).all()
    _check_read(k[3:33], x[3:33].cpu())


# ---------------------------------------------------------------------------
# Attention.
# ---------------------------------------------------------------------------
SHAPES = [(8, 8, 32), (4, 1, 32), (6, 3, 64), (4, 4, 64), (8, 2, 128), (5, 5, 128), (16, 1, 128),
          (24, 1, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_single_tokens(cuda_device, dtype, H, Hkv, D):
    total = [1, 2, 63, 64, 65, 127, 128, 129, 300, 17, 511]
    s = Setup(cuda_device, [1] * len(total), total, H, Hkv, D, dtype, seed=H + D)
    a = s.check(max_new=1)
    b = s.check(causal=False)
    assert torch.equal(a, b)  # a sequence's last token sees all of it either way


def test_more_sequences_than_warps(cuda_device):
    """A warp for a sequence's head, over up to 12 pages."""
    g = torch.Generator().manual_seed(17)
    total = [int(torch.randint(1, 740, (), generator=g)) for _ in range(240)]
    Setup(cuda_device, [1] * 240, total, 16, 16, 32, torch.bfloat16, seed=18).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_several_tokens(cuda_device, dtype, H, Hkv, D, causal):
    new = [1, 7, 0, 64, 65, 3, 130, 16, 2]
    total = [64, 7, 50, 64, 200, 129, 131, 300, 66]
    s = Setup(cuda_device, new, total, H, Hkv, D, dtype, seed=H + D)
    s.check(causal=causal, max_new=130)


@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 32), (4, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("new,total", [([500], [700]), ([257, 1, 300], [900, 1000, 300]),
                                       ([1, 1], [3000, 5]), ([5, 40], [4100, 2500])])
def test_long_sequences(cuda_device, H, Hkv, D, new, total):
    s = Setup(cuda_device, new, total, H, Hkv, D, torch.bfloat16, seed=sum(new))
    s.check()
    s.check(causal=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hkv,D,n", [(2, 2, 32, 100), (4, 2, 64, 64), (4, 1, 128, 25),
                                       (8, 1, 32, 16), (1, 1, 128, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_about_a_hundred_rows(cuda_device, dtype, H, Hkv, D, n, causal):
    """97 to 128 query rows of a KV head: one 128-row tile, of one page range or several."""
    s = Setup(cuda_device, [n, 1, n - 3], [n + 40, 1, 200], H, Hkv, D, dtype, seed=n)
    s.check(causal=causal, max_new=n)
    s = Setup(cuda_device, [n], [2500], H, Hkv, D, dtype, seed=n + 1)
    s.check(causal=causal, max_new=n)


@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 32), (4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("n", [1, 12, 60, 150])
def test_magnitudes_far_from_one(cuda_device, H, Hkv, D, n):
    """Keys and values of 1e-5 to 1e5, other ones in every page: what a page is scaled by must not
    show.  The scores' scale keeps the largest of them within a few hundred."""
    total = 400
    k, v = (_values(total, Hkv, D, torch.bfloat16, i).float() for i in (1, 2))
    size = torch.tensor([1e5, 1e-3, 1.0, 3e4, 1e-5, 40.0, 1e-4])[torch.arange(total) // 64]
    k = (k * size[:, None, None]).bfloat16()
    v = (v * size.flip(0)[:, None, None]).bfloat16()
    s = Setup(cuda_device, [n], [total], H, Hkv, D, torch.bfloat16, k=k, v=v)
    s.check(scale=1e-4, max_new=n)
    s.check(scale=-1e-4, causal=False)
    s.check(scale=4e-6, max_new=n)


def test_scale_and_large_scores(cuda_device):
    """Scores of hundreds: the running maximum keeps every exponential in range.  The scale enters
    the bound of a score's error."""
    for D in (32, 64, 128):
        s = Setup(cuda_device, [1, 40, 3], [400, 300, 64], 4, 2, D, torch.float16, seed=D)
        s.check(scale=0.0)
        s.check(scale=-0.3)
        s.check(scale=4.0)


def test_split_and_order_hints_do_not_matter(cuda_device):
    """max_new and max_kv_len are bounds that only steer how work is split."""
    s = Setup(cuda_device, [1, 9, 70, 0], [2000, 40, 1000, 10], 8, 2, 64, torch.bfloat16, seed=8)
    for max_new in (0, 1, 9, 70, 1000):
        for max_kv in (0, 1, 100, 2000, 10 ** 6, None):
            s.check(max_new=max_new, max_kv_len=max_kv)


def test_rows_that_see_nothing_are_zero(cuda_device):
    """No cached token at all, and more new tokens than the sequence has (the first ones have no
    position)."""
    import cti_b200
    from cti_b200 import _lib, ops

    dev, H, D = cuda_device, 4, 64
    c = cti_b200.KV4Cache(8, H, D, device=dev)
    c.pages.fill_(0xff)
    x = _values(140, H, D, torch.bfloat16, 0)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=dev)
    lens = torch.tensor([0, 100], dtype=torch.int32, device=dev)
    ops.kv4_append(c, x[40:].to(dev), x[40:].to(dev),
                   torch.tensor([0, 0, 100], dtype=torch.int32, device=dev), lens, table)
    for n, m in ((3, 137), (20, 120), (1, 104)):
        q = x[:n + m].to(dev)
        cu = torch.tensor([0, n, n + m], dtype=torch.int32, device=dev)
        out = ops.kv4_attention(q, c, cu, lens, table)
        _lib.raise_on_status(dev)
        assert not out[:n + m - 100].any()
        want, tol = ref.attention(x[n + m - 100:n + m], ref.held(x[40:]), ref.held(x[40:]), [100],
                                  [100], True, D ** -0.5)
        assert ((out[n + m - 100:].double().cpu() - want).abs() <= tol).all()
        out = ops.kv4_attention(q, c, cu, lens, table, causal=False)
        assert not out[:n].any() and out[n:].any(-1).all()
    empty = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    none = torch.zeros(2, dtype=torch.int32, device=dev)
    out = ops.kv4_attention(x[:5].to(dev), c, torch.tensor([0, 2, 5], dtype=torch.int32,
                                                           device=dev), none, empty)
    _lib.raise_on_status(dev)
    assert not out.any()


@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 32), (4, 1, 64), (2, 1, 128)])
@pytest.mark.parametrize("new,total", [([70], [100]), ([300], [300]), ([10, 64], [64, 190])])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(cuda_device, H, Hkv, D, new,
                                                                    total):
    T = sum(total)
    k, v = _values(T, Hkv, D, torch.bfloat16, 1), _values(T, Hkv, D, torch.bfloat16, 2)
    k[total[0] - 5, 0, 3] = float("nan")
    v[total[0] - 20 if new[0] > 20 else total[0] - 3, Hkv - 1, 7] = float("inf")
    v[T - 1, 0, 0] = float("nan")
    s = Setup(cuda_device, new, total, H, Hkv, D, torch.bfloat16, k=k, v=v)
    from cti_b200 import ops

    out = ops.kv4_attention(s.q.to(cuda_device), s.cache, s.cu, s.lens, s.table,
                            max_new=max(new))
    want, tol = ref.attention(s.q, ref.held(k), ref.held(v), new, total, True, D ** -0.5)
    got = out.double().cpu()
    # A NaN of a value may spoil its group of head dims or the whole row.
    rows = torch.isnan(want).any(-1)
    assert torch.equal(torch.isnan(got).any(-1), rows)
    assert ((got - want).abs() <= tol)[~rows].all()


def test_attention_with_bad_pages(cuda_device):
    """Keys of a page outside the cache are left out; so are keys past the table."""
    from cti_b200 import _lib, ops

    s = Setup(cuda_device, [2, 30], [150, 300], 4, 2, 64, torch.bfloat16, seed=2)
    q = s.q.to(cuda_device)
    bad = s.table.clone()
    bad[0, 1] = s.cache.num_pages
    bad[1, 0] = -5
    out = ops.kv4_attention(q, s.cache, s.cu, s.lens, bad, max_new=30)
    code, _ = _lib.read_status(cuda_device)
    assert code == _lib.CTI_ERR_BOUNDS
    k, v = ref.held(s.k), ref.held(s.v)
    keep = torch.ones(450, dtype=torch.bool)
    keep[64:128] = False
    keep[150:150 + 64] = False
    want, tol = ref.attention(s.q, k[keep], v[keep], [2, 30], [150 - 64, 300 - 64], True, 0.125)
    assert ((out.double().cpu() - want).abs() <= tol).all()
    out = ops.kv4_attention(q, s.cache, s.cu, s.lens, s.table[:, :2].contiguous(), max_new=30,
                            causal=False)
    assert _lib.read_status(cuda_device)[0] == _lib.CTI_ERR_BOUNDS
    keep = torch.zeros(450, dtype=torch.bool)
    keep[:128] = True
    keep[150:150 + 128] = True
    want, tol = ref.attention(s.q, k[keep], v[keep], [2, 30], [128, 128], False, 0.125)
    assert ((out.double().cpu() - want).abs() <= tol).all()


def test_strided_queries_tables_and_shared_pages(cuda_device):
    from cti_b200 import _lib, ops

    s = Setup(cuda_device, [3, 12, 1], [140, 80, 64], 8, 8, 32, torch.bfloat16, seed=4, extra=3)
    dev = cuda_device
    qkv = torch.zeros(16, 3, 8, 32, dtype=torch.bfloat16, device=dev)
    qkv[:, 0] = s.q.to(dev)
    wide = torch.full((3, 3, s.table.shape[1]), -1, dtype=torch.int32, device=dev)
    wide[:, 1] = s.table
    out = ops.kv4_attention(qkv[:, 0], s.cache, s.cu, s.lens, wide[:, 1], max_new=12)
    _lib.raise_on_status(dev)
    s.compare(out)
    # Two sequences on the same pages.
    table = s.table[[0, 0]].contiguous()
    lens = torch.tensor([140, 140], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    twice = ops.kv4_attention(torch.cat([qkv[:3, 0]] * 2), s.cache, cu, lens, table, max_new=3)
    assert torch.equal(twice[:3], twice[3:])
    # Another bound of the new tokens may take another variant, which sums in another order: it is
    # held to the same bound as the first call.
    s.compare(torch.cat([twice[:3], out[3:]]))


def test_results_repeat_and_survive_streams_and_graphs(cuda_device):
    """Two streams at once, and two captured graphs replayed one after the other and at once, with
    new contents in the same tensors."""
    from cti_b200 import ops

    dev = cuda_device
    a = Setup(dev, [1, 1, 4], [3000, 50, 700], 8, 2, 128, torch.bfloat16, seed=1)
    b = Setup(dev, [100, 1], [2100, 400], 8, 2, 128, torch.bfloat16, seed=2)

    def call(s):
        return ops.kv4_attention(s.q_dev, s.cache, s.cu, s.lens, s.table, max_new=max(s.new),
                                 max_kv_len=max(s.total))

    for s in (a, b):
        s.q_dev = s.q.to(dev)
        s.want = call(s)
        s.compare(s.want)
        s.stream = torch.cuda.Stream(dev)
    torch.cuda.synchronize(dev)
    got = []
    for _ in range(10):
        for s in (a, b):
            with torch.cuda.stream(s.stream):
                got.append((s, call(s)))
    torch.cuda.synchronize(dev)
    assert all(torch.equal(o, s.want) for s, o in got)
    for s in (a, b):
        s.q_dev.zero_()
        s.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s.graph, stream=s.stream):
            s.out = call(s)
        s.q_dev.copy_(s.q)
    torch.cuda.synchronize(dev)
    for _ in range(5):
        for s in (a, b):
            s.out.zero_()
            torch.cuda.synchronize(dev)
        for s in (a, b):
            with torch.cuda.stream(s.stream):
                s.graph.replay()
        torch.cuda.synchronize(dev)
        for s in (a, b):
            assert torch.equal(s.out, s.want)


def test_a_step_appends_and_attends(cuda_device):
    """Histories built one call at a time, as a server does: each call's new tokens are appended and
    attend; after the last call every output equals the attention over the history so far."""
    import cti_b200
    from cti_b200 import _lib, ops

    dev, H, Hkv, D = cuda_device, 8, 4, 64
    dtype = torch.bfloat16
    steps = [[30, 1, 0], [1, 1, 70], [0, 1, 1], [40, 64, 1], [1, 1, 1]]
    total = [sum(c) for c in zip(*steps)]
    k, v, q = (_values(sum(total), h, D, dtype, i) for i, h in enumerate((Hkv, Hkv, H)))
    c = cti_b200.KV4Cache(12, Hkv, D, dtype=dtype, device=dev)
    table = ref.page_table(total, 12).to(dev)
    first = ref.offsets(total).tolist()
    done = [0, 0, 0]
    for n in steps:
        rows = [first[i] + done[i] + j for i in range(3) for j in range(n[i])]
        done = [d + m for d, m in zip(done, n)]
        cu = ref.offsets(n).to(dev)
        lens = torch.tensor(done, dtype=torch.int32, device=dev)
        ops.kv4_append(c, k[rows].to(dev), v[rows].to(dev), cu, lens, table)
        out = ops.kv4_attention(q[rows].to(dev), c, cu, lens, table, max_new=max(n))
        _lib.raise_on_status(dev)
        held = [first[i] + j for i in range(3) for j in range(done[i])]
        want, tol = ref.attention(q[rows], ref.held(k[held]), ref.held(v[held]), n, done, True,
                                  D ** -0.5)
        assert ((out.double().cpu() - want).abs() <= tol).all()


def test_pages_past_four_gigabytes(cuda_device):
    """A cache whose bytes need more than 32 bits: the last pages hold what the first ones do."""
    import cti_b200
    from cti_b200 import _lib, ops

    dev, H, D = cuda_device, 8, 128
    pages = 2 ** 32 // _lib.lib.cti_kv4_page_bytes(H, D) + 60
    c = cti_b200.KV4Cache(pages, H, D, device=dev)
    x = _values(260, H, D, torch.bfloat16, 0).to(dev)
    lens = torch.tensor([130, 130], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 130, 260], dtype=torch.int32, device=dev)
    table = torch.tensor([[0, 1, 2], [pages - 1, pages - 3, pages - 2]], dtype=torch.int32,
                         device=dev)
    x[130:] = x[:130]
    ops.kv4_append(c, x, x, cu, lens, table)
    k, v = ops.kv4_read(c, cu, lens, table, 260)
    assert torch.equal(k[:130], k[130:]) and torch.equal(v, k)
    _check_read(k[130:], x[130:].cpu())
    for n in (1, 130):
        q = x[:n].repeat(2, 1, 1)
        out = ops.kv4_attention(q, c, torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev),
                                lens, table, n)
        _lib.raise_on_status(dev)
        assert torch.equal(out[:n], out[n:])
        want, tol = ref.attention(q[:n].cpu(), ref.held(x[:130].cpu()), ref.held(x[:130].cpu()),
                                  [n], [130], True, D ** -0.5)
        assert ((out[:n].double().cpu() - want).abs() <= tol).all()


def test_wrappers_refuse_wrong_tensors(cuda_device):
    from cti_b200 import ops

    s = Setup(cuda_device, [3], [70], 4, 2, 64, torch.bfloat16)
    dev = cuda_device
    q, k, v = s.q.to(dev), s.k.to(dev), s.v.to(dev)
    cu = torch.tensor([0, 70], dtype=torch.int32, device=dev)

    def attend(q=q, cu=s.cu, lens=s.lens, table=s.table, **kw):
        return ops.kv4_attention(q, s.cache, cu, lens, table, **kw)

    for call in (lambda: attend(q.half()), lambda: attend(s.q), lambda: attend(cu=s.cu.long()),
                 lambda: attend(lens=s.lens.float()), lambda: attend(table=s.table.long()),
                 lambda: ops.kv4_append(s.cache, k.half(), v, cu, s.lens, s.table)):
        with pytest.raises((TypeError, RuntimeError)):
            call()
    for call in (lambda: attend(q[:, :3]), lambda: attend(q[..., :32]),
                 lambda: attend(q.transpose(1, 2)), lambda: attend(cu=cu[:1]),
                 lambda: attend(table=s.table[:0]), lambda: attend(table=s.table[0]),
                 lambda: attend(table=torch.cat([s.table] * 2, 1)[:, ::2]),
                 lambda: attend(lens=s.lens[None]), lambda: attend(out=q[:2]),
                 lambda: ops.kv4_append(s.cache, k, v[:5], cu, s.lens, s.table),
                 lambda: ops.kv4_append(s.cache, q, v, cu, s.lens, s.table),
                 lambda: ops.kv4_read(s.cache, cu, s.lens, s.table, 70, out=(k[:5], v)),
                 lambda: ops.kv4_read(s.cache, cu, s.lens, s.table, -1)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: attend(max_new=-1), lambda: attend(scale=float("nan"))):
        with pytest.raises(RuntimeError):
            call()
