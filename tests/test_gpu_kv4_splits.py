"""How attention over the 4-bit cache is shared among warps and blocks: each page counts once and
wholly, whatever the split; nothing of the workspace is used that the call did not write; rows of
a sequence that is refused are left as they were."""
import pytest
import torch

import kv4_pages as pages
from test_gpu_kv4 import Setup

pytestmark = pytest.mark.gpu

SHAPES = [(2, 2, 32), (4, 2, 64), (4, 1, 128)]


def _call(s, q, cu, lens, table, max_new, max_kv_len, fill, out=None, splits=True, causal=1):
    """The C entry point with a workspace of `fill` bytes."""
    from cti_b200 import _lib, ops

    T, H, D = q.shape
    c = s.cache
    n = lens.numel()
    need = _lib.lib.cti_kv4_attention_workspace_bytes(n, T, max_new, max_kv_len, H, c.kv_heads, D)
    assert (need > 0) == splits
    ws = torch.full((max(need, 256),), fill, dtype=torch.uint8, device=q.device)
    out = torch.full_like(q, 7.0) if out is None else out
    rc = _lib.lib.cti_kv4_attention(
        q.data_ptr(), H * D, c.dtype_code, cu.data_ptr(), lens.data_ptr(), table.data_ptr(),
        table.stride(0), table.shape[1], n, T, max_new, max_kv_len, H, c.kv_heads, D, D ** -0.5,
        causal, c.pages.data_ptr(), c.num_pages, out.data_ptr(), ws.data_ptr(), need,
        _lib.status_word(q.device).data_ptr(), torch.cuda.current_stream(q.device).cuda_stream)
    assert rc == _lib.CTI_OK
    assert ops.PAGE_TOKENS == 64
    return out


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
@pytest.mark.parametrize("n", [1, 9, 140])
@pytest.mark.parametrize("fill", [0x3f, 0xff])
def test_rows_of_a_refused_sequence_are_left_as_they_were(cuda_device, H, Hkv, D, n, fill):
    """Offsets that pass the tokens, or start before them, with split sequences."""
    from cti_b200 import _lib

    dev = cuda_device
    s = Setup(dev, [n, n], [4000, 4000], H, Hkv, D, torch.bfloat16, seed=n)
    q = s.q.to(dev)
    max_kv = 4000
    good = _call(s, q, s.cu, s.lens, s.table, n, max_kv, fill)
    _lib.raise_on_status(dev)
    s.compare(good)
    for cu, kept in (([0, n, 2 * n + 5], slice(n, 2 * n)), ([-3, n, 2 * n], slice(0, n))):
        cu = torch.tensor(cu, dtype=torch.int32, device=dev)
        out = _call(s, q, cu, s.lens, s.table, n, max_kv, fill)
        assert _lib.read_status(dev)[0] == _lib.CTI_ERR_INVALID_ARG
        assert (out[kept] == 7.0).all()
        other = slice(0, n) if kept.start else slice(n, 2 * n)
        assert torch.equal(out[other], good[other])


@pytest.mark.parametrize("H,Hkv,D", [(32, 8, 128), (8, 8, 32)])
@pytest.mark.parametrize("n", [1, 8])
def test_one_long_history_among_many_short_ones(cuda_device, H, Hkv, D, n):
    """A bound that one sequence needs, and a table as wide: most splits have no pages, and the
    workspace holds NaN where they would be."""
    from cti_b200 import _lib

    total = [9000] + [n + i % 90 for i in range(40)]
    s = Setup(cuda_device, [n] * len(total), total, H, Hkv, D, torch.bfloat16, seed=D)
    out = _call(s, s.q.to(cuda_device), s.cu, s.lens, s.table, n, 9000, 0xff)
    _lib.raise_on_status(cuda_device)
    s.compare(out)
    need = _lib.lib.cti_kv4_attention_workspace_bytes(len(total), sum(s.new), n, 9000, H, Hkv, D)
    assert need <= 64 << 20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 32), (4, 2, 64), (4, 1, 128), (4, 4, 128)])
@pytest.mark.parametrize("new,total", pages.CALLS)
def test_every_page_counts_once(cuda_device, dtype, H, Hkv, D, new, total):
    """Whatever the bounds say of the work: no split, splits of other sizes, tiles or not."""
    from cti_b200 import _lib, ops

    s = Setup(cuda_device, new, total, H, Hkv, D, dtype, v=pages.values(total, Hkv, D, dtype))
    q = s.q.to(cuda_device)
    for causal in (True, False):
        want, tol = pages.expected(s.v, H, new, total, causal)
        for max_new in (max(new), 1, 200):
            for max_kv_len in (None, max(total), 64, 100000):
                out = ops.kv4_attention(q, s.cache, s.cu, s.lens, s.table, max_new, causal, 0.0,
                                        max_kv_len)
                off = ((out.double().cpu() - want).abs() / tol).max()
                assert off <= 1, (causal, max_new, max_kv_len, float(off))
    _lib.raise_on_status(cuda_device)


def test_every_page_counts_once_with_a_warp_for_each(cuda_device):
    """More heads of sequences than warps, up to 12 pages each."""
    from cti_b200 import _lib, ops

    total = [1 + 37 * i % 760 for i in range(450)]
    new = [1] * len(total)
    v = pages.values(total, 8, 32, torch.bfloat16)
    s = Setup(cuda_device, new, total, 8, 8, 32, torch.bfloat16, v=v)
    out = ops.kv4_attention(s.q.to(cuda_device), s.cache, s.cu, s.lens, s.table, 1, scale=0.0)
    _lib.raise_on_status(cuda_device)
    want, tol = pages.expected(v, 8, new, total, True)
    assert ((out.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 32), (4, 1, 128)])
@pytest.mark.parametrize("n", [1, 9, 140])
def test_bounds_far_past_any_table(cuda_device, H, Hkv, D, n):
    """max_kv_len and max_new only steer how work is split, also where a split's pages would pass
    32 bits."""
    from cti_b200 import _lib, ops

    s = Setup(cuda_device, [n, 2], [3000, 70], H, Hkv, D, torch.bfloat16,
              v=pages.values([3000, 70], Hkv, D, torch.bfloat16))
    q = s.q.to(cuda_device)
    want, tol = pages.expected(s.v, H, s.new, s.total, True)
    for max_new in (n, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
        for max_kv_len in (2 ** 31, 2 ** 37 + 64, 2 ** 40, 2 ** 45 - 1, 2 ** 62, 2 ** 63 - 1, 2 ** 80):
            out = ops.kv4_attention(q, s.cache, s.cu, s.lens, s.table, max_new, True, 0.0,
                                    max_kv_len)
            assert ((out.double().cpu() - want).abs() <= tol).all()
    _lib.raise_on_status(cuda_device)
    out = _call(s, q, s.cu, s.lens, s.table, 2 ** 31 - 1, 2 ** 63 - 1, 0xff)
    _lib.raise_on_status(cuda_device)
    s.compare(out, causal=True)
