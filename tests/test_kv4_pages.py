"""That the values of kv4_pages show each page that attention may lose (host only)."""
import pytest
import torch

import kv4_pages as pages


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("new,total", pages.CALLS)
def test_a_lost_page_is_outside_the_tolerance(dtype, D, new, total):
    v = pages.values(total, 1, D, dtype)
    out, tol = pages.expected(v, 1, new, total, False)
    last = 0
    for i, L in enumerate(total):
        rows = slice(last, last + new[i])
        last += new[i]
        for p in range(0, -(-L // 64), 1 if L < 1500 else 7):
            less, _ = pages.expected(v, 1, new, total, False, (i, p))
            off = ((less - out).abs() - tol)[rows]
            assert (off.amax(-1) > 0).all(), (i, p)
