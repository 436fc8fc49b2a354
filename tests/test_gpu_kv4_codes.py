"""Codes of the 4-bit cache where fp32 rounds a value onto a border between two of them."""
import pytest
import torch

import kv4_borders as borders
import kv4_ref as ref
from test_gpu_kv4 import TYPES, Setup, _check_read

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_values_that_fp32_rounds_onto_a_border(cuda_device, dtype, D):
    from cti_b200 import ops

    x = borders.groups(dtype, 4096, seed=D)
    x = torch.cat([x, -x]).reshape(-1, 1, D)
    # The other order of dims, so that each lane of a group sees each kind.
    x = torch.cat([x, x.flip(-1)])
    a = (x.unflatten(-1, (-1, 32)).float() - ref.quantise(x)[2].float()).double()
    n, s, _ = ref.quantise(x)
    assert (((torch.round(a / s) - 16).clamp(0, 15) != n).sum() > 4096)  # fp32 alone is not enough
    T = x.shape[0]
    t = Setup(cuda_device, [T], [T], 1, 1, D, dtype, k=x, v=x.flip(0).contiguous())
    k, v = ops.kv4_read(t.cache, t.cu, t.lens, t.table, T)
    _check_read(k, t.k)
    _check_read(v, t.v)


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_many_ordinary_values(cuda_device, dtype):
    """20 million values: what is rare happens."""
    from cti_b200 import ops
    import cti_b200

    dev, H, D, T = cuda_device, 8, 128, 64 * 160
    cache = cti_b200.KV4Cache(160, H, D, dtype=dtype, device=dev)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    lens = torch.tensor([T], dtype=torch.int32, device=dev)
    table = torch.arange(160, dtype=torch.int32, device=dev)[None]
    for seed in range(2):
        g = torch.Generator(device=dev).manual_seed(seed)
        x = torch.randn(2, T, H, D, generator=g, device=dev)
        x = (x * torch.exp(0.5 * torch.randn(1, 1, H, D, generator=g, device=dev))).to(dtype)
        ops.kv4_append(cache, x[0], x[1], cu, lens, table)
        for got, y in zip(ops.kv4_read(cache, cu, lens, table, T), x):
            n, s, b = ref.quantise(y)
            step = (got.double().unflatten(-1, (-1, 32)) - ((16 + n) * s + b)).abs() / s
            assert step.max() < 0.25, int((step >= 0.25).sum())
