"""The 4-bit key/value cache without a GPU: refusals of its entry points before they touch the
device, and the format's arithmetic on the CPU."""
import pytest
import torch

import kv4_ref as ref

P = 1 << 20  # a 16-byte aligned address that is never read


def _append(lib, **kw):
    a = dict(k=P, v=P, ks=256, vs=256, dtype=1, cu=P, lens=P, table=P, stride=4, cols=4, n=2,
             tokens=8, heads=8, hd=32, pages=P, num_pages=8)
    a.update(kw)
    return lib.cti_kv4_append(a["k"], a["v"], a["ks"], a["vs"], a["dtype"], a["cu"], a["lens"],
                              a["table"], a["stride"], a["cols"], a["n"], a["tokens"], a["heads"],
                              a["hd"], a["pages"], a["num_pages"], None, None)


def _read(lib, **kw):
    a = dict(k=P, v=P, ks=256, vs=256, dtype=1, cu=P, lens=P, table=P, stride=4, cols=4, n=2,
             tokens=8, heads=8, hd=32, pages=P, num_pages=8)
    a.update(kw)
    return lib.cti_kv4_read(a["pages"], a["num_pages"], a["dtype"], a["cu"], a["lens"],
                            a["table"], a["stride"], a["cols"], a["n"], a["tokens"], a["heads"],
                            a["hd"], a["k"], a["v"], a["ks"], a["vs"], None, None)


def _attend(lib, **kw):
    a = dict(q=P, qs=256, dtype=1, cu=P, lens=P, table=P, stride=4, cols=4, n=2, tokens=8,
             max_new=1, max_kv=100, heads=8, kv_heads=8, hd=32, scale=0.1, causal=1, pages=P,
             num_pages=8, out=P, ws=None, ws_bytes=0)
    a.update(kw)
    return lib.cti_kv4_attention(a["q"], a["qs"], a["dtype"], a["cu"], a["lens"], a["table"],
                                 a["stride"], a["cols"], a["n"], a["tokens"], a["max_new"],
                                 a["max_kv"], a["heads"], a["kv_heads"], a["hd"], a["scale"],
                                 a["causal"], a["pages"], a["num_pages"], a["out"], a["ws"],
                                 a["ws_bytes"], None, None)


BAD_ARGS = [dict(n=-1), dict(tokens=-1), dict(num_pages=-1), dict(cols=-1), dict(stride=3),
            dict(pages=None), dict(cu=None), dict(lens=None), dict(table=None), dict(pages=P + 8)]


@pytest.mark.parametrize("kw", BAD_ARGS + [dict(k=None), dict(v=None), dict(k=P + 2),
                                           dict(v=P + 8), dict(ks=255), dict(vs=248),
                                           dict(heads=0)])
def test_write_and_read_refuse_bad_arguments(kw):
    from cti_b200 import _lib

    assert _append(_lib.lib, **kw) == _lib.CTI_ERR_INVALID_ARG
    assert _read(_lib.lib, **kw) == _lib.CTI_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", BAD_ARGS + [dict(q=None), dict(out=None), dict(q=P + 2),
                                           dict(out=P + 4), dict(qs=252), dict(qs=128),
                                           dict(heads=0), dict(heads=9), dict(kv_heads=0),
                                           dict(max_new=-1), dict(max_kv=-1),
                                           dict(scale=float("nan")), dict(scale=float("inf"))])
def test_attention_refuses_bad_arguments(kw):
    from cti_b200 import _lib

    assert _attend(_lib.lib, **kw) == _lib.CTI_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(dtype=0), dict(dtype=7), dict(hd=16), dict(hd=96),
                                dict(hd=256), dict(tokens=2 ** 31)])
def test_shapes_and_types_outside_the_kernels(kw):
    from cti_b200 import _lib

    for call in (_append, _read, _attend):
        assert call(_lib.lib, **kw) == _lib.CTI_ERR_UNSUPPORTED


def test_token_strides_past_the_kernels_offsets():
    from cti_b200 import _lib

    for call in (_append, _read):
        for kw in (dict(ks=2 ** 24 + 8), dict(vs=2 ** 24 + 8)):
            assert call(_lib.lib, **kw) == _lib.CTI_ERR_UNSUPPORTED


def test_nothing_to_do_is_no_error():
    from cti_b200 import _lib

    for call in (_append, _read, _attend):
        assert call(_lib.lib, tokens=0) == _lib.CTI_OK
        assert call(_lib.lib, n=0) == _lib.CTI_OK


def test_page_bytes():
    from cti_b200 import _lib

    f = _lib.lib.cti_kv4_page_bytes
    assert [f(1, 32), f(8, 64), f(3, 128)] == [2560, 8 * 5120, 3 * 10240]
    assert [f(0, 32), f(8, 48), f(-1, 64)] == [0, 0, 0]


def test_attention_workspace_must_hold_what_the_query_says():
    from cti_b200 import _lib

    need = _lib.lib.cti_kv4_attention_workspace_bytes(1, 1, 1, 200000, 32, 8, 128)
    kw = dict(n=1, tokens=1, max_kv=200000, heads=32, kv_heads=8, hd=128, qs=4096)
    if need:
        assert need % 256 == 0
        assert _attend(_lib.lib, **kw) == _lib.CTI_ERR_INVALID_ARG
        assert _attend(_lib.lib, ws=P, ws_bytes=need - 1, **kw) == _lib.CTI_ERR_INVALID_ARG
        assert _attend(_lib.lib, ws=P + 16, ws_bytes=need, **kw) == _lib.CTI_ERR_INVALID_ARG
    assert _lib.lib.cti_kv4_attention_workspace_bytes(0, 0, 1, 100, 8, 8, 32) == 0


def test_cache_refuses_what_it_cannot_hold():
    import cti_b200

    with pytest.raises(TypeError):
        cti_b200.KV4Cache(4, 8, 32, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError):
        cti_b200.KV4Cache(0, 8, 32, device="cpu")
    for heads, hd in ((8, 48), (0, 32), (8, 256)):
        with pytest.raises(RuntimeError):
            cti_b200.KV4Cache(4, heads, hd, device="cpu")


def test_wrappers_refuse_tensors_that_are_not_on_the_gpu():
    import cti_b200
    from cti_b200 import ops

    c = cti_b200.KV4Cache(4, 2, 32, device="cpu")
    x = torch.zeros(3, 2, 32, dtype=torch.bfloat16)
    cu, lens = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: ops.kv4_append(c, x, x, cu, lens, table),
                 lambda: ops.kv4_read(c, cu, lens, table, 3),
                 lambda: ops.kv4_attention(x, c, cu, lens, table)):
        with pytest.raises((RuntimeError, TypeError)):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_format_is_within_half_a_step(dtype):
    """The formula itself: a value is off by at most half a step, plus the base's rounding and the
    top code's shortfall from the scale's rounding."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(500, 4, 64, generator=g) * torch.exp(torch.randn(4, 64, generator=g))).to(dtype)
    n, s, b = ref.quantise(x)
    off = (ref.held(x).unflatten(-1, (-1, 32)) - x.double().unflatten(-1, (-1, 32))).abs()
    e = ref.rounding(dtype)
    # base: e |b|; scale: 15 s (1 + e) may fall short of max - min by 15 e s
    assert (off <= 0.5 * s + e * b.abs() + 16 * e * s).all()
    assert n.min() >= 0 and n.max() <= 15


# ---------------------------------------------------------------------------
# SequenceCache: which sequence holds which pages (host only).
# ---------------------------------------------------------------------------
def _sequence_cache(pages=6, seqs=4, tokens=300):
    import cti_b200

    return cti_b200.SequenceCache(2, seqs, pages, 2, 32, tokens, device="cpu")


def test_sequence_cache_gives_pages_as_sequences_grow():
    c = _sequence_cache()
    e = c.extend([2, 0], [64, 1])
    assert e["cu_seqlens"].tolist() == [0, 64, 65] and e["kv_lens"].tolist() == [64, 1]
    assert e["page_table"].shape == (2, 1) and e["max_seqlen"] == 64 and e["max_kv_len"] == 64
    assert e["cache"] is c and c.free_pages == 4 and (c.length(2), c.length(0)) == (64, 1)
    f = c.extend([0, 2, 1], [63, 1, 0])
    assert f["kv_lens"].tolist() == [64, 65, 0] and f["cu_seqlens"].tolist() == [0, 63, 64, 64]
    t = f["page_table"]
    assert t.shape == (3, 2) and t[0, 0] == e["page_table"][1, 0] and t[0, 1] == -1
    assert t[1, 0] == e["page_table"][0, 0] and t[1, 1] >= 0 and t[2].tolist() == [-1, -1]
    used = [p for p in t.flatten().tolist() if p >= 0]
    assert len(set(used)) == len(used) == 3 and c.free_pages == 3
    c.release([2])
    assert c.free_pages == 5 and c.length(2) == 0
    assert c.extend([], [])["kv_lens"].numel() == 0


def test_sequence_cache_refuses_and_then_changes_nothing():
    c = _sequence_cache()
    c.extend([0, 1], [65, 64])
    state = (c.free_pages, [c.length(i) for i in range(4)])
    for error, seqs, new in ((RuntimeError, [2, 3], [128, 65]), (ValueError, [0], [236]),
                             (ValueError, [0, 0], [1, 1]), (IndexError, [4], [1]),
                             (IndexError, [-1], [1]), (ValueError, [0, 1], [1]),
                             (ValueError, [2], [-1])):
        with pytest.raises(error):
            c.extend(seqs, new)
        assert (c.free_pages, [c.length(i) for i in range(4)]) == state
    c.extend([2], [192])
    assert c.free_pages == 0
    with pytest.raises(RuntimeError):
        c.extend([3], [1])
    for bad in ([4], [0, 0]):
        with pytest.raises((IndexError, ValueError)):
            c.release(bad)
    import cti_b200

    with pytest.raises(ValueError):
        cti_b200.SequenceCache(0, 4, 4, 2, 32, 100, device="cpu")
