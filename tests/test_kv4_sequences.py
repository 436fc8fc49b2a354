"""SequenceCache's undo: an extension whose forward did not run leaves no trace (host only)."""
import pytest
import torch


def _cache(pages=12, seqs=5, tokens=300, layers=2):
    import cti_b200

    return cti_b200.SequenceCache(layers, seqs, pages, 2, 32, tokens, device="cpu")


def _state(c):
    return (c.free_pages, [c.length(i) for i in range(c.max_seqs)])


def _same(a, b):
    return all(torch.equal(a[n], b[n]) for n in ("cu_seqlens", "kv_lens", "page_table"))


def test_undo_restores_lengths_and_pages():
    c, twin = _cache(), _cache()
    for x in (c, twin):
        x.extend([1, 3], [70, 64])
        x.release([3])
        x.extend([0], [10])
    before = _state(c)
    e = c.extend([3, 1, 0], [129, 58, 0])
    assert _state(c) != before
    c.undo(e)
    assert _state(c) == before
    # A second try gets what the first one got, and what a cache gets that saw no first one.
    f, g = c.extend([3, 1, 0], [129, 58, 0]), twin.extend([3, 1, 0], [129, 58, 0])
    assert _same(e, f) and _same(f, g) and _state(c) == _state(twin)


def test_undo_of_several_extensions_from_the_last_back():
    c = _cache()
    start = _state(c)
    a = c.extend([0, 2], [100, 3])
    middle = _state(c)
    b = c.extend([2, 0], [200, 1])
    with pytest.raises(ValueError):
        c.undo(a)  # not the last one of its sequences
    c.undo(b)
    assert _state(c) == middle
    c.undo(a)
    assert _state(c) == start
    for e in (a, b):
        with pytest.raises(ValueError):
            c.undo(e)  # once
    assert _state(c) == start


def test_undo_refuses_what_it_cannot_take_back():
    c = _cache()
    e = c.extend([0], [65])
    c.release([0])
    state = _state(c)
    with pytest.raises(ValueError):
        c.undo(e)
    with pytest.raises(ValueError):
        _cache().undo(c.extend([1], [1]))
    c.release([1])
    assert _state(c) == state
    # A sequence that was released and has grown to the same length is another one.
    e = c.extend([0], [65])
    c.release([0])
    c.extend([0], [65])
    with pytest.raises(ValueError):
        c.undo(e)
    assert c.length(0) == 65


def test_extension_tells_how_many_tokens_it_holds():
    assert _cache().extend([1, 0], [5, 7])["tokens"] == 12
