"""The workspace of attention over the 4-bit cache: what the splits of long sequences may ask for
(host only)."""
import pytest

LIMIT = 64 << 20


def _bytes(*sizes):
    from cti_b200 import _lib

    return _lib.lib.cti_kv4_attention_workspace_bytes(*sizes)


@pytest.mark.parametrize("num_seqs,tokens,max_new,max_kv_len,heads,kv_heads,head_dim", [
    (2048, 2048, 1, 131072, 32, 8, 128), (512, 8192, 16, 32768, 32, 8, 128),
    (1024, 8192, 8, 131072, 32, 8, 128), (2048, 2048, 1, 2048 * 64, 8, 8, 32),
    (1, 2 ** 20, 1, 2 ** 31 - 64, 8, 1, 128), (3, 10 ** 6, 2 ** 30, 2 ** 31 - 64, 16, 2, 64),
    (200000, 200000, 1, 10 ** 6, 8, 8, 32)])
def test_workspace_is_limited(num_seqs, tokens, max_new, max_kv_len, heads, kv_heads, head_dim):
    """Whatever the bounds: a table that is wide for one sequence, or for none."""
    assert _bytes(num_seqs, tokens, max_new, max_kv_len, heads, kv_heads, head_dim) <= LIMIT


def test_long_sequences_are_still_split():
    """One sequence, and a few, take what they need to fill the GPU."""
    for n, heads, kv_heads, head_dim in ((1, 32, 8, 128), (48, 32, 8, 128), (4, 8, 8, 32)):
        assert 0 < _bytes(n, n, 1, 131072, heads, kv_heads, head_dim) <= LIMIT
    assert _bytes(1, 256, 256, 131072, 32, 8, 128) > 0
    assert _bytes(2048, 2048, 1, 100, 8, 8, 32) == 0


def test_bounds_past_any_table_are_as_good_as_the_widest():
    """A table holds 2^31 keys of a sequence at most."""
    for sizes in ((1, 1, 1), (3, 300, 100), (48, 48, 1)):
        widest = _bytes(*sizes, 2 ** 31 - 1, 32, 8, 128)
        for bound in (2 ** 31, 2 ** 37 + 64, 2 ** 40, 2 ** 62, 2 ** 63 - 1):
            assert _bytes(*sizes, bound, 32, 8, 128) == widest
