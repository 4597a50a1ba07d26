"""Sizes at the ends of their types: what the cache operators refuse before they touch a device
(this runs without a GPU)."""
import pytest

from test_cache_ops_host import _accept, _attend, _kv_read, _rope_append


@pytest.mark.parametrize("bad", [
    dict(n_heads=1 << 26),                                         # times 64 dims: 2^32, which is 0 in 32 bits
    dict(n_heads=(1 << 26) + 4),
    dict(cache=dict(n_kv_heads=1 << 26)), dict(cache=dict(n_kv_heads=(1 << 26) + 1))])
def test_rope_append_refuses_heads_beyond_the_rows(sb, bad):
    with pytest.raises(RuntimeError, match="rope_append: bad arguments"):
        _rope_append(sb, **bad)


@pytest.mark.parametrize("call", [_rope_append, _kv_read, _attend, _accept])
@pytest.mark.parametrize("pages", [(1 << 26) + 1, (1 << 27) - 1])
def test_tables_whose_tokens_come_near_32_bits_are_refused(sb, call, pages):
    """A context, its 64 nodes and the tiles looked ahead have to stay within an int."""
    with pytest.raises(RuntimeError, match="bad cache descriptor"):
        call(sb, cache=dict(max_pages=pages))


def test_kv_read_refuses_products_beyond_64_bits(sb):
    n = 0x7fffffff
    with pytest.raises(RuntimeError, match="too many"):
        _kv_read(sb, cache=dict(n_layers=n, n_kv_heads=n), n_layers=n, rows=n)
