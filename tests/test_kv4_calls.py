"""Paged 4-bit KV cache without a GPU: what the restated pool serves."""
from oracle import kv4 as okv


def test_restated_pool_serves_whoever_fits():
    p = okv.Pool(5, 4, 12, 16)
    assert p.extend([0, 1, 2, 3], [160, 1, 80, 60]) == ([-1, 0, -1, 0], [])
    assert p.tables[1].tolist()[:2] == [0, -1] and p.tables[3].tolist()[:5] == [1, 2, 3, 4, -1] and p.refs.tolist() == [1] * 5
    p.fork([1, 3], [0, 2])
    p.free([1])
    # page 0 is not shared any more; the copy of page 4 that sequences 2 and 3 want does not exist
    assert p.extend([0, 2, 3], [3, 1, 4]) == ([1, -1, -1], [])
