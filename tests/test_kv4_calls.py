"""Paged 4-bit KV cache without a GPU: what the restated pool serves, and what the Python surface does before it calls."""
import pytest
import torch

from oracle import kv4 as okv


class Recorder:
    """In place of the library: every call succeeds and is kept."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


def surface(seqs=4):
    """A PagedKV4 whose tensors lie on the CPU and whose calls go to a Recorder."""
    from chadslab_b200 import PagedKV4
    kv = object.__new__(PagedKV4)
    kv.layers, kv.kv_heads, kv.head_dim, kv.page, kv.n_pages, kv.max_seqs, kv.max_pages = 1, 2, 64, 16, 8, seqs, 4
    kv.device, kv._index, kv._lib, kv._pool, kv._p, kv._attn_ints = torch.device("cpu"), 0, Recorder(), None, None, {}
    kv.changes = 0
    kv.lens, kv.refs = torch.zeros(seqs, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)
    kv._stream = lambda: 0
    return kv


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_restated_pool_serves_whoever_fits():
    p = okv.Pool(5, 4, 12, 16)
    assert p.extend([0, 1, 2, 3], [160, 1, 80, 60]) == ([-1, 0, -1, 0], [])
    assert p.tables[1].tolist()[:2] == [0, -1] and p.tables[3].tolist()[:5] == [1, 2, 3, 4, -1] and p.refs.tolist() == [1] * 5
    p.fork([1, 3], [0, 2])
    p.free([1])
    # page 0 is not shared any more; the copy of page 4 that sequences 2 and 3 want does not exist
    assert p.extend([0, 2, 3], [3, 1, 4]) == ([1, -1, -1], [])


def test_gather_of_ranges_needs_their_rows():
    kv = surface()
    with pytest.raises(ValueError):
        kv.gather(0, i32(0, 1), i32(0, 0), i32(0, 3, 5))
    assert not kv._lib.calls
    k, v = kv.gather(0, i32(0, 1), i32(0, 0), i32(0, 3, 5), rows=5)
    assert k.shape == v.shape == (5, 2, 64) and kv._lib.calls[-1][1][9] == 5
    assert kv.gather(0, i32(0, 1), i32(0, 0), i32(0, 0, 0), rows=0)[0].shape == (0, 2, 64)
    assert kv.gather(0, i32(0, 1), i32(0, 0))[0].shape == (2, 2, 64)


def test_extend_needs_to_know_the_batch():
    kv = surface()
    with pytest.raises(ValueError):
        kv.extend()
    with pytest.raises(ValueError):
        kv.extend(None, i32())
    assert not kv._lib.calls
    assert kv.extend(batch=3).shape == (3,) and kv.extend(i32(1, 2)).shape == (2,) and kv.extend(None, i32(0, 4)).shape == (1,)
    assert [c[1][3] for c in kv._lib.calls] == [3, 2, 1] and kv.extend(batch=0).shape == (0,)


def test_scratch_sizes_do_not_pile_up():
    kv = surface()
    for n in range(2000):
        kv.attention(0, torch.zeros((n, 2, 64)), i32(0), i32(0), i32(0, n))
    assert len(kv._attn_ints) <= 256 and sum(name == "bq_kv4_attention" for name, _ in kv._lib.calls) == 2000
    kv._lib.calls.clear()
    for _ in range(10):                                      # a size that repeats is asked for once
        kv.attention(0, torch.zeros((7, 2, 64)), i32(0), i32(0), i32(0, 7))
    assert sum(name == "bq_kv4_attention_work_bytes" for name, _ in kv._lib.calls) <= 1


def test_rope_append_names_a_type_it_does_not_have():
    kv = surface()
    with pytest.raises(TypeError):
        kv.rope_append(0, torch.zeros((2, 8 * 64)), 4, 1e4, None, i32(0, 0), dtype=torch.float16)
    assert not kv._lib.calls
