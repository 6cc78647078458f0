"""Paged 4-bit KV cache without a GPU: the restatement of its layout and bookkeeping, and refusals before any launch."""
import ctypes as C

import numpy as np
import pytest

from oracle import kv4 as okv


@pytest.mark.parametrize("D", [32, 96, 256])
def test_every_nibble_has_a_place_of_its_own(D):
    for values in (False, True):
        places = {okv.code_place(r, d, values) for r in range(16) for d in range(D)}
        assert len(places) == 16 * D and max(b for b, _ in places) == 8 * D - 1
        # the nibbles of one position fill whole bytes
        for r in range(16):
            mine = [okv.code_place(r, d, values) for d in range(D)]
            assert {b for b, h in mine if h} == {b for b, h in mine if not h}


def test_restated_values_are_the_weight_quantisers_but_for_the_last_bit_of_a_scale():
    from chadslab_b200 import packing
    x = np.random.default_rng(0).normal(0, 1, (500, 64)).astype(np.float32)
    codes, scales = packing.quantize(x, packing.FMT_Q4)
    mine, s = okv.quantise(x)
    agree = s == scales
    assert agree.mean() > 0.99 and np.max(np.abs(s.view(np.int16).astype(int) - scales.view(np.int16))) <= 1
    same = np.repeat(agree, 32, axis=1)
    assert np.array_equal(mine[same], packing.unpack_nibbles(codes)[same])
    assert len(okv.block_bytes(np.zeros((16, 64), np.float32), np.zeros((16, 64), np.float32))) == 576 * 2


def test_restated_attention_of_one_position_is_its_value():
    rng = np.random.default_rng(1)
    q, K, V = rng.normal(size=(1, 4, 32)), rng.normal(size=(1, 2, 32)), rng.normal(size=(1, 2, 32))
    o, mag, _ = okv.attention(q, K, V, 0)
    assert np.allclose(o[0], np.repeat(V[0], 2, axis=0)) and np.allclose(mag, np.abs(o))


def test_restated_pool_shares_and_copies():
    p = okv.Pool(6, 4, 3, 16)
    assert p.extend([0], [20]) == ([0], [])
    p.fork([0, 0], [1, 2])
    assert p.refs.tolist() == [3, 3, 0, 0, 0, 0]
    assert p.extend([1, 2], [1, 0]) == ([20, 20], [(1, 2)])             # only the one that writes copies
    assert p.refs.tolist() == [3, 2, 1, 0, 0, 0] and p.tables[1].tolist() == [0, 2, -1]
    p.free([0, 0, 2])
    assert p.refs.tolist() == [1, 0, 1, 0, 0, 0]
    to, old = p.compact(2)
    assert old.tolist() == [0, 2] and to.tables[1].tolist() == [0, 1, -1] and to.lens.tolist() == [0, 21, 0, 0]


def pool(**kw):
    from chadslab_b200 import _lib
    f = dict(n_pages=4, max_seqs=4, max_pages=4, layers=2, kv_heads=2, head_dim=64, page=16)
    f.update(kw)
    return _lib.Kv4Pool(16, 16, 16, 16, 16, *f.values())


def test_sizes(built_lib):
    p = pool()
    assert built_lib.bq_kv4_page_bytes(C.byref(p)) == 2 * 2 * 1 * 576 * 2
    assert built_lib.bq_kv4_work_bytes(C.byref(p)) >= 4 * (4 + 4 + 8 + 4 * 5)
    assert built_lib.bq_kv4_page_bytes(None) == 0


def test_calls_need_the_library_to_be_bound(built_lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("state test is for the GPU-less container")
    p = C.byref(pool())
    assert built_lib.bq_kv4_extend(p, None, None, 1, None, None) == -4
    assert built_lib.bq_kv4_append(p, 0, None, None, 128, 128, 0, None, None, None, 1, 1, None) == -4
    assert built_lib.bq_kv4_attention(p, 0, None, 128, None, 2, 0, None, None, None, 1, 1, None, None) == -4
    assert built_lib.bq_kv4_free(p, None, 1, None) == -4 and built_lib.bq_kv4_fork(p, None, None, 1, None) == -4


@pytest.mark.parametrize("bad", [dict(head_dim=48), dict(head_dim=288), dict(head_dim=0), dict(page=24), dict(page=8), dict(layers=0),
                                 dict(n_pages=0), dict(max_seqs=9000), dict(max_pages=1 << 27), dict(kv_heads=0)])
def test_python_refuses_bad_pools(bad):
    from chadslab_b200 import PagedKV4
    f = dict(n_pages=4, max_seqs=4, max_pages=4, layers=2, kv_heads=2, head_dim=64, page=16)
    f.update(bad)
    with pytest.raises(ValueError):
        PagedKV4(f["layers"], f["kv_heads"], f["head_dim"], n_pages=f["n_pages"], max_seqs=f["max_seqs"], max_pages=f["max_pages"],
                 page=f["page"], device="cuda:0")


def test_python_refuses_host_tensors():
    import torch
    import chadslab_b200 as cb
    t = torch.zeros((4, 4), dtype=torch.int32)
    with pytest.raises(cb.BqError):
        cb.PagedKV4(1, 1, 64, pages=torch.zeros(4 * 1152, dtype=torch.uint8), tables=t, lens=t[0], refs=t[0], page=16)
    with pytest.raises(ValueError):
        cb.PagedKV4(1, 1, 64, tables=t)
    with pytest.raises(cb.BqError):
        cb.PagedKV4(1, 1, 64, n_pages=4, max_seqs=4, max_pages=4, device="cpu")
