"""Pages of the 4-bit KV cache on the GPU: who is served when there are too few, and page tables in any order."""
import numpy as np
import pytest
import torch

from oracle import kv4 as okv
from test_gpu_kv4 import DT, check, ints, make, many_rows, num, rows, same, starts_of, status

pytestmark = pytest.mark.gpu


def starts_list(n):
    return np.concatenate([[0], np.cumsum(n)]).tolist()


def test_extend_serves_whoever_fits(cuda_lib):
    """One sequence that needs more than there is does not take the pages from those behind it."""
    kv = make(1, 1, 32, n_pages=5, max_seqs=4, max_pages=12, page=16)
    assert kv.extend([0, 1, 2, 3], starts_list([160, 1, 80, 60])).tolist() == [-1, 0, -1, 0]
    assert kv.lens.tolist() == [0, 1, 0, 60] and kv.refs.tolist() == [1] * 5 and kv.tables[3].tolist()[:4] == [1, 2, 3, 4]
    assert kv.extend([0, 1, 3], starts_list([160, 15, 4])).tolist() == [-1, 1, 60] and kv.lens.tolist() == [0, 16, 0, 64]
    assert status() == 0                                     # none of this is an error


@pytest.mark.parametrize("seqs,n_pages", [(40, 70), (1500, 2000), (2500, 300)])
def test_extend_with_too_few_pages(cuda_lib, seqs, n_pages):
    """Against the restated pool: shared last pages (copies) among the needs, refusals at every place of the batch."""
    rng = np.random.default_rng(seqs)
    most, page = 6, 16
    kv, model = make(1, 1, 32, n_pages=n_pages, max_seqs=seqs, max_pages=most, page=page), okv.Pool(n_pages, seqs, most, page)
    kv.pages.random_(0, 256)
    served = refused = 0
    for _ in range(6):
        slots = rng.permutation(seqs)[:int(seqs * 0.9)].tolist()
        n = rng.choice([0, 1, 2, 5, 16, 40, 70, 90], len(slots)).tolist()
        before = kv.pages.clone()
        pos = kv.extend(slots, starts_list(n)).tolist()
        want, copies = model.extend(slots, n)
        assert pos == want
        for a, b in copies:
            before[b] = before[a]
        assert torch.equal(before, kv.pages)
        same(kv, model)
        short = [b for b, p in enumerate(pos) if p < 0]
        refused += len(short)
        served += sum(1 for b, p in enumerate(pos) if p >= 0 and n[b] and short and b > short[0])
        kv.free(slots[:len(slots) // 3]), model.free(slots[:len(slots) // 3])
        src, dst = rng.permutation(seqs)[:20].tolist(), rng.permutation(seqs)[:20].tolist()
        kv.fork(src, dst), model.fork(src, dst)
        same(kv, model)
    assert served and refused                                # behind the first refusal
    status()


def test_extend_of_ranges_that_overlap(cuda_lib):
    """The caller's mistake, and far more pages than there are: nothing is given out."""
    kv = make(1, 1, 32, n_pages=64, max_seqs=64, max_pages=1 << 20, page=16)
    big = (1 << 24) - 16
    starts = [0 if i % 2 == 0 else big for i in range(65)]   # rows: big, -big, big, ...
    pos = kv.extend(list(range(64)), starts).tolist()
    assert pos == [-1] * 64 and kv.refs.sum().item() == 0 and kv.lens.sum().item() == 0 and status() == -1


def scatter(kv, rng):
    """Every page moves to another place of the pool; the sequences' tables follow."""
    perm = torch.from_numpy(rng.permutation(kv.n_pages)).cuda()
    pages, refs = kv.pages.clone(), kv.refs.clone()
    kv.pages[perm], kv.refs[perm] = pages, refs
    kv.tables.copy_(torch.where(kv.tables >= 0, perm[kv.tables.clamp(min=0).long()].int(), -1))
    steps = (kv.tables[:, 1:] - kv.tables[:, :-1])[kv.tables[:, 1:] >= 0]
    assert (steps != 1).float().mean() > 0.5 and (steps < 0).any()      # no consecutive, no ascending rows


def filled(kv, layer, lens, rng, dtype):
    """Sequences of these lengths in two calls with the pages moved after each -> what the cache holds of each."""
    first = [n // 2 for n in lens]
    K, V = [[] for _ in lens], [[] for _ in lens]
    for new in (first, [n - m for n, m in zip(lens, first)]):
        starts = starts_of(new)
        k, v = (rows(rng, sum(new), kv.kv_heads, kv.head_dim, dtype) for _ in range(2))
        kv.append(layer, k, v, None, kv.extend(None, starts), starts)
        scatter(kv, rng)
        at = np.concatenate([[0], np.cumsum(new)])
        k, v = okv.held(num(k)), okv.held(num(v))
        for b in range(len(lens)):
            K[b].append(k[at[b]:at[b + 1]]), V[b].append(v[at[b]:at[b + 1]])
    return [(np.concatenate(k), np.concatenate(v)) for k, v in zip(K, V)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Hkv,rep,page", [(32, 2, 4, 16), (64, 1, 1, 16), (64, 2, 8, 32), (96, 2, 3, 16), (128, 1, 1, 16), (128, 2, 4, 32), (160, 1, 2, 16),
                                            (192, 1, 1, 32), (224, 1, 6, 16), (256, 2, 1, 32), (256, 1, 8, 16)])
def test_attention_over_pages_in_any_order(cuda_lib, D, Hkv, rep, page, dtype):
    """One token per sequence, then chunks, then everything read back, over tables whose entries are in no order."""
    rng = np.random.default_rng(D + page)
    lens = [300, 1, 17, 129, 64, 333]
    kv = make(2, Hkv, D, n_pages=90, max_seqs=6, max_pages=24, page=page)
    kv.pages.random_(0, 256)
    data = filled(kv, 1, lens, rng, dtype)
    check(kv, 1, data, lens, [1] * len(lens), Hkv * rep, dtype, rng)
    check(kv, 1, data, lens, [20, 1, 0, 33, 64, 7], Hkv * rep, dtype, rng)
    k, v = kv.gather(1, None, ints([0] * len(lens)), starts_of(lens), rows=sum(lens))
    assert np.array_equal(num(k), np.concatenate([d[0] for d in data]).astype(np.float32))
    assert np.array_equal(num(v), np.concatenate([d[1] for d in data]).astype(np.float32))


@pytest.mark.parametrize("D,Hkv,rep,page", [(64, 8, 3, 16), (128, 4, 4, 32), (128, 1, 16, 16), (256, 2, 8, 16), (256, 8, 2, 32)])
def test_many_rows_over_pages_in_any_order(cuda_lib, D, Hkv, rep, page):
    rng = np.random.default_rng(D + rep)
    lens, new = [333, 70, 260, 5, 64, 129], [140, 70, 1, 0, 64, 128]
    kv = make(2, Hkv, D, n_pages=90, max_seqs=6, max_pages=24, page=page)
    assert many_rows(kv, Hkv * rep, len(lens), sum(new))
    kv.pages.random_(0, 256)
    check(kv, 0, filled(kv, 0, lens, rng, "bf16"), lens, new, Hkv * rep, "bf16", rng)


@pytest.mark.parametrize("D,rep,dtype", [(128, 8, "bf16"), (256, 1, "f32")])
def test_long_context_over_pages_in_any_order(cuda_lib, D, rep, dtype):
    """Positions of one sequence that are split over the machine and joined."""
    rng = np.random.default_rng(D)
    lens = [9011, 4097]
    kv = make(1, 1, D, n_pages=500, max_seqs=2, max_pages=300, page=32)
    check(kv, 0, filled(kv, 0, lens, rng, dtype), lens, [1, 1], rep, dtype, rng)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rotated_rows_into_pages_in_any_order(cuda_lib, dtype):
    """rope_append over scattered pages writes what it writes over consecutive ones."""
    rng = np.random.default_rng(8)
    Hq, Hkv, D, before, new = 4, 2, 128, [30, 7, 50], [40, 1, 25]
    got = []
    for move in (False, True):
        kv = make(1, Hkv, D, n_pages=40, max_seqs=3, max_pages=8, page=16)
        kv.pages.zero_()
        kv.extend(None, starts_of(before))
        if move:
            scatter(kv, np.random.default_rng(1))
        starts = starts_of(new)
        pos = kv.extend(None, starts)
        qkv = torch.randn((sum(new), (Hq + 2 * Hkv) * D), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
        q = kv.rope_append(0, qkv, Hq, 1e4, None, pos, starts, dtype=DT[dtype])
        got.append((q, *kv.gather(0, None, pos, starts, rows=sum(new))))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and status() == 0
