"""Pages of the 4-bit KV cache on the GPU: who is served when there are too few, and page tables in any order."""
import numpy as np
import pytest
import torch

from oracle import kv4 as okv
from test_gpu_kv4 import make, same, status

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
