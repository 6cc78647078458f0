"""Entry points of the 4-bit KV cache: calls that are refused, and what the Python surface does with its arguments."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import kv4 as okv
from test_gpu_kv4 import fill, ints, make, num, rows, starts_of, status

pytestmark = pytest.mark.gpu


def test_addresses_between_elements_are_refused(cuda_lib):
    """Every pointer that the kernels read or write elements through; nothing is launched."""
    from chadslab_b200 import _lib
    kv = make(1, 2, 64, n_pages=8, max_seqs=4)
    lib, p, s = _lib.lib(), kv._p, torch.cuda.current_stream().cuda_stream
    x, i = torch.zeros(4096, device="cuda").data_ptr(), ints(range(16)).data_ptr()
    n0 = lib.bq_launch_count()
    bad = []
    for slots, pos, starts in ((i + 2, i, i), (i, i + 1, i), (i, i, i + 2)):
        bad += [lib.bq_kv4_append(p, 0, x, x, 128, 128, 0, slots, pos, starts, 2, 2, s),
                lib.bq_kv4_gather(p, 0, x, x, 0, slots, pos, starts, 2, 2, s),
                lib.bq_kv4_rope_append(p, 0, x, x, 4, 1e4, 0, slots, pos, starts, 2, 2, s),
                lib.bq_kv4_attention(p, 0, x, 256, x, 4, 0, slots, pos, starts, 2, 2, x, s),
                lib.bq_kv4_extend(p, slots, starts, 2, pos, s)]
    bad += [lib.bq_kv4_gather(p, 0, x + 2, x, 0, i, i, i, 2, 2, s), lib.bq_kv4_gather(p, 0, x, x + 1, 1, i, i, i, 2, 2, s),
            lib.bq_kv4_rope_append(p, 0, x + 2, x, 4, 1e4, 0, i, i, i, 2, 2, s), lib.bq_kv4_rope_append(p, 0, x, x + 2, 4, 1e4, 0, i, i, i, 2, 2, s),
            lib.bq_kv4_rope_append(p, 0, x, x + 1, 4, 1e4, 1, i, i, i, 2, 2, s), lib.bq_kv4_rope_append(p, 0, x, x, 1 << 18, 1e4, 0, i, i, i, 2, 2, s),
            lib.bq_kv4_fork(p, i + 2, i, 1, s), lib.bq_kv4_fork(p, i, i + 2, 1, s), lib.bq_kv4_free(p, i + 1, 1, s)]
    for field in ("tables", "lens"):
        q = _lib.Kv4Pool.from_buffer_copy(kv._pool)
        setattr(q, field, getattr(q, field) + 2)
        bad.append(lib.bq_kv4_free(C.byref(q), i, 1, s))
    assert bad == [-1] * len(bad) and lib.bq_launch_count() == n0
    assert status() == 0
