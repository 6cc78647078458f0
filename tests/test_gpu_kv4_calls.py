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


def test_ints_do_not_make_the_host_wait(cuda_lib):
    kv = make(1, 2, 64, max_seqs=4)
    q = torch.zeros((1, 2, 64), device="cuda")
    calls = [lambda: kv.extend([0], [0, 1]), lambda: kv.attention(0, q, [0], [0]), lambda: kv.append(0, q, q, [0], [0]), lambda: kv.gather(0, [0], [0]),
             lambda: kv.fork([0], range(1, 2)), lambda: kv.free([1])]
    torch.cuda._sleep(20_000_000)
    for call in calls * 2:                                   # the allocators have seen these sizes, this many at a time
        call()
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)                           # about 0.2 s of the stream
    done = torch.cuda.Event()
    done.record()
    for call in calls:
        call()
    assert not done.query()
    torch.cuda.synchronize()
    assert kv.lens.tolist() == [3, 0, 0, 0] and status() == 0


def test_ints_are_refused_during_capture(cuda_lib):
    """... before anything is issued: the capture goes on and the graph replays."""
    import chadslab_b200 as cb
    kv = make(1, 2, 64, max_seqs=4)
    q, slots, starts = torch.ones((1, 2, 64), device="cuda"), ints([1]), ints([0, 1])
    at = kv.extend(slots)
    kv.append(0, q, q, slots, at)
    kv.attention(0, q, slots, at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: kv.extend([1]), lambda: kv.extend(slots, [0, 1]), lambda: kv.attention(0, q, [1], at), lambda: kv.attention(0, q, slots, [0]),
                     lambda: kv.append(0, q, q, slots, at, [0, 1]), lambda: kv.free(range(1)), lambda: kv.fork([1], slots)):
            with pytest.raises(cb.BqError):
                call()
        at = kv.extend(slots, starts)
        kv.append(0, q, q, slots, at, starts)
        out = kv.attention(0, q, slots, at, starts)
    for _ in range(3):
        graph.replay()
    assert kv.lens.tolist() == [0, 4, 0, 0] and at.tolist() == [3] and status() == 0
    assert np.allclose(num(out), okv.held(np.ones((1, 2, 64), np.float32)), rtol=1e-5)


def test_decoder_refuses_positions_that_the_pages_do_not_have(cuda_lib):
    """Rows go behind what a sequence holds; a pass at another position would rotate them wrongly without a word."""
    from chadslab_b200.decoder import DecoderConfig, MoEDecoder, QuantDecoder
    from oracle import model as omodel
    from test_gpu_decoder_kv4 import MOE_SMALL, SMALL
    cfg = dict(SMALL, fmt=1)
    w = omodel.random_weights(cfg, seed=5)
    dec = QuantDecoder.from_numpy(DecoderConfig(**cfg), w, act_dtype=torch.float32, max_seq=48, max_batch=3, kv_bits=4, kv_page=16)
    prompt = torch.from_numpy(np.random.default_rng(1).integers(0, cfg["vocab"], (3, 9))).cuda()

    def refused(tokens):
        before = [t.clone() for t in (dec.kv.lens, dec.kv.refs, dec.kv.tables, dec.kv.pages)]
        with pytest.raises(ValueError):
            dec.hidden_states(tokens)
        assert all(torch.equal(a, b) for a, b in zip(before, (dec.kv.lens, dec.kv.refs, dec.kv.tables, dec.kv.pages)))

    dec.hidden_states(prompt[:1])
    refused(prompt)                                          # sequences 1 and 2 are empty
    dec.share_prefix(3)
    want = dec.logits(prompt[:, :2])
    dec.pos -= 1                                             # a position once more
    refused(prompt[:, :1])
    dec.pos += 1
    dec.hidden_states(prompt[:2, :1])
    refused(prompt[:, :1])                                   # sequence 2 stayed behind
    dec.kv.free([1])
    refused(prompt[:2, :1])                                  # gone behind the decoder's back
    dec.reset()
    dec.hidden_states(prompt[:1])
    dec.share_prefix(3)
    assert torch.equal(dec.logits(prompt[:, :2]), want)
    # a captured step moves the sequences on, and eager passes go on from there
    eager = dec.next_tokens(prompt[:, 2:3])
    dec.reset()
    dec.hidden_states(prompt[:, :5])
    step, tokens = dec.make_graph_stepper(3, prompt[:, 5], start_pos=5)
    step()
    step()
    assert dec.logits(tokens[:, None]).shape[0] == 3 and dec.kv.lens.tolist() == [8] * 3 and eager.shape == (3,)
    refused(torch.zeros((3, 48), dtype=torch.int64, device="cuda"))
    moe = MoEDecoder.from_numpy(DecoderConfig(**MOE_SMALL), omodel.random_weights(MOE_SMALL, seed=11), act_dtype=torch.float32, max_seq=32, max_batch=2,
                                kv_bits=4, kv_page=16)
    moe.prefill(prompt[:2, :5] % MOE_SMALL["vocab"], 1)
    moe.pos = 3
    with pytest.raises(ValueError):
        moe.hidden_states(prompt[:2, :1] % MOE_SMALL["vocab"])
    assert status() == 0
