"""Decoders on the paged 4-bit KV cache: against the numpy decoder oracle that keeps the same values, the captured step
against the eager path, shared prefixes."""
import numpy as np
import pytest

from oracle import model as omodel
from oracle import spec

pytestmark = pytest.mark.gpu
SMALL = dict(layers=2, hidden=256, n_heads=4, n_kv_heads=1, head_dim=64, ffn=512, vocab=1024)
MOE_SMALL = dict(layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=0, vocab=1024, fmt=1, n_experts=8, top_k=2,
                 moe_ffn=256)


@pytest.mark.parametrize("fmt", [0, 1])
def test_decoder_logits_and_greedy_tokens(cuda_lib, fmt):
    """The bound of the dense-cache test: the oracle keeps the same 4-bit values, so only the arithmetic differs."""
    import torch
    from chadslab_b200.decoder import DecoderConfig, QuantDecoder
    cfg = dict(SMALL, fmt=fmt)
    w = omodel.random_weights(cfg, seed=3)
    prompt = np.random.default_rng(0).integers(0, cfg["vocab"], 21)
    ref_tokens, ref_logits = omodel.OracleDecoder(cfg, w, kv_bits=4).generate(list(prompt), 4)
    dec = QuantDecoder.from_numpy(DecoderConfig(**cfg), w, act_dtype=torch.float32, max_seq=64, kv_bits=4, kv_page=16)
    pt = torch.from_numpy(prompt)[None].cuda()
    lg = dec.logits(pt)[0, -1].cpu().numpy()
    assert spec.rel_err(lg, ref_logits[0]) <= 1e-3
    toks, tok = [], int(np.argmax(lg))
    for i in range(4):
        toks.append(tok)
        lg = dec.logits(torch.tensor([[tok]], device="cuda"))[0, -1].cpu().numpy()
        assert spec.rel_err(lg, ref_logits[i + 1]) <= 1e-3
        tok = int(np.argmax(lg))
    assert toks == ref_tokens
    dec.reset()
    assert dec.kv.refs.sum().item() == 0
    assert dec.generate(pt, 4)[0].cpu().numpy().tolist() == ref_tokens
    with pytest.raises(ValueError):
        dec.hidden_states(torch.zeros((1, 64), dtype=torch.int64, device="cuda"))
    assert cuda_lib.bq_status_poll() == 0


@pytest.mark.parametrize("which", ["dense", "moe"])
def test_captured_step_equals_eager(cuda_lib, which):
    import torch
    from chadslab_b200.decoder import DecoderConfig, MoEDecoder, QuantDecoder
    cfg = dict(SMALL, fmt=1) if which == "dense" else dict(MOE_SMALL)
    w = omodel.random_weights(cfg, seed=11)
    cls = QuantDecoder if which == "dense" else MoEDecoder
    dec = cls.from_numpy(DecoderConfig(**cfg), w, act_dtype=torch.float32, max_seq=48, max_batch=3, kv_bits=4, kv_page=16)
    prompt = torch.from_numpy(np.random.default_rng(6).integers(0, cfg["vocab"], (2, 13))).cuda()
    eager = dec.generate(prompt, 8).cpu().numpy()
    dec.reset()
    first = dec.next_tokens(prompt)
    with pytest.raises(ValueError):
        dec.make_graph_stepper(2, first, start_pos=dec.pos - 1)
    step, tokens = dec.make_graph_stepper(2, first, start_pos=dec.pos)
    got = [first.cpu().numpy()]
    for _ in range(7):                               # crosses a page
        step()
        got.append(tokens.cpu().numpy().copy())
    assert np.array_equal(np.stack(got, axis=1), eager)
    assert dec.kv.lens.tolist() == [20, 20, 0] and cuda_lib.bq_status_poll() == 0


def test_prefill_in_chunks_of_sequences(cuda_lib):
    import torch
    from chadslab_b200.decoder import DecoderConfig, MoEDecoder
    w = omodel.random_weights(MOE_SMALL, seed=11)
    dec = MoEDecoder.from_numpy(DecoderConfig(**MOE_SMALL), w, act_dtype=torch.float32, max_seq=32, max_batch=2, kv_bits=4, kv_page=16)
    prompt = torch.from_numpy(np.random.default_rng(6).integers(0, MOE_SMALL["vocab"], (2, 5))).cuda()
    first = dec.next_tokens(prompt).cpu().numpy()
    dec.reset()
    assert np.array_equal(dec.prefill(prompt, 1).cpu().numpy(), first) and dec.kv.lens.tolist() == [5, 5]


def test_shared_prefix(cuda_lib):
    """One prompt, three continuations: the same logits as the oracle that runs each of them alone."""
    import torch
    from chadslab_b200.decoder import DecoderConfig, QuantDecoder
    cfg = dict(SMALL, fmt=1)
    w = omodel.random_weights(cfg, seed=5)
    rng = np.random.default_rng(1)
    prompt, more = rng.integers(0, cfg["vocab"], 22), rng.integers(0, cfg["vocab"], (3, 4))
    dec = QuantDecoder.from_numpy(DecoderConfig(**cfg), w, act_dtype=torch.float32, max_seq=32, max_batch=3, kv_bits=4, kv_page=16)
    dec.hidden_states(torch.from_numpy(prompt)[None].cuda())
    dec.share_prefix(3)
    assert dec.kv.refs.sum().item() == 6 and (dec.kv.refs > 0).sum().item() == 2
    lg = dec.logits(torch.from_numpy(more).cuda()).cpu().numpy()           # a chunk behind shared context
    tok = torch.from_numpy(np.argmax(lg[:, -1], -1))[:, None].cuda()
    nxt = dec.logits(tok).cpu().numpy()
    for b in range(3):
        ref = omodel.OracleDecoder(cfg, w, kv_bits=4)
        ref.forward(list(prompt))
        want = ref.forward(list(more[b]))
        assert spec.rel_err(lg[b], want) <= 1e-3
        assert spec.rel_err(nxt[b, 0], ref.forward([int(np.argmax(want[-1]))])[-1]) <= 1e-3
    dense = QuantDecoder.from_numpy(DecoderConfig(**cfg), w, act_dtype=torch.float32, max_seq=32, max_batch=3)
    with pytest.raises(ValueError):
        dense.share_prefix(2)
    with pytest.raises(ValueError):
        dec.share_prefix(4)
    with pytest.raises(ValueError):
        QuantDecoder.from_numpy(DecoderConfig(**cfg), w, kv_bits=8)
    assert cuda_lib.bq_status_poll() == 0
