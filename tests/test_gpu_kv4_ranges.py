"""Attention over the paged 4-bit KV cache where its operands leave the middle of fp16's range, against 64 bits."""
import numpy as np
import pytest
import torch

from oracle import kv4 as okv
from test_gpu_kv4 import DT, ints, make, many_rows, num, rows, starts_of, status

pytestmark = pytest.mark.gpu


def limit(o, mag, size, V, dtype):
    """Per element.  What is lost of small weights and products shrinks with the values.  The largest weight is held as 2^11 or
    more, the largest value scale as 1/16 or more (2^-15 of it where the scales are below that).  bf16 rows: a weight loses up to
    half a step of the smallest fp16, 2^-25, which is 2^-36 of the largest weight, times a value; its product with a scale the
    same 2^-25 times a code of at most 7: 2^-25 / 2^11 * 16 * (7 times the largest scale) = 2^-32 of the largest value.  fp32
    rows hold both in two halves, the second of them 2^-11 of the first.  The rest as for values around one: roundings to
    fp16 (twice, 2^-11 each), exponents and sums in fp32 (2^-20), scores (their sum of |q k| times 2^-22 and 16 additions of
    2^-24, for subnormal keys 2^-18, numerator and denominator)."""
    most = np.abs(V).max()
    score = 2.0 * size * (2.0 ** -22 + 16 * 2.0 ** (-24 if dtype == "f32" else -18))
    lost = len(V) * (2.0 ** -36 * most + max(2.0 ** -32 * most, 7 * 2.0 ** -51))
    if dtype == "f32":
        return (2.0 ** -20 + score) * mag + lost * 2.0 ** -11
    return ((2 * 2.0 ** -11 + 2.0 ** -20 + score) * mag + lost) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(o)


def put(kv, ks, vs, dtype):
    """Sequences with the given keys and values [len, heads, D] (numpy) -> what the cache holds of each, in 64 bits."""
    lens = [len(k) for k in ks]
    starts = starts_of(lens)
    k, v = (torch.from_numpy(np.concatenate(x).astype(np.float32)).cuda().to(DT[dtype]) for x in (ks, vs))
    kv.append(0, k, v, None, kv.extend(None, starts), starts)
    at = np.concatenate([[0], np.cumsum(lens)])
    K, V = okv.held(num(k)), okv.held(num(v))
    return [(K[at[b]:at[b + 1]], V[at[b]:at[b + 1]]) for b in range(len(lens))]


def compare(kv, data, q, new, dtype):
    lens = [len(k) for k, _ in data]
    pos = [n - m for n, m in zip(lens, new)]
    out = num(kv.attention(0, q, None, ints(pos), None if all(m == 1 for m in new) else starts_of(new)))
    at = np.concatenate([[0], np.cumsum(new)])
    for b, (K, V) in enumerate(data):
        one = slice(at[b], at[b + 1])
        o, mag, size = okv.attention(num(q)[one], K, V, pos[b])
        err, tol = np.abs(out[one] - o), limit(o, mag, size, V, dtype)
        assert (err <= tol).all(), f"sequence {b}: {np.nanmax(err / tol):.3g} x the bound, {np.abs(out[one] - o).max() / np.abs(o).max():.3g} relative"
    assert status() == 0


SHAPES = [("f32", 64, 1, 1, 1), ("f32", 128, 2, 2, 1), ("f32", 256, 1, 8, 3), ("bf16", 64, 1, 1, 1), ("bf16", 64, 1, 2, 1), ("bf16", 96, 2, 2, 1),
          ("bf16", 128, 1, 4, 1), ("bf16", 128, 1, 8, 5), ("bf16", 256, 2, 1, 1), ("bf16", 256, 1, 8, 1), ("bf16", 64, 24, 2, 60),
          ("bf16", 128, 24, 2, 60), ("bf16", 256, 24, 2, 60)]


def pool(dtype, D, Hkv, rep, rows_each, seqs=2):
    kv = make(1, Hkv, D, n_pages=64, max_pages=24, page=32)
    assert many_rows(kv, Hkv * rep, seqs, seqs * rows_each) == (rows_each == 60)
    return kv


@pytest.mark.parametrize("vscale", [1.0, 1e-2, 1e-3, 1e-4, 1e-6])
@pytest.mark.parametrize("nats", [15, 18])
@pytest.mark.parametrize("dtype,D,Hkv,rep,rows_each", SHAPES)
def test_small_values_below_a_position_without_any(cuda_lib, dtype, D, Hkv, rep, rows_each, nats, vscale):
    """Every sixteenth position takes nearly all the weight and has the value zero: the output is what is left of the others."""
    rng = np.random.default_rng(nats)
    kv = pool(dtype, D, Hkv, rep, rows_each)
    b = np.sign(rng.normal(size=D))
    ks, vs = [], []
    for n in (75, 200):
        k, v = rng.normal(0, 0.05, (n, Hkv, D)), rng.normal(0, vscale, (n, Hkv, D))
        k[5::16], v[5::16] = b * nats / np.sqrt(D), 0.0
        ks.append(k), vs.append(v)
    data = put(kv, ks, vs, dtype)
    q = torch.from_numpy((b + rng.normal(0, 0.05, (2 * rows_each, Hkv * rep, D))).astype(np.float32)).cuda().to(DT[dtype])
    compare(kv, data, q, [rows_each] * 2, dtype)


@pytest.mark.parametrize("order", ["rising", "falling", "mixed", "one large"])
@pytest.mark.parametrize("dtype,D,Hkv,rep,rows_each", SHAPES)
def test_values_of_many_magnitudes(cuda_lib, dtype, D, Hkv, rep, rows_each, order):
    """From 1e-6 to 1e5 within a sequence: the range that products are held in follows the largest one so far."""
    rng = np.random.default_rng(3)
    kv = pool(dtype, D, Hkv, rep, rows_each)
    ks, vs = [], []
    for n in (130, 333):
        e = np.linspace(-6, 5, n)
        e = {"rising": e, "falling": e[::-1], "mixed": rng.permutation(e), "one large": np.where(np.arange(n) == n - 20, 3.0, -4.0)}[order]
        ks.append(rng.normal(0, 1, (n, Hkv, D))), vs.append(rng.normal(0, 1, (n, Hkv, D)) * 10.0 ** e[:, None, None])
    data = put(kv, ks, vs, dtype)
    compare(kv, data, rows(rng, 2 * rows_each, Hkv * rep, D, dtype, 1.5), [rows_each] * 2, dtype)


@pytest.mark.parametrize("size", [1e4, 1e7, 1e9, 1e12, 1e20, 1e30, 1e35])
@pytest.mark.parametrize("dtype,D,Hkv,rep,rows_each", SHAPES)
def test_queries_of_any_size(cuda_lib, dtype, D, Hkv, rep, rows_each, size):
    """Scores up to 1e37, one position far above the others: its value.  Its weight is rounded to fp16 alone and times the scale
    (2^-11 each) in bf16 calls, and the result to bf16 (2^-8); fp32 calls hold 22 bits of both and add in fp32 (2^-20)."""
    rng = np.random.default_rng(7)
    kv = pool(dtype, D, Hkv, rep, rows_each)
    b = np.sign(rng.normal(size=D))
    ks, vs, at = [], [], (3, 77)
    for n, w in zip((75, 333), at):
        ks.append(rng.normal(0, 0.05, (n, Hkv, D))), vs.append(rng.normal(0, 1, (n, Hkv, D)))
        ks[-1][w] = 2.0 * b
    data = put(kv, ks, vs, dtype)
    q = b * rng.uniform(0.5, 1.0, (2 * rows_each, Hkv * rep, D)) * size
    q = torch.from_numpy(q.astype(np.float32)).cuda().to(DT[dtype])
    out = num(kv.attention(0, q, None, ints([75 - rows_each, 333 - rows_each]), None if rows_each == 1 else starts_of([rows_each] * 2)))
    for s in range(2):
        want = np.repeat(data[s][1][at[s]], rep, axis=0)
        err = np.abs(out[s * rows_each:(s + 1) * rows_each] - want)
        assert (err <= (2.0 ** -20 if dtype == "f32" else 2 * 2.0 ** -11 + 2.0 ** -20 + 2.0 ** -8) * np.abs(want)).all(), err.max()
    assert status() == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype,D,Hkv,rep,rows_each", SHAPES)
def test_rows_that_are_not_finite_keep_to_themselves(cuda_lib, dtype, D, Hkv, rep, rows_each, bad):
    """A query row with a NaN or an infinity gives NaN; every other row has the bits that it has without it.  A value that is NaN
    shows in its group of 32 dimensions only, in the rows that see it."""
    rng = np.random.default_rng(9)
    kv = pool(dtype, D, Hkv, rep, rows_each)
    ks, vs = ([rng.normal(0, 1, (n, Hkv, D)) for n in (75, 200)] for _ in range(2))
    put(kv, ks, vs, dtype)
    pos, starts = ints([75 - rows_each, 200 - rows_each]), None if rows_each == 1 else starts_of([rows_each] * 2)
    q = rows(rng, 2 * rows_each, Hkv * rep, D, dtype)
    ref = kv.attention(0, q, None, pos, starts)
    hit, head = rows_each - 1, Hkv * rep - 1
    broken = q.clone()
    broken[hit, head, 5] = bad
    out = kv.attention(0, broken, None, pos, starts)
    keep = torch.ones(ref.shape[:2], dtype=torch.bool, device="cuda")
    keep[hit, head] = False
    assert torch.isnan(out[hit, head]).all() and torch.equal(out[keep], ref[keep]) and torch.isfinite(ref).all()
    # sequence 0's last position: its value becomes NaN in one group of head 0
    k, v = (torch.from_numpy(x[0][-1:].astype(np.float32)).cuda() for x in (ks, vs))
    v[0, 0, 3] = float("nan")
    kv.append(0, k.to(DT[dtype]), v.to(DT[dtype]), [0], [74])
    out = kv.attention(0, q, None, pos, starts)
    sees = torch.zeros_like(out, dtype=torch.bool)
    sees[hit, :rep, :32] = True                              # only the last row of sequence 0 sees position 74
    assert torch.isnan(out[sees]).all() and torch.isfinite(out[~sees]).all() and status() == 0


@pytest.mark.parametrize("dtype,D,Hkv,rep,rows_each", SHAPES)
def test_bytes_behind_small_values_do_not_matter(cuda_lib, dtype, D, Hkv, rep, rows_each):
    """The rest of a last block can hold anything, also where the scales in front of it are raised."""
    got = []
    for fill_with in (0, 0x7C00, 0x7E00, 0x7BFF, -0x8000 + 0x7C00, -1):
        rng = np.random.default_rng(21)
        kv = pool(dtype, D, Hkv, rep, rows_each)
        kv.pages.view(torch.int16).fill_(fill_with)
        data = put(kv, [rng.normal(0, 1, (n, Hkv, D)) for n in (61, 131)], [rng.normal(0, 1e-3, (n, Hkv, D)) for n in (61, 131)], dtype)
        q = rows(rng, 2 * rows_each, Hkv * rep, D, dtype)
        got.append(kv.attention(0, q, None, ints([61 - rows_each, 131 - rows_each]), None if rows_each == 1 else starts_of([rows_each] * 2)))
        assert torch.equal(got[-1], got[0])
    compare(kv, data, q, [rows_each] * 2, dtype)


@pytest.mark.parametrize("vscale", [1e-1, 1e-3])
@pytest.mark.parametrize("dtype,D,Hkv,rep", [("bf16", 64, 1, 2), ("bf16", 128, 1, 8), ("bf16", 256, 2, 1), ("bf16", 96, 1, 3), ("f32", 128, 1, 2)])
def test_small_values_over_long_and_short_contexts(cuda_lib, dtype, D, Hkv, rep, vscale):
    """Segments that are cut and joined, whose pieces raise their scales by different powers of two; and sequences of a few positions."""
    rng = np.random.default_rng(D)
    kv = make(1, Hkv, D, n_pages=300, max_seqs=6, max_pages=160, page=64)
    lens = [9001, 1, 2, 16, 17, 4000]
    vs = [rng.normal(0, vscale, (n, Hkv, D)) * np.where(np.arange(n) > n // 2, 1.0, 0.03)[:, None, None] for n in lens]
    data = put(kv, [rng.normal(0, 1, (n, Hkv, D)) for n in lens], vs, dtype)
    compare(kv, data, rows(rng, len(lens), Hkv * rep, D, dtype, 1.5), [1] * len(lens), dtype)
