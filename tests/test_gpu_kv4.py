"""Paged 4-bit KV cache on the GPU: rows in and out bit for bit, page bookkeeping against a restatement, attention against
64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import kv4 as okv

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def starts_of(rows):
    return ints(np.concatenate([[0], np.cumsum(rows)]))


def make(layers=1, heads=1, D=64, n_pages=32, max_seqs=8, max_pages=16, page=16):
    from chadslab_b200 import PagedKV4
    return PagedKV4(layers, heads, D, n_pages=n_pages, max_seqs=max_seqs, max_pages=max_pages, page=page)


def rows(rng, n, heads, D, dtype, scale=1.0):
    x = torch.from_numpy(rng.normal(0, scale, (n, heads, D)).astype(np.float32)).cuda().to(DT[dtype])
    return x


def num(t):
    return t.float().cpu().numpy()


def status():
    from chadslab_b200 import _lib
    return _lib.lib().bq_status_poll()


def fill(kv, layer, lens, rng, dtype="bf16", vscale=1.0):
    """Sequences 0 .. len(lens) - 1 of the given lengths, in one call -> what the cache holds of each, in 64 bits."""
    starts = starts_of(lens)
    k, v = rows(rng, sum(lens), kv.kv_heads, kv.head_dim, dtype), rows(rng, sum(lens), kv.kv_heads, kv.head_dim, dtype, vscale)
    pos = kv.extend(ints(range(len(lens))), starts)
    assert pos.cpu().tolist() == [0] * len(lens)
    kv.append(layer, k, v, None, pos, starts)
    at = np.concatenate([[0], np.cumsum(lens)])
    K, V = okv.held(num(k)), okv.held(num(v))
    return [(K[at[b]:at[b + 1]], V[at[b]:at[b + 1]]) for b in range(len(lens))]


def shuffle(kv, rng):
    """Gives and takes back pages so that later sequences get theirs out of order."""
    n = kv.n_pages
    perm = torch.from_numpy(rng.permutation(n)).cuda()
    kv.pages.random_(0, 256)                     # free pages hold anything: NaN and infinite scales among it
    kv.pages.copy_(kv.pages[perm])


# ---- rows --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,heads,page", [(32, 1, 16), (64, 2, 32), (96, 3, 16), (128, 4, 64), (256, 5, 16)])
def test_append_bytes_and_gather(cuda_lib, D, heads, page, dtype):
    rng = np.random.default_rng(D + heads)
    kv = make(2, heads, D, n_pages=24, page=page, max_pages=8)
    kv.pages.fill_(0xA5)
    lens = [page + 3, 16, 0, 1, 31]
    starts = starts_of(lens)
    k, v = rows(rng, sum(lens), heads, D, dtype), rows(rng, sum(lens), heads, D, dtype, 3.0)
    k[0, 0, :32] = 0.0                           # a group of zeros
    v[1, heads - 1, :32] = 1e30                  # one whose scale saturates
    pos = kv.extend(None, starts, batch=len(lens))
    kv.append(1, k, v, None, pos, starts)
    gk, gv = kv.gather(1, None, pos, starts, rows=sum(lens))
    wk, wv = okv.held(num(k)).astype(np.float32), okv.held(num(v)).astype(np.float32)
    assert np.array_equal(num(gk), wk) and np.array_equal(num(gv), wv)
    bk, bv = kv.gather(1, None, pos, starts, rows=sum(lens), dtype=torch.bfloat16)
    assert torch.equal(bk, gk.bfloat16()) and torch.equal(bv, gv.bfloat16())
    # the bytes: whole blocks as documented, layer 0 and free pages untouched
    pages = kv.pages.view(kv.n_pages, 2, heads, page // 16, -1).cpu().numpy()
    assert (pages[:, 0] == 0xA5).all() and (pages[kv.refs.cpu().numpy() == 0] == 0xA5).all()
    table, at = kv.tables.cpu().numpy(), np.concatenate([[0], np.cumsum(lens)])
    for b, n in enumerate(lens):
        for p in range(0, n - 15, 16):
            for h in range(heads):
                want = okv.block_bytes(num(k)[at[b] + p:at[b] + p + 16, h], num(v)[at[b] + p:at[b] + p + 16, h])
                assert np.array_equal(pages[table[b, p // page], 1, h, p % page // 16], want)
    assert status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_in_steps_equals_append_at_once(cuda_lib, dtype):
    """Row by row, in odd pieces and at once: the same bytes; a piece leaves its neighbours' bytes alone."""
    rng = np.random.default_rng(1)
    D, heads, total = 96, 2, 53
    k, v = rows(rng, total, heads, D, dtype), rows(rng, total, heads, D, dtype)
    got = []
    for pieces in ([total], [1] * total, [5, 16, 1, 20, 11], [15, 2, 36]):
        kv = make(1, heads, D, page=32)
        kv.pages.zero_()
        at = 0
        for n in pieces:
            pos = kv.extend([3], [0, n])
            assert pos.tolist() == [at]
            # every other piece comes as a strided slice of a wider buffer
            wide = torch.zeros((n, 2 * heads + 1, D), dtype=k.dtype, device="cuda")
            wide[:, :heads], wide[:, heads:2 * heads] = k[at:at + n], v[at:at + n]
            kv.append(0, wide[:, :heads], wide[:, heads:2 * heads], [3], pos, [0, n])
            at += n
        got.append(kv.pages.clone())
    for g in got[1:]:
        assert torch.equal(got[0], g)


def test_nan_and_infinity_in_rows(cuda_lib):
    kv = make(1, 1, 64)
    k = torch.ones((3, 1, 64), device="cuda")
    k[1, 0, 5], k[2, 0, 40] = float("nan"), float("inf")
    pos = kv.extend([0], [0, 3])
    kv.append(0, k, k, [0], pos, [0, 3])
    for g in kv.gather(0, [0], pos, [0, 3], rows=3):
        g = num(g)[:, 0]
        assert np.array_equal(g[0], okv.held(num(k)[0, 0]))
        assert np.isnan(g[1, :32]).all() and not np.isnan(g[1, 32:]).any()      # the group of the NaN
        assert g[2, 40] == 7 * 65504.0 and (g[2, 32:40] == 0).all()               # saturates; the rest of the group vanishes
    # a row that cannot see them is not touched by them
    q = torch.ones((3, 2, 64), device="cuda")
    o = num(kv.attention(0, q, [0], pos, [0, 3]))
    assert np.allclose(o[0], okv.held(num(k)[0, 0]), rtol=1e-5) and np.isnan(o[1]).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rowcounts", [[1, 1, 1], [17, 0, 33, 2]])
def test_rope_append_is_rotation_then_append(cuda_lib, dtype, rowcounts):
    """Same q and same cache as bq_rope_kv_append (dense cache) followed by append."""
    from chadslab_b200 import _lib
    rng = np.random.default_rng(4)
    Hq, Hkv, D, base = 4, 2, 64, 10000.0
    B, T = len(rowcounts), sum(rowcounts)
    kv, ref = make(1, Hkv, D), make(1, Hkv, D)
    kv.pages.zero_(), ref.pages.zero_()
    before = [7, 16, 0, 30][:B]
    for p in (kv, ref):
        p.extend(None, starts_of(before), batch=B)
    qkv = torch.from_numpy(rng.normal(0, 1, (T, (Hq + 2 * Hkv) * D)).astype(np.float32)).cuda()
    starts = starts_of(rowcounts)
    pos = kv.extend(None, starts, batch=B)
    assert torch.equal(pos, ref.extend(None, starts, batch=B))
    one = all(n == 1 for n in rowcounts)
    q = kv.rope_append(0, qkv, Hq, base, None, pos, None if one else starts, dtype=DT[dtype])
    S = 128
    wq = torch.empty((T, Hq, D), dtype=DT[dtype], device="cuda")
    wk, wv = (torch.zeros((T, Hkv, D), dtype=DT[dtype], device="cuda") for _ in range(2))
    row = 0
    for b, n in enumerate(rowcounts):
        for i in range(n):
            p = torch.tensor([before[b] + i], dtype=torch.int64, device="cuda")
            kc, vc = (torch.zeros((1, S, Hkv, D), dtype=DT[dtype], device="cuda") for _ in range(2))
            _lib.check(_lib.lib().bq_rope_kv_append(qkv[row].data_ptr(), p.data_ptr(), wq[row].data_ptr(), kc.data_ptr(), vc.data_ptr(), 1, Hq,
                                                    Hkv, D, S, base, 0 if dtype == "f32" else 1, torch.cuda.current_stream().cuda_stream))
            wk[row], wv[row] = kc[0, before[b] + i], vc[0, before[b] + i]
            row += 1
    ref.append(0, wk, wv, None, pos, starts)
    assert torch.equal(q, wq) and torch.equal(kv.pages, ref.pages) and status() == 0


# ---- pages -------------------------------------------------------------------------------------------------------------
def same(kv, model):
    assert np.array_equal(kv.tables.cpu().numpy(), model.tables)
    assert np.array_equal(kv.lens.cpu().numpy(), model.lens)
    assert np.array_equal(kv.refs.cpu().numpy(), model.refs)


@pytest.mark.parametrize("seed", range(4))
def test_page_bookkeeping_against_restatement(cuda_lib, seed):
    rng = np.random.default_rng(seed)
    n_pages, seqs, most, page = [(20, 6, 5, 16), (300, 33, 9, 32), (17000, 40, 600, 16), (50, 12, 12, 64)][seed]
    kv = make(2, 1, 32, n_pages=n_pages, max_seqs=seqs, max_pages=most, page=page)
    model = okv.Pool(n_pages, seqs, most, page)
    kv.pages.random_(0, 256)
    for _ in range(60):
        what = rng.integers(0, 5)
        slots = rng.permutation(seqs)[:rng.integers(1, seqs + 1)].tolist()
        if what <= 1:
            n = [int(rng.choice([0, 1, 1, 2, page - 1, page, 3 * page + 1, most * page // 2])) for _ in slots]
            before = kv.pages.clone()
            pos = kv.extend(slots, np.concatenate([[0], np.cumsum(n)]).tolist())
            want, copies = model.extend(slots, n)
            assert pos.tolist() == want
            for a, b in copies:
                before[b] = before[a]
            assert torch.equal(before, kv.pages)               # the copies are made, nothing else is written
        elif what == 2:
            dst = rng.integers(0, seqs, len(slots)).tolist()   # destinations may repeat and may be sources
            kv.fork(slots, dst)
            model.fork(slots, dst)
        elif what == 3:
            slots = slots[:max(1, len(slots) // 3)]
            kv.free(slots + slots[:2])                         # the same slot twice
            model.free(slots)
        else:
            live = int((model.refs > 0).sum())
            room = live + int(rng.integers(1, 5))
            to = make(2, 1, 32, n_pages=room, max_seqs=seqs, max_pages=most, page=page)
            to.pages.fill_(7)
            kv.compact(to)
            moved, old = model.compact(room)
            same(to, moved)
            assert torch.equal(to.pages[:live], kv.pages[torch.from_numpy(old).cuda()]) and (to.pages[live:] == 7).all()
        same(kv, model)
    assert status() in (0, -1)           # -1: a sequence would have outgrown its table


def test_extend_refusals(cuda_lib):
    kv = make(1, 1, 32, n_pages=4, max_seqs=4, max_pages=3, page=16)
    assert kv.extend([0, 1, 2], [0, 20, 40, 60]).tolist() == [0, 0, -1]      # 2 + 2 pages; none are left
    assert kv.refs.tolist() == [1, 1, 1, 1] and kv.lens.tolist() == [20, 20, 0, 0] and status() == 0
    assert kv.extend([1, 3, 0], [0, 12, 13, 13]).tolist() == [20, -1, 20] and status() == 0    # what needs no page is served
    assert kv.extend([0, 0], [0, 1, 2]).tolist() == [20, -1] and status() == -1               # twice in one batch
    assert kv.extend([0, 9, -1], [0, 1, 2, 3]).tolist() == [21, -1, -1] and status() == -1    # no such slot
    assert kv.extend([0], [0, 40]).tolist() == [-1] and status() == -1                        # longer than the table
    small = make(1, 1, 32, n_pages=3, max_seqs=4, max_pages=3, page=16)
    kv.compact(small)
    assert status() == -4 and small.lens.tolist() == [0] * 4 and small.refs.tolist() == [0] * 3
    kv.free([7])
    assert status() == -1
    kv.fork([0, 9], [1, 2])
    assert status() == -1 and kv.lens.tolist() == [22, 22, 0, 0] and kv.refs.tolist() == [2, 2, 0, 0]
    # an append or attention that names a place outside the pool takes no part
    k = torch.ones((2, 1, 32), device="cuda")
    kept = kv.pages.clone()
    kv.append(0, k, k, [9, 0], [0, 48])
    assert torch.equal(kept, kv.pages) and status() == -1
    kv.append(0, k, k, [3, 2], [0, 0])                                        # sequences without pages
    assert torch.equal(kept, kv.pages) and status() == -1
    o = kv.attention(0, torch.ones((2, 1, 32), device="cuda"), [9, 0], [3, -1])
    assert (o == 0).all() and status() == -1


# ---- attention ---------------------------------------------------------------------------------------------------------
def bound(o, mag, size, V, dtype):
    """Per element.  fp32: queries and weights are held in 22 bits or more (2^-22 relative to every product), sums in fp32.
    A score's sum has D products in at most 16 dependent additions on any path (a matrix instruction's 16 products count as
    two, groups of 32 are added one after the other, lanes pairwise), each off by up to 2^-24 of the sum of |q k|: the
    score is off by at most (2^-22 + 16 * 2^-24) * sum |q k| / sqrt(D), which moves every weight by that share, numerator
    and denominator; exp2 and the division add a few 2^-23.  bf16: a key's
    code is a subnormal fp16 n * 2^-24 with n < 16, whose products the matrix unit aligns as if they had their exponent's
    whole 2^-14: up to 2^6 times coarser, i.e. 16 * 2^-18 in place of 16 * 2^-24; weights (times a scale) are rounded to
    fp16 twice (2^-11 each) and the result once (2^-8 of itself).  Weights far below the largest, which is held as 2^11 or more, are
    lost: a weight, and its product with a scale, is off by up to 2^-25 (fp32: the 2^-36 of its second half), times a code
    of at most 7 or a value."""
    lost = len(V) * 2.0 ** (-36 if dtype == "bf16" else -47) * (7.0 + np.abs(V).max())
    score = 2.0 * size * (2.0 ** -22 + 16 * 2.0 ** (-24 if dtype == "f32" else -18))
    if dtype == "f32":
        return (2.0 ** -20 + score) * mag + lost
    return (2 * 2.0 ** -11 + 2.0 ** -20 + score) * mag * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(o) + lost


def check(kv, layer, data, lens, new, Hq, dtype, rng, q_scale=1.5, strided=False):
    """Attention of the last new[b] rows of every sequence against 64 bits."""
    T, D = sum(new), kv.head_dim
    q = rows(rng, T, Hq, D, dtype, q_scale)
    if strided:
        wide = torch.zeros((T, Hq + 3, D), dtype=q.dtype, device="cuda")
        wide[:, :Hq] = q
        q = wide[:, :Hq]
    pos = [n - m for n, m in zip(lens, new)]
    one = all(m == 1 for m in new)
    out = kv.attention(layer, q, ints(range(len(lens))), ints(pos), None if one else starts_of(new))
    at = np.concatenate([[0], np.cumsum(new)])
    for b in range(len(lens)):
        if new[b] == 0:
            continue
        o, mag, size = okv.attention(num(q)[at[b]:at[b + 1]], data[b][0], data[b][1], pos[b])
        err = np.abs(num(out)[at[b]:at[b + 1]] - o)
        tol = bound(o, mag, size, data[b][1], dtype)
        assert (err <= tol).all(), f"sequence {b} (len {lens[b]}): {np.nanmax(err / np.maximum(tol, 1e-300)):.2f} x the bound"
    assert status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Hkv,rep", [(32, 2, 1), (32, 1, 16), (64, 2, 1), (64, 1, 4), (64, 3, 8), (96, 2, 3), (128, 2, 1), (128, 2, 2),
                                       (128, 1, 4), (128, 2, 8), (128, 1, 16), (128, 1, 5), (160, 2, 2), (192, 1, 1), (224, 1, 6), (256, 2, 1),
                                       (256, 1, 2), (256, 1, 3), (256, 1, 8), (256, 1, 17)])
def test_decode_attention(cuda_lib, D, Hkv, rep, dtype):
    rng = np.random.default_rng(D * 100 + Hkv * 10 + rep)
    kv = make(2, Hkv, D, n_pages=150, max_seqs=9, max_pages=40, page=16)
    shuffle(kv, rng)
    lens = [1, 2, 15, 16, 17, 63, 65, 300, 129]
    data = fill(kv, 1, lens, rng, dtype)
    check(kv, 1, data, lens, [1] * len(lens), Hkv * rep, dtype, rng)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Hkv,rep,page", [(64, 1, 2, 64), (128, 2, 4, 32), (256, 1, 1, 128), (256, 1, 8, 16), (96, 2, 1, 64)])
def test_chunk_attention(cuda_lib, D, Hkv, rep, page, dtype):
    """Chunks behind context, whole prompts, single tokens and sequences without rows in one batch."""
    rng = np.random.default_rng(D + rep)
    lens, new = [70, 33, 200, 5, 64, 1], [17, 33, 1, 0, 30, 1]
    kv = make(1, Hkv, D, n_pages=64, max_pages=16, page=page)
    shuffle(kv, rng)
    data = fill(kv, 0, lens, rng, dtype)
    check(kv, 0, data, lens, new, Hkv * rep, dtype, rng, strided=True)


def many_rows(kv, heads, B, n_rows):
    """Whether a call of these sizes takes the kernel that works on 128 (row, head) pairs at a time (its scratch tells)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    need = kv._lib.bq_kv4_attention_work_bytes(kv._p, heads, 1, B, n_rows)
    return need == 1024 * 32 + sms * 2 * 128 * (kv.head_dim + 4) * 4


@pytest.mark.parametrize("D,Hkv,rep,page", [(64, 8, 3, 16), (64, 8, 2, 32), (128, 4, 4, 64), (128, 1, 16, 16), (256, 2, 8, 64), (256, 8, 2, 16)])
def test_many_rows_attention(cuda_lib, D, Hkv, rep, page):
    """Chunks long enough for the kernel that works on 128 (row, head) pairs at a time: odd lengths, whole prompts, sequences
    without rows, several tiles of pairs and of positions, cut segments."""
    rng = np.random.default_rng(D + rep)
    lens, new = [333, 70, 260, 5, 64, 129], [140, 70, 1, 0, 64, 128]
    kv = make(2, Hkv, D, n_pages=80, max_pages=24, page=page)
    assert many_rows(kv, Hkv * rep, len(lens), sum(new)) and not many_rows(kv, Hkv * rep, 6, 6)
    shuffle(kv, rng)
    data = fill(kv, 1, lens, rng, "bf16", 20.0 if D == 64 else 1.0)
    check(kv, 1, data, lens, new, Hkv * rep, "bf16", rng, strided=True)


@pytest.mark.parametrize("vscale", [1e-3, 2000.0])
def test_many_rows_ranges_and_bytes_behind(cuda_lib, vscale):
    """Values far from one; the rest of a last block can hold anything and one row behind another sees the same bits."""
    lens, new, got = [100, 83], [90, 83], []
    for fill_with in (0, 0x7C00, 0x7E00, 0x7BFF, -1):
        rng = np.random.default_rng(8)
        kv = make(1, 24, 128, page=32)
        assert many_rows(kv, 48, 2, sum(new))
        kv.pages.view(torch.int16).fill_(fill_with)
        data = fill(kv, 0, lens, rng, "bf16", vscale)
        q = rows(rng, sum(new), 48, 128, "bf16", 6.0)
        pos = ints([n - m for n, m in zip(lens, new)])
        got.append(kv.attention(0, q, None, pos, starts_of(new)))
        assert torch.equal(got[-1], got[0])
    check(kv, 0, data, lens, new, 48, "bf16", np.random.default_rng(3))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Hkv,rep", [(64, 1, 1), (128, 1, 8), (256, 2, 1)])
def test_long_context_attention(cuda_lib, D, Hkv, rep, dtype):
    rng = np.random.default_rng(9)
    lens = [20011, 3, 4097]
    kv = make(1, Hkv, D, n_pages=400, max_seqs=4, max_pages=320, page=64)
    shuffle(kv, rng)
    data = fill(kv, 0, lens, rng, dtype)
    check(kv, 0, data, lens, [1, 1, 1], Hkv * rep, dtype, rng)


@pytest.mark.parametrize("D,Hkv,rep,lens", [(64, 4, 1, [6000] * 90), (128, 4, 4, [5000] * 70), (256, 2, 2, [4500] * 60)])
def test_fp32_rows_keep_their_precision_over_long_runs(cuda_lib, D, Hkv, rep, lens):
    """Many steps of one run into the same sums.  Their errors are to be those of single steps, not of their number: 2-norm of
    the error over that of the result.  The exponent of a weight, up to 16, is rounded to 2^-21 absolute (a share of 2^-21.5 of
    the weight, at random), weights and queries are held to 2^-22 of themselves and sums rounded to nearest: below 2^-20
    together.  Truncated sums would be off by their number of steps, 100 and more here, times 2^-25."""
    rng = np.random.default_rng(D)
    kv = make(1, Hkv, D, n_pages=len(lens) * -(-lens[0] // 64), max_seqs=len(lens), max_pages=-(-lens[0] // 64), page=64)
    starts = starts_of(lens)
    k = torch.randn((sum(lens), Hkv, D), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    v = torch.randn((sum(lens), Hkv, D), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    kv.append(0, k, v, None, kv.extend(None, starts), starts)
    q = rows(rng, len(lens), Hkv * rep, D, "f32")
    out = num(kv.attention(0, q, None, ints([n - 1 for n in lens])))
    for b in (0, len(lens) // 2, len(lens) - 1):
        one = slice(sum(lens[:b]), sum(lens[:b + 1]))
        o, _, _ = okv.attention(num(q)[b:b + 1], okv.held(num(k[one])), okv.held(num(v[one])), lens[b] - 1)
        assert np.linalg.norm(out[b] - o[0]) <= 2.0 ** -20 * np.linalg.norm(o), b


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_scale,vscale", [(12.0, 1.0), (1e-3, 1e-3), (3.0, 2000.0), (1e4, 1.0), (0.0, 50.0)])
def test_attention_ranges(cuda_lib, q_scale, vscale, dtype):
    """Peaked and flat weights, values far below and above one (whose scales leave the range that fp16 weights have)."""
    rng = np.random.default_rng(11)
    lens = [700, 40]
    kv = make(1, 2, 128, n_pages=64, max_pages=60, page=16)
    shuffle(kv, rng)
    data = fill(kv, 0, lens, rng, dtype, vscale)
    check(kv, 0, data, lens, [1, 1], 4, dtype, rng, q_scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,rep", [(64, 1), (64, 5), (128, 3), (256, 1), (256, 17), (96, 2)])
def test_bytes_behind_a_sequence_do_not_matter(cuda_lib, D, rep, dtype):
    """The rest of a last block can hold anything (scales of infinity, NaN, 65504, negative ones): the same bits."""
    lens, new = [3, 17, 64, 41, 1], [1, 1, 1, 9, 1]
    got = []
    for fill_with in (0, 0x7C00, 0x7E00, 0x7BFF, -0x8000 + 0x7C00, -1):
        rng = np.random.default_rng(21)
        kv = make(1, 1, D, page=32)
        kv.pages.view(torch.int16).fill_(fill_with)
        fill(kv, 0, lens, rng, dtype)
        q = rows(rng, sum(new), rep, D, dtype)
        pos = [n - m for n, m in zip(lens, new)]
        got.append([kv.attention(0, q, None, ints(pos), starts_of(new)), kv.attention(0, q[:5], None, ints([n - 1 for n in lens]))])
    for g in got[1:]:
        assert torch.equal(g[0], got[0][0]) and torch.equal(g[1], got[0][1])
    assert torch.isfinite(got[0][0]).all() and status() == 0


def test_attention_rows_of_nobody(cuda_lib):
    """Rows behind the last sequence stay as they were, rows of a refused sequence are zero."""
    rng = np.random.default_rng(2)
    kv = make(1, 2, 64)
    fill(kv, 0, [20, 9, 30], rng)
    q = rows(rng, 9, 4, 64, "bf16")
    out = torch.full((9, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    kv.attention(0, q, [0, 1, 2], [18, -1, 27], [0, 2, 4, 7], out=out)
    o = num(out)
    assert (o[7:] == 5).all() and (o[2:4] == 0).all() and np.isfinite(o).all() and (o[:2] != 5).any() and (o[4:7] != 5).any()
    assert kv.attention(0, q[:0], [], []).shape == (0, 4, 64)


def test_calls_repeat_bit_for_bit_and_streams(cuda_lib):
    rng = np.random.default_rng(3)
    kv = make(1, 2, 128, n_pages=200, max_pages=100, page=16)
    fill(kv, 0, [1500, 800], rng)
    q = rows(rng, 2, 8, 128, "bf16")
    slots, pos = ints([0, 1]), ints([1499, 799])
    ref = kv.attention(0, q, slots, pos)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:                            # at the same time on several streams: every call has scratch of its own
        with torch.cuda.stream(s):
            outs += [kv.attention(0, q, slots, pos) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(ref, o) for o in outs)


def test_serving_run_in_a_graph(cuda_lib):
    """Prompts, a fork of one of them, decode steps replayed from a captured graph, one sequence leaves, the pool is
    compacted: at every step what 64 bits say."""
    rng = np.random.default_rng(5)
    L, Hkv, rep, D, steps = 2, 2, 2, 64, 20
    kv = make(L, Hkv, D, n_pages=40, max_seqs=4, max_pages=8, page=16)
    shuffle(kv, rng)
    lens = [19, 40]
    starts = starts_of(lens)
    pos = kv.extend([0, 1], starts)
    hist = [[None, None] for _ in range(L)]
    K = [[[] for _ in range(3)] for _ in range(L)]
    V = [[[] for _ in range(3)] for _ in range(L)]
    for l in range(L):
        k, v = rows(rng, sum(lens), Hkv, D, "bf16"), rows(rng, sum(lens), Hkv, D, "bf16")
        kv.append(l, k, v, [0, 1], pos, starts)
        for b, (a, e) in enumerate(((0, 19), (19, 59))):
            K[l][b], V[l][b] = list(okv.held(num(k)[a:e])), list(okv.held(num(v)[a:e]))
    kv.fork([0], [2])
    for l in range(L):
        K[l][2], V[l][2] = list(K[l][0]), list(V[l][0])
    lens = [19, 40, 19]
    slots = ints([0, 1, 2])
    k, v = (torch.zeros((L, 3, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, out = (torch.zeros((L, 3, Hkv * rep, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def step():
        at = kv.extend(slots)
        for l in range(L):
            kv.append(l, k[l], v[l], slots, at)
            kv.attention(l, q[l], slots, at, out=out[l])

    keep = [t.clone() for t in (kv.tables, kv.lens, kv.refs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for t, s in zip((kv.tables, kv.lens, kv.refs), keep):
        t.copy_(s)
    for i in range(steps):
        for t in (k, v, q):
            t.copy_(torch.from_numpy(rng.normal(0, 1, tuple(t.shape)).astype(np.float32)))
        graph.replay()
        for l in range(L):
            for b in range(3):
                K[l][b].append(okv.held(num(k[l, b])))
                V[l][b].append(okv.held(num(v[l, b])))
                o, mag, size = okv.attention(num(q[l, b])[None], np.array(K[l][b]), np.array(V[l][b]), lens[b] + i)
                assert (np.abs(num(out[l, b])[None] - o) <= bound(o, mag, size, np.array(V[l][b]), "bf16")).all(), (i, l, b)
    assert kv.lens.tolist()[:3] == [n + steps for n in lens]
    kv.free([1])
    small = make(L, Hkv, D, n_pages=7, max_seqs=4, max_pages=8, page=16)
    kv.compact(small)
    assert small.lens.tolist() == [39, 0, 39, 0] and status() == 0
    q1 = q[1, [0, 2]].contiguous()
    a, b = (p.attention(1, q1, [0, 2], [38, 38]) for p in (kv, small))
    assert torch.equal(a, b)


def test_many_sequences(cuda_lib):
    """Batches of several hundred sequences (the searches over sequences take more than one pass), some without rows, some
    refused."""
    rng = np.random.default_rng(17)
    B, Hkv, rep, D = 700, 1, 2, 64
    lens = [int(x) for x in rng.choice([0, 1, 2, 15, 16, 17, 40], B)]
    kv = make(1, Hkv, D, n_pages=1800, max_seqs=1000, max_pages=4, page=16)
    shuffle(kv, rng)
    slots = rng.permutation(1000)[:B]
    starts = starts_of(lens)
    k, v = rows(rng, sum(lens), Hkv, D, "bf16"), rows(rng, sum(lens), Hkv, D, "bf16")
    pos = kv.extend(ints(slots), starts)
    assert (pos == 0).all()
    kv.append(0, k, v, ints(slots), pos, starts)
    gk, gv = kv.gather(0, ints(slots), pos, starts, rows=sum(lens))
    K, V = okv.held(num(k)), okv.held(num(v))
    assert np.array_equal(num(gk), K.astype(np.float32)) and np.array_equal(num(gv), V.astype(np.float32))
    q = rows(rng, sum(lens), Hkv * rep, D, "bf16")
    refused = rng.random(B) < 0.1
    some = torch.where(torch.from_numpy(refused).cuda(), -1, pos).int()
    out = num(kv.attention(0, q, ints(slots), some, starts))
    at = np.concatenate([[0], np.cumsum(lens)])
    for b in range(B):
        one = slice(at[b], at[b + 1])
        if refused[b]:
            assert (out[one] == 0).all()
        elif lens[b]:
            o, mag, size = okv.attention(num(q)[one], K[one], V[one], 0)
            assert (np.abs(out[one] - o) <= bound(o, mag, size, V[one], "bf16")).all(), b
    assert status() == 0


@pytest.mark.parametrize("many", [False, True])
def test_pool_past_32_bits(cuda_lib, many):
    """Pages, layers and tables whose byte offsets pass 2^32, and rows of q and out that do not start at the tensor's start."""
    rng = np.random.default_rng(4)
    L, Hkv, rep, D, page = 40, 8, 2, 128, 64
    from chadslab_b200 import PagedKV4
    kv = PagedKV4(L, Hkv, D, n_pages=2300, max_seqs=8, max_pages=8, page=page)
    assert kv.pages.numel() > 2 ** 32 + 2 ** 31
    kv.refs[:2270] = 1                                # all that is given out lies behind 2^32 bytes
    lens = [200, 1, 130, 64, 77, 300]
    data = fill(kv, L - 1, lens, rng)
    assert int(kv.tables[kv.tables >= 0].min()) >= 2270
    new = [130, 1, 130, 64, 60, 100] if many else [1] * 6
    assert many_rows(kv, Hkv * rep, 6, sum(new)) == many
    check(kv, L - 1, data, lens, new, Hkv * rep, "bf16", rng, strided=True)
    kv.fork([0, 5], [6, 7])
    assert kv.extend([6, 7]).tolist() == [200, 300]      # copies of whole pages, all layers
    a, b = (kv.gather(L - 1, [s], [0], [0, 200], rows=200)[0] for s in (0, 6))
    assert torch.equal(a, b) and status() == 0


def test_refusals_of_the_c_abi(cuda_lib):
    """Bad arguments come back as codes and nothing is launched."""
    from chadslab_b200 import _lib
    kv = make(2, 2, 64, n_pages=8, max_seqs=4)
    lib, p = _lib.lib(), kv._p
    x = torch.zeros(4096, device="cuda")
    i = ints(range(8))
    at, ip, s = x.data_ptr(), i.data_ptr(), torch.cuda.current_stream().cuda_stream
    n0 = lib.bq_launch_count()
    att = lambda layer=0, q=at, ldq=256, out=at, Hq=4, dt=0, pos=ip, B=2, rows=2, work=at: lib.bq_kv4_attention(
        p, layer, q, ldq, out, Hq, dt, None, pos, None, B, rows, work, s)
    app = lambda layer=0, k=at, v=at, ldk=128, ldv=128, dt=0, pos=ip, B=2, rows=2: lib.bq_kv4_append(
        p, layer, k, v, ldk, ldv, dt, None, pos, None, B, rows, s)
    rope = lambda Hq=4, q=at, B=2, rows=2, dt=0: lib.bq_kv4_rope_append(p, 0, at, q, Hq, 1e4, dt, None, ip, None, B, rows, s)
    bad = [att(layer=2), att(layer=-1), att(q=None), att(out=None), att(work=None), att(pos=None), att(Hq=3), att(Hq=0), att(dt=2), att(ldq=255),
           att(ldq=254), att(B=5, rows=5), att(B=-1), att(rows=3), att(q=at + 4), att(out=at + 4), att(work=at + 8), app(layer=2), app(k=None),
           app(v=None), app(ldk=127), app(dt=7), app(k=at + 2), app(B=5, rows=5), app(rows=1), app(pos=None), rope(Hq=3), rope(q=None), rope(dt=2),
           rope(rows=3), lib.bq_kv4_gather(p, 0, None, at, 0, None, ip, None, 2, 2, s), lib.bq_kv4_gather(p, 0, at, at, 0, None, ip, None, 2, 1, s),
           lib.bq_kv4_extend(p, None, None, 5, ip, s), lib.bq_kv4_extend(p, None, None, 2, None, s), lib.bq_kv4_extend(None, None, None, 1, ip, s),
           lib.bq_kv4_fork(p, None, ip, 1, s), lib.bq_kv4_fork(p, ip, ip, 5, s), lib.bq_kv4_free(p, None, 1, s), lib.bq_kv4_free(p, ip, -1, s),
           lib.bq_kv4_compact(p, p, s), lib.bq_kv4_compact(p, make(2, 2, 64, max_seqs=5)._p, s), lib.bq_kv4_compact(p, None, s)]
    assert bad == [-1] * len(bad) and lib.bq_launch_count() == n0
    for field, value in (("head_dim", 40), ("page", 48), ("n_pages", 0), ("max_seqs", 9000), ("pages", None), ("refs", at + 4)):
        q = _lib.Kv4Pool.from_buffer_copy(kv._pool)
        setattr(q, field, value)
        assert lib.bq_kv4_free(C.byref(q), ip, 1, s) == -1 and lib.bq_last_error()
    # nothing to do is not an error
    assert att(B=0, rows=0) == 0 and app(B=0, rows=0) == 0 and lib.bq_kv4_free(p, ip, 0, s) == 0 and lib.bq_launch_count() == n0


def test_refusals_of_the_python_surface(cuda_lib):
    import chadslab_b200 as cb
    kv = make(1, 2, 64)
    k, q = torch.zeros((2, 2, 64), device="cuda"), torch.zeros((2, 4, 64), device="cuda")
    for call, error in [(lambda: kv.append(0, k.half(), k.half(), [0, 1], [0, 0]), TypeError), (lambda: kv.append(0, k, k.bfloat16(), [0, 1], [0, 0]), ValueError),
                        (lambda: kv.append(0, k[:, :1], k, [0, 1], [0, 0]), ValueError), (lambda: kv.append(0, k.cpu(), k, [0, 1], [0, 0]), cb.BqError),
                        (lambda: kv.append(0, k, k, [0], [0, 0]), ValueError), (lambda: kv.append(0, k, k, [0, 1], [0, 0], [0, 1]), ValueError),
                        (lambda: kv.append(0, k, k, torch.tensor([0, 1], device="cuda"), [0, 0]), cb.BqError),
                        (lambda: kv.append(1, k, k, [0, 1], [0, 0]), cb.BqError), (lambda: kv.attention(0, q[:, :3], [0, 1], [0, 0]), ValueError),
                        (lambda: kv.attention(0, q[..., :32], [0, 1], [0, 0]), ValueError), (lambda: kv.attention(0, q, [0, 1], [0, 0], out=q.bfloat16()), ValueError),
                        (lambda: kv.attention(0, q, [0, 1, 2], [0, 0, 0]), cb.BqError), (lambda: kv.fork([0], [1, 2]), ValueError),
                        (lambda: kv.extend([0, 1], [0, 1]), ValueError), (lambda: kv.rope_append(0, k.flatten(1), 2, 1e4, [0, 1], [0, 0]), ValueError),
                        (lambda: kv.rope_append(0, torch.zeros((2, 512), device="cuda").bfloat16(), 4, 1e4, [0, 1], [0, 0]), cb.BqError),
                        (lambda: kv.compact(kv), cb.BqError), (lambda: kv.gather(0, [0], [0], dtype=torch.float16), TypeError)]:
        with pytest.raises(error):
            call()
    # rows that are not dense, or not aligned, are copied
    kv.extend([0, 1], [0, 1, 2])
    odd = torch.randn((2, 64, 2), device="cuda").transpose(1, 2)
    kv.append(0, odd, odd, [0, 1], [0, 0])
    assert np.array_equal(num(kv.gather(0, [0, 1], [0, 0])[0]), okv.held(num(odd)).astype(np.float32)) and status() == 0


@pytest.mark.parametrize("many", [False, True])
def test_rows_in_front_of_the_first_sequence(cuda_lib, many):
    """Row ranges need not begin at row 0: what lies in front is neither read nor written, by any call."""
    rng = np.random.default_rng(6)
    Hkv, rep, D, front = 8, 2, 64, 21
    lens = [70, 33, 90, 64, 1, 80] if many else [20, 3, 0, 17]
    kv, ref = make(1, Hkv, D, n_pages=64, max_pages=8), make(1, Hkv, D, n_pages=64, max_pages=8)
    T = front + sum(lens)
    assert many_rows(kv, Hkv * rep, len(lens), T) == many
    k, v, q = rows(rng, T, Hkv, D, "bf16"), rows(rng, T, Hkv, D, "bf16"), rows(rng, T, Hkv * rep, D, "bf16")
    k[:front] = float("nan")
    starts = starts_of(lens) + front
    for pool, kk, vv, st in ((kv, k, v, starts), (ref, k[front:], v[front:], starts_of(lens))):
        pool.pages.zero_()
        pos = pool.extend(None, st, batch=len(lens))
        assert pos.tolist() == [0] * len(lens)
        pool.append(0, kk, vv, None, pos, st)
    assert torch.equal(kv.pages, ref.pages)
    out = torch.full((T, Hkv * rep, D), 9.0, dtype=torch.bfloat16, device="cuda")
    kv.attention(0, q, None, pos, starts, out=out)
    want = ref.attention(0, q[front:].contiguous(), None, pos, starts_of(lens))
    # both within half a bf16 step (2^-8) of the same value but for the fp16 weights (2^-10 of values of about one)
    assert (out[:front] == 9).all() and torch.allclose(out[front:].float(), want.float(), rtol=2 ** -6, atol=1e-3)
    gk, gv = kv.gather(0, None, pos, starts, rows=T)
    assert np.array_equal(num(gk)[front:], okv.held(num(k)[front:]).astype(np.float32))
    qkv = torch.randn((T, (Hkv * rep + 2 * Hkv) * D), device="cuda")
    q_out = torch.full((T + 2, Hkv * rep, D), 9.0, dtype=torch.bfloat16, device="cuda")[:T]
    skip = torch.where(torch.arange(len(lens), device="cuda") == 0, -1, pos).int()        # the first sequence takes no part
    kv.rope_append(0, qkv, Hkv * rep, 1e4, None, skip, starts, q_out=q_out)
    first = front + lens[0]
    assert (q_out[:first] == 9).all() and (q_out[first:] != 9).any() and status() == 0


@pytest.mark.parametrize("page", [512, 4096])
def test_large_pages(cuda_lib, page):
    rng = np.random.default_rng(page)
    lens = [5000, 511, 513, 1]
    kv = make(1, 1, 64, n_pages=24, max_seqs=4, max_pages=-(-5120 // page) + 1, page=page)
    shuffle(kv, rng)
    data = fill(kv, 0, lens, rng, "bf16")
    check(kv, 0, data, lens, [1, 3, 1, 1], 2, "bf16", rng)
    kv.fork([0, 1], [2, 3])
    assert kv.extend([2, 3]).tolist() == [5000, 511] and kv.lens.tolist() == [5000, 511, 5001, 512] and status() == 0


def test_bookkeeping_of_thousands_of_sequences(cuda_lib):
    """More sequences than the planning CTA has threads, more pages than it looks at in one pass."""
    rng = np.random.default_rng(30)
    seqs, most, page, n_pages = 3000, 4, 16, 40000
    kv, model = make(1, 1, 32, n_pages=n_pages, max_seqs=seqs, max_pages=most, page=page), okv.Pool(n_pages, seqs, most, page)
    taken = rng.random(n_pages) < 0.9                        # pages that belong to somebody else
    kv.refs[torch.from_numpy(taken).cuda()] = 1
    model.refs[taken] = 1
    for _ in range(3):
        slots = rng.permutation(seqs)[:2700].tolist()
        n = rng.integers(0, 20, len(slots)).tolist()         # the last ones find no pages left, or outgrow their table
        pos = kv.extend(slots, np.concatenate([[0], np.cumsum(n)]).tolist())
        want, _ = model.extend(slots, n)
        assert pos.tolist() == want
        same(kv, model)
    dst = rng.integers(0, seqs, 1500).tolist()
    src = rng.permutation(seqs)[:1500].tolist()
    kv.fork(src, dst)
    model.fork(src, dst)
    same(kv, model)
    kv.free(list(range(0, seqs, 2)))
    model.free(list(range(0, seqs, 2)))
    same(kv, model)
    status()
