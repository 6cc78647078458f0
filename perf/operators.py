"""What the paged 4-bit KV cache is measured on.

Four operators: `append` (rows are quantised into pages, and read back), `attend` (attention of one token per sequence, or
of a chunk of tokens, over the pages), `branch` (sequences are freed, forked and extended: page tables, reference counts,
copies of shared pages) and `compact` (live pages move into another pool).  `run` computes them with elementary torch
operations, or, with `own`, through `chadslab_b200.PagedKV4`.

Page layout (bytes): pages[n_pages][layers][kv_heads][page / 16 blocks of 16 positions][576 * head_dim / 32]; a block holds
K codes, K scales, V codes, V scales of its 16 positions.  See `_layout` for the place of every nibble.
"""
import math
import random

import torch

own = False

SHARE = 0.6180339887498949          # golden ratio: spreads the ragged lengths without a random source


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step's new rows of a batch of 64 (16 heads of 256): launch-bound, runs once per layer and token
        dict(name="append_step_b64", op="append", batch=64, new=1, ctx=2048, ragged=False, kv_heads=16, head_dim=256, page=64,
             layers=1, dtype="bf16"),
        # prompts of different lengths arriving behind earlier context, fp32 activations
        dict(name="append_prompts_f32", op="append", batch=9, new=1111, ctx=333, ragged=True, kv_heads=4, head_dim=128, page=32,
             layers=2, dtype="f32"),
        # a single chat turn on the small dense shape (8 query heads on one KV head): latency counts
        dict(name="decode_b1", op="attend", batch=1, new=1, ctx=131, ragged=False, heads=8, kv_heads=1, head_dim=256, page=64,
             layers=1, dtype="bf16"),
        # the large dense shape (16 heads, one KV head each) at batch 64 behind 2048 positions: the ordinary decode step
        dict(name="decode_b64_mha", op="attend", batch=64, new=1, ctx=2048, ragged=False, heads=16, kv_heads=16, head_dim=256,
             page=64, layers=1, dtype="bf16"),
        # the sparse-MoE shape (32 query heads on 4 KV heads) with sequences of very different lengths
        dict(name="decode_b96_ragged", op="attend", batch=96, new=1, ctx=8000, ragged=True, heads=32, kv_heads=4, head_dim=128,
             page=64, layers=1, dtype="bf16"),
        # two long contexts: few rows, the positions have to be split
        dict(name="decode_long_b2", op="attend", batch=2, new=1, ctx=131072, ragged=False, heads=32, kv_heads=4, head_dim=128,
             page=128, layers=1, dtype="bf16"),
        # fp32 activations, small heads, odd lengths, small pages
        dict(name="decode_f32_b7", op="attend", batch=7, new=1, ctx=1801, ragged=True, heads=4, kv_heads=2, head_dim=64, page=16,
             layers=2, dtype="f32"),
        # chunks of prompts behind cached context
        dict(name="chunk_b4", op="attend", batch=4, new=512, ctx=2500, ragged=True, heads=8, kv_heads=1, head_dim=256, page=64,
             layers=1, dtype="bf16"),
        # three continuations of one prompt on a small model
        dict(name="branch_small", op="branch", prompts=1, branches=3, new=1, ctx=100, ragged=False, layers=2, kv_heads=1,
             head_dim=64, page=16),
        # seven continuations of each of eight prompts, all layers of the small dense shape
        dict(name="branch_p8x7", op="branch", prompts=8, branches=7, new=5, ctx=2000, ragged=True, layers=18, kv_heads=1,
             head_dim=256, page=64),
        # a small pool after a few sequences have left
        dict(name="compact_small", op="compact", batch=5, ctx=200, ragged=True, layers=2, kv_heads=1, head_dim=64, page=16),
        # a pool of the sparse-MoE shape (4 KV heads of 128, a few layers' worth), two thirds full
        dict(name="compact_moe", op="compact", batch=40, ctx=2048, ragged=True, layers=24, kv_heads=4, head_dim=128, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "branch", "compact"])
    D, page = rng.choice([32, 64, 96, 128, 160, 256, 256]), rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    c = dict(op=op, kv_heads=kv, head_dim=D, page=page, ragged=rng.random() < 0.7)
    if op == "append":
        c.update(batch=_log(rng, 1, 64), new=_log(rng, 1, 400), ctx=_log(rng, 1, 1000), layers=rng.choice([1, 2]),
                 dtype=rng.choice(["bf16", "f32"]))
        while c["batch"] * (c["new"] + c["ctx"]) * kv * D > 1 << 26:
            c["batch"], c["new"] = max(1, c["batch"] // 2), max(1, c["new"] // 2)
    elif op == "attend":
        c.update(batch=_log(rng, 1, 128), ctx=_log(rng, 1, 60000), heads=kv * rng.choice([1, 1, 2, 3, 4, 8, 16]), layers=rng.choice([1, 2]),
                 new=rng.choice([1, 1, 1, 1, _log(rng, 2, 9), _log(rng, 10, 150)]), dtype=rng.choice(["bf16", "bf16", "f32"]))
        while (c["batch"] * c["ctx"] * kv * D > 1 << 28 or c["batch"] * c["new"] * c["ctx"] * c["heads"] * D > 1 << 32
               or c["batch"] * c["new"] * c["ctx"] * c["heads"] > 1 << 28):
            if c["batch"] > 1 and rng.random() < 0.5:
                c["batch"] = c["batch"] // 2
            else:
                c["ctx"] = max(1, c["ctx"] * 2 // 3)
    else:
        c.update(ctx=_log(rng, 1, 2000), layers=_log(rng, 1, 24))
        if op == "branch":
            c.update(prompts=_log(rng, 1, 10), branches=rng.choice([1, 2, 3, 5, 8]), new=rng.choice([1, 1, 2, 7, page + 3]))
        else:
            c.update(batch=_log(rng, 1, 50))
        while _pool_bytes(c) > 1 << 29:
            if c["layers"] > 2:
                c["layers"] //= 2
            else:
                c["ctx"] = max(1, c["ctx"] * 2 // 3)
    return c


def _spread(n, most, shift):
    """n lengths in 1..most, the first of them `most`."""
    return [most if i == 0 else 1 + int((most - 1) * ((i * SHARE + shift) % 1.0)) for i in range(n)]


def _lengths(c):
    """(positions before the new rows, new rows) of every sequence."""
    B = c["batch"]
    if c["op"] == "append":
        before = _spread(B, c["ctx"], 0.1) if c["ragged"] else [c["ctx"]] * B
        return before, _spread(B, c["new"], 0.4) if c["ragged"] else [c["new"]] * B
    after = _spread(B, c["ctx"], 0.2) if c["ragged"] else [c["ctx"]] * B
    new = [min(a, n) for a, n in zip(after, _spread(B, c["new"], 0.7) if c["ragged"] else [c["new"]] * B)]
    return [a - n for a, n in zip(after, new)], new


def _page_bytes(c):
    return c["layers"] * c["kv_heads"] * (c["page"] // 16) * 576 * (c["head_dim"] // 32)


def _seqs(c):
    """Lengths of the sequences of a `branch` or `compact` case."""
    n = c["prompts"] if c["op"] == "branch" else c["batch"]
    return _spread(n, c["ctx"], 0.3) if c["ragged"] else [c["ctx"]] * n


def _new_pages(c):
    """(pages that the branches get, how many of those are copies) of a `branch` case."""
    got = copies = 0
    for n in _seqs(c):
        cow = int(n % c["page"] != 0)
        got += c["branches"] * (-(-(n + c["new"]) // c["page"]) - -(-n // c["page"]) + cow)
        copies += c["branches"] * cow
    return got, copies


def _pool_pages(c):
    live = sum(-(-n // c["page"]) for n in _seqs(c))
    return live + _new_pages(c)[0] + 3 if c["op"] == "branch" else live + live // 2 + 2


def _pool_bytes(c):
    return _pool_pages(c) * _page_bytes(c)


def work(c):
    D = c["head_dim"]
    if c["op"] == "append":
        rows = sum(_lengths(c)[1]) * c["kv_heads"]
        e = 2 if c["dtype"] == "bf16" else 4
        # rows in, codes and scales out; then read again and written as fp32 rows
        return {"bytes": rows * (2 * D * e + 2 * 1.125 * D + 2 * 4 * D), "flops": 0}
    if c["op"] == "attend":
        e = 2 if c["dtype"] == "bf16" else 4
        before, new = _lengths(c)
        pairs = sum(n * b + n * (n + 1) // 2 for b, n in zip(before, new))
        return {"bytes": sum(b + n for b, n in zip(before, new)) * c["kv_heads"] * 1.125 * D + 2 * sum(new) * c["heads"] * D * e,
                "flops": 4 * pairs * c["heads"] * D}
    if c["op"] == "branch":
        got, copies = _new_pages(c)
        shared = c["branches"] * sum(-(-n // c["page"]) for n in _seqs(c))
        return {"bytes": 2 * copies * _page_bytes(c) + 16 * (shared + got), "flops": 0}
    live = sum(-(-n // c["page"]) for n in _seqs(c))
    return {"bytes": 2 * live * _page_bytes(c) + 8 * (live + _pool_pages(c)), "flops": 0}


# ---- the 4-bit rule and the layout of a block, in torch ---------------------------------------------------------------------
def _quantise(x):
    """x [..., D] -> codes (fp32 whole numbers, [..., D/32, 32]) and scales (fp16, [..., D/32, 1])."""
    g = x.float().unflatten(-1, (-1, 32))
    scale = (g.abs().amax(-1, keepdim=True) / 7.0).clamp(max=65504.0).half()
    s = scale.float()
    code = torch.where(s > 0, torch.round(g / torch.where(s > 0, s, torch.ones_like(s))).clamp(-7, 7), torch.zeros_like(g))
    return code, scale


_LAYOUT = {}


def _layout(D, device):
    """Where element (position r of 16, dimension d) of K and of V sits among the nibbles of its codes, and the scale of
    (position r, group) among the scales.  A 16 x 16 tile is 32 words, word 4 * g + t; nibble = 2 * byte + (0 low, 1 high)."""
    key = (D, str(device))
    if key not in _LAYOUT:
        r, d = torch.arange(16)[:, None], torch.arange(D)[None, :]
        G, tile, e = d // 32, d % 32 // 16, d % 16
        word_k = (r % 8) * 4 + e % 8 // 2
        k = (G * 256 + word_k * 8 + tile * 4 + r // 8 + 2 * (e % 2)) * 2 + e // 8
        word_v = (e % 8) * 4 + r % 8 // 2
        v = (G * 256 + word_v * 8 + tile * 4 + r // 8 + 2 * (r % 2)) * 2 + e // 8
        q, grp = torch.arange(16)[:, None], torch.arange(D // 32)[None, :]
        sk = q * (D // 32) + grp
        sv = grp * 16 + q % 8 // 2 * 4 + q // 8 * 2 + q % 2
        _LAYOUT[key] = tuple(x.contiguous().to(device) for x in (k, v, sk, sv))
    return _LAYOUT[key]


def _pack(k, v):
    """k, v [..., 16, D] of whole blocks -> bytes [..., 576 * D / 32]."""
    D = k.shape[-1]
    parts = []
    for x, at, at_scale in zip((k, v), _layout(D, k.device)[:2], _layout(D, k.device)[2:]):
        code, scale = _quantise(x)
        lead = code.shape[:-3]
        nib = torch.empty((*lead, 16 * D), dtype=torch.uint8, device=k.device)
        nib[..., at.reshape(-1)] = (code + 8).to(torch.uint8).reshape(*lead, 16 * D)
        parts.append(nib[..., 0::2] | (nib[..., 1::2] << 4))
        s = torch.empty((*lead, D // 2), dtype=torch.float16, device=k.device)
        s[..., at_scale.reshape(-1)] = scale.reshape(*lead, D // 2)
        parts.append(s.view(torch.uint8))
    return torch.cat(parts, -1)


def _unpack(blocks, D):
    """bytes [..., 576 * D / 32] -> k, v [..., 16, D] in fp32."""
    out, codes, scales = [], 8 * D, D
    for n, (at, at_scale) in enumerate(zip(_layout(D, blocks.device)[:2], _layout(D, blocks.device)[2:])):
        b = blocks[..., n * (codes + scales):]
        c = b[..., :codes]
        nib = torch.stack([c & 15, c >> 4], -1).flatten(-2)[..., at.reshape(-1)].unflatten(-1, (16, D // 32, 32))
        s = b[..., codes:codes + scales].contiguous().view(torch.float16)[..., at_scale.reshape(-1)].unflatten(-1, (16, D // 32, 1))
        out.append(((nib.float() - 8.0) * s.float()).flatten(-2))
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _generator(case, seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed % (1 << 40)) + 17)


def _rows(case, g, shape, values=False):
    """Rows as a model's projections give them: keys with a few channels far larger than the rest, values without."""
    x = torch.randn(shape, generator=g, device="cuda")
    if not values:
        c = torch.rand(shape[-1], generator=g, device="cuda")
        x = x * torch.where(c > 0.95, 4.0, 1.0) + torch.randn(shape[-1], generator=g, device="cuda") * 0.3
    return x if case["dtype"] == "f32" else x.bfloat16()


def _tables(counts, width, n_pages, seqs, g):
    """Page tables of sequences with counts[i] pages each, the pages in random order of a pool of n_pages."""
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    n = torch.tensor(counts + [0] * (seqs - len(counts)), device="cuda")
    col = torch.arange(width, device="cuda")[None, :]
    at = (n.cumsum(0) - n)[:, None] + col
    tables = torch.where(col < n[:, None], order[at.clamp(max=n_pages - 1)], torch.full((), -1, device="cuda", dtype=torch.int32))
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[order[: sum(counts)].long()] = 1
    return tables.int().contiguous(), refs


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _cached(case, g):
    """K and V of every position of an `append` or `attend` case, [batch, blocks, 16, kv_heads, head_dim]."""
    before, new = _lengths(case)
    blocks = max(-(-(b + n) // case["page"]) for b, n in zip(before, new)) * case["page"] // 16
    shape = (case["batch"], blocks, 16, case["kv_heads"], case["head_dim"])
    return _rows(case, g, shape), _rows(case, g, shape, True)


def prepare(case, seed):
    """The pool of a serving program (pages, page tables, lengths, reference counts) and the call's inputs."""
    g = _generator(case, seed)
    if case["op"] in ("branch", "compact"):
        lens = _seqs(case)
        kids = [i for i in range(len(lens)) for _ in range(case["branches"])] if case["op"] == "branch" else []
        n_pages, seqs = _pool_pages(case), len(lens) + len(kids) + 2
        width = -(-(case["ctx"] + case.get("new", 0)) // case["page"]) + 1
        tables, refs = _tables([-(-n // case["page"]) for n in lens], width, n_pages, seqs, g)
        state = dict(case=case, tables=tables, refs=refs, lens=torch.tensor(lens + [0] * (len(kids) + 2), dtype=torch.int32, device="cuda"),
                     pages=torch.randint(0, 256, (n_pages, _page_bytes(case)), generator=g, device="cuda", dtype=torch.uint8))
        if case["op"] == "branch":
            state.update(src=torch.tensor(kids, dtype=torch.int32, device="cuda"),
                         dst=torch.arange(len(lens), len(lens) + len(kids), dtype=torch.int32, device="cuda"),
                         starts=_starts([case["new"]] * len(kids)))
        else:
            # the pool that the live pages move to: a little larger than what they need
            room = sum(-(-n // case["page"]) for n in lens) + 1
            state.update(to=dict(pages=torch.zeros((room, _page_bytes(case)), dtype=torch.uint8, device="cuda"),
                                 tables=torch.full_like(tables, -1), lens=torch.zeros_like(state["lens"]),
                                 refs=torch.zeros(room, dtype=torch.int32, device="cuda")))
        return state
    before, new = _lengths(case)
    B, page, layers = case["batch"], case["page"], case["layers"]
    k, v = _cached(case, g)
    counts = [-(-(b + n) // page) for b, n in zip(before, new)]
    n_pages, seqs = sum(counts) + 2, B + 1
    tables, refs = _tables(counts, k.shape[1] * 16 // page, n_pages, seqs, g)
    slots = torch.randperm(seqs, generator=g, device="cuda")[:B].int()      # the batch's place in the pool, in any order
    by_slot = torch.full_like(tables, -1)
    by_slot[slots.long()] = tables[:B]
    after = torch.tensor([b + n for b, n in zip(before, new)], dtype=torch.int32, device="cuda")
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    lens[slots.long()] = after
    pages = torch.zeros((n_pages, layers, case["kv_heads"], page // 16, 576 * case["head_dim"] // 32), dtype=torch.uint8, device="cuda")
    layer = layers - 1
    for b in range(B):          # sequence by sequence: the quantiser's fp32 copies stay small
        nb = counts[b] * page // 16
        data = _pack(k[b, :nb].transpose(1, 2), v[b, :nb].transpose(1, 2)).unflatten(0, (counts[b], page // 16))
        pages[tables[b, : counts[b]].long(), layer] = data.transpose(1, 2)
    state = dict(case=case, pages=pages.view(n_pages, -1), tables=by_slot, lens=lens, refs=refs, slots=slots, layer=layer,
                 pos=torch.tensor(before, dtype=torch.int32, device="cuda"), starts=_starts(new), max_len=max(b + n for b, n in zip(before, new)),
                 max_new=max(new))
    if case["op"] == "append":
        state.update(zip(("k", "v"), _appended(case, g)))
    else:
        state.update(q=_query(case, g))
    return state


def _appended(case, g):
    shape = (sum(_lengths(case)[1]), case["kv_heads"], case["head_dim"])
    return _rows(case, g, shape), _rows(case, g, shape, True)


def _query(case, g):
    x = torch.randn((sum(_lengths(case)[1]), case["heads"], case["head_dim"]), generator=g, device="cuda") * 1.5
    return x if case["dtype"] == "f32" else x.bfloat16()


# ---- one pass -----------------------------------------------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _pool(state, key="pool", of=None):
    """The framework's handle on the pool: a serving program makes it once."""
    if key not in state:
        from chadslab_b200 import PagedKV4
        c, t = state["case"], of or state
        state[key] = PagedKV4(c["layers"], c["kv_heads"], c["head_dim"], page=c["page"], pages=t["pages"], tables=t["tables"],
                              lens=t["lens"], refs=t["refs"])
    return state[key]


def _own_append(s):
    kv = _pool(s)
    kv.append(s["layer"], s["k"], s["v"], s["slots"], s["pos"], s["starts"])
    return kv.gather(s["layer"], s["slots"], s["pos"], s["starts"], rows=s["k"].shape[0])


def _own_attend(s):
    return _pool(s).attention(s["layer"], s["q"], s["slots"], s["pos"], s["starts"])


def _own_branch(s):
    kv = _pool(s)
    kv.free(s["dst"])
    kv.fork(s["src"], s["dst"])
    pos = kv.extend(s["dst"], s["starts"])
    return pos, kv.tables, kv.lens, kv.refs, kv.pages


def _own_compact(s):
    to = _pool(s, "pool_to", s["to"])
    _pool(s).compact(to)
    return to.tables, to.lens, to.refs, to.pages


_own = dict(append=_own_append, attend=_own_attend, branch=_own_branch, compact=_own_compact)


def _places(s):
    """Sequence, position, page and place in the page of every new row."""
    starts = s["starts"].long()
    n = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=n.device), n)
    at = torch.arange(seq.numel(), device=n.device) - starts[seq] + s["pos"].long()[seq]
    page = s["case"]["page"]
    return seq, at, s["tables"].long()[s["slots"].long()[seq], at // page], at % page


def _view(s):
    c = s["case"]
    return s["pages"].view(-1, c["layers"], c["kv_heads"], c["page"] // 16, 576 * c["head_dim"] // 32)[:, s["layer"]]


def _plain_append(s):
    c = s["case"]
    D, H, T = c["head_dim"], c["kv_heads"], s["k"].shape[0]
    _, _, page, at = _places(s)
    view = _view(s)
    block, r, head = (at // 16)[:, None, None], at % 16, torch.arange(H, device=at.device)[None, :, None]
    back = []
    for n, x in enumerate((s["k"], s["v"])):
        where, where_scale = _layout(D, x.device)[n][r][:, None, :], _layout(D, x.device)[2 + n][r][:, None, :]
        code, scale = _quantise(x)
        back.append((code * scale.float()).flatten(-2))
        code = (code + 8).to(torch.uint8).flatten(-2)
        first = n * 9 * D
        # a byte holds two nibbles of one row: elements d and d + 8 of a 16-wide tile
        low, pair = code.unflatten(-1, (-1, 2, 8))[..., 0, :].flatten(-2), code.unflatten(-1, (-1, 2, 8))[..., 1, :].flatten(-2)
        byte = where.unflatten(-1, (-1, 2, 8))[..., 0, :].flatten(-2) // 2
        view[page[:, None, None], head, block, first + byte] = low | (pair << 4)
        two = scale.reshape(T, H, D // 32, 1).view(torch.uint8)
        at_byte = first + 8 * D + 2 * where_scale[..., None] + torch.arange(2, device=x.device)
        view[page[:, None, None, None], head[..., None], block[..., None], at_byte] = two
    return tuple(back)


def _plain_attend(s):
    c = s["case"]
    D, H, Q, page = c["head_dim"], c["kv_heads"], c["heads"], c["page"]
    B, N = s["slots"].numel(), s["max_new"]
    width = -(-s["max_len"] // page)
    table = s["tables"].long()[s["slots"].long(), :width].clamp(min=0)
    k, v = _unpack(_view(s)[table].transpose(2, 3).flatten(1, 2), D)         # [B, blocks, H, 16, D]
    k, v = (x.transpose(2, 3).flatten(1, 2).transpose(1, 2) for x in (k, v))   # [B, H, S, D]
    seq, at, _, _ = _places(s)
    i = at - s["pos"].long()[seq]
    q = torch.zeros((B, N, Q, D), device=k.device)
    q[seq, i] = s["q"].float()
    q = q.view(B, N, H, Q // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, Q // H * N, D)
    seen = torch.arange(k.shape[2], device=k.device)[None, None, :] <= (s["pos"].long()[:, None] + torch.arange(N, device=k.device))[:, :, None]
    score = (q @ k.transpose(-1, -2)).view(B, H, Q // H, N, -1) / math.sqrt(D)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(B, H, Q // H * N, -1) @ v).view(B, H, Q // H, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Q, D)
    return o[seq, i].to(s["q"].dtype)


def _plain_branch(s):
    tables, lens, refs, pages, page = s["tables"], s["lens"], s["refs"], s["pages"], s["case"]["page"]
    src, dst = s["src"].long(), s["dst"].long()

    def count(rows, by):
        rows = rows.reshape(-1)
        live = (rows >= 0).int() * by
        refs.index_add_(0, rows.clamp(min=0).long(), live.int())
    count(tables[dst], -1)                                   # free
    tables[dst], lens[dst] = -1, 0
    taken = tables[src]                                      # fork
    count(taken, 1)
    tables[dst], lens[dst] = taken, lens[src]
    pos = lens[dst]                                          # extend
    n = s["starts"][1:] - s["starts"][:-1]
    had, has = -(-pos // page), -(-(pos + n) // page)
    last = taken.gather(1, (had - 1).clamp(min=0).long()[:, None])[:, 0]
    cow = ((pos % page != 0) & (n > 0) & (refs[last.long()] > 1)).int()
    need = has - had + cow
    free = torch.nonzero(refs == 0)[:, 0].int()
    col = torch.arange(tables.shape[1], device=pos.device)[None, :]
    j = col - (had - cow)[:, None]
    mine = (j >= 0) & (j < need[:, None])
    new = free[((need.cumsum(0) - need)[:, None] + j).clamp(0, free.numel() - 1).long()]
    tables[dst] = torch.where(mine, new, taken)
    refs[new[mine].long()] = 1
    copied = cow.bool()
    to = tables[dst].gather(1, (had - 1).clamp(min=0).long()[:, None])[:, 0]
    pages[to[copied].long()] = pages[last[copied].long()]
    count(last[copied], -1)
    lens[dst] = pos + n.int()
    return pos, tables, lens, refs, pages


def _plain_compact(s):
    to = s["to"]
    live = torch.nonzero(s["refs"] > 0)[:, 0]
    place = torch.full_like(s["refs"], -1)
    place[live] = torch.arange(live.numel(), dtype=torch.int32, device=live.device)
    to["pages"][: live.numel()] = s["pages"][live]
    to["refs"].zero_()
    to["refs"][: live.numel()] = s["refs"][live]
    to["tables"].copy_(torch.where(s["tables"] >= 0, place[s["tables"].clamp(min=0).long()], -1))
    to["lens"].copy_(s["lens"])
    return to["tables"], to["lens"], to["refs"], to["pages"]


_plain = dict(append=_plain_append, attend=_plain_attend, branch=_plain_branch, compact=_plain_compact)


# ---- the same in 64 bits, from the definition ---------------------------------------------------------------------------------
def _held(x):
    """What 4 bits hold of rows x: in groups of 32, multiples of fp16(absmax / 7) up to 7 of them."""
    x = x.double().unflatten(-1, (-1, 32))
    step = torch.clamp((x.abs().amax(-1, keepdim=True).float() / 7), max=65504).half().double()
    # x / step is rounded to fp32 before it is rounded to a whole number: part of the definition
    times = (x / step).float().double().round().clamp(-7, 7)
    return torch.where(step > 0, times * step, torch.zeros_like(x)).flatten(-2)


def exact(case, seed):
    if case["op"] in ("branch", "compact"):
        return None                                          # whole numbers only
    g = _generator(case, seed)
    k, v = _cached(case, g)
    before, new = _lengths(case)
    counts = [-(-(b + n) // case["page"]) for b, n in zip(before, new)]
    torch.randperm(sum(counts) + 2, generator=g, device="cuda")   # prepare draws the tables and slots here
    torch.randperm(case["batch"] + 1, generator=g, device="cuda")
    if case["op"] == "append":
        return tuple(_held(x) for x in _appended(case, g))
    if 4 * sum((b + n) * n for b, n in zip(before, new)) * case["heads"] * case["head_dim"] > 4e12:
        return None
    q, rows, first = _query(case, g).double(), [], 0
    for b in range(case["batch"]):
        n, end = new[b], before[b] + new[b]
        K, V = (_held(x[b].flatten(0, 1)[:end]).transpose(0, 1) for x in (k, v))       # [H, end, D]
        one = q[first:first + n].unflatten(1, (case["kv_heads"], -1)).permute(1, 2, 0, 3)   # [H, rep, n, D]
        w = torch.einsum("hrnd,hsd->hrns", one, K) * case["head_dim"] ** -0.5
        hidden = torch.arange(end, device="cuda")[None, :] > torch.arange(before[b], end, device="cuda")[:, None]
        w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
        rows.append(torch.einsum("hrns,hsd->nhrd", w, V).flatten(1, 2))
        first += n
    return torch.cat(rows)
