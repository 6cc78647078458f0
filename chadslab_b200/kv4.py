"""Paged KV cache held in 4 bits (codes in groups of 32 along head_dim with an fp16 scale each), and attention over it.

    kv = PagedKV4(layers, kv_heads, head_dim, n_pages=..., max_seqs=..., max_pages=...)
    pos = kv.extend(slots, starts)                     room for new rows: once per step, for all layers
    kv.append(layer, k, v, slots, pos, starts)         quantise rows into the pages
    out = kv.attention(layer, q, slots, pos, starts)   causal attention of those rows over everything before them
    kv.fork(src, dst); kv.free(slots)                  share a prefix, end a sequence
    kv.compact(other)                                  move the live pages into a pool of another size

Token rows are [n_rows, heads, head_dim]; `starts` (int32 [B + 1]) gives the rows of every sequence of the batch, None means
one row per sequence.  `slots` (int32 [B], None: 0 .. B-1) are rows of the page table, `pos` (int32 [B]) the position of every
sequence's first row, as `extend` returns it (-1: refused, no pages left).  All three are CUDA tensors, or sequences of ints, which
are copied to the device.  Nothing here waits for the GPU.  Calls whose arguments are tensors can be captured in a graph; a
sequence of ints is refused during capture, since a replay would read host memory that is gone.  Calls that change a pool are to
be ordered on the device, like the library's other calls; compact counts as one for both pools.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import BqError, DT_BF16, DT_F32

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class PagedKV4:
    """A pool of 4-bit KV pages, its page tables, lengths and reference counts (all on one device)."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, n_pages: int = 0, max_seqs: int = 0, max_pages: int = 0, page: int = 64,
                 device=None, *, pages=None, tables=None, lens=None, refs=None):
        """Allocates an empty pool of n_pages pages for max_seqs sequences of up to max_pages pages, or adopts the given
        tensors: pages uint8 (n_pages * page_bytes of them), tables int32 [max_seqs, max_pages], lens int32 [max_seqs],
        refs int32 [n_pages]."""
        given = (pages, tables, lens, refs)
        if any(t is not None for t in given):
            if any(t is None for t in given):
                raise ValueError("give all of pages, tables, lens and refs, or none")
            if pages.dtype != torch.uint8 or any(t.dtype != torch.int32 for t in (tables, lens, refs)):
                raise TypeError("pages must be uint8; tables, lens and refs int32")
            if not all(t.is_cuda and t.is_contiguous() and t.device == pages.device for t in given):
                raise BqError(_lib.ERR_ARG, "pages, tables, lens and refs must be contiguous tensors on one CUDA device")
            n_pages = refs.numel()
            if tables.dim() != 2 or lens.numel() != tables.shape[0]:
                raise ValueError("tables must be [max_seqs, max_pages] and lens [max_seqs]")
            max_seqs, max_pages = tables.shape
            device = pages.device
        else:
            device = torch.device(device if device is not None else "cuda")
            if device.type != "cuda":
                raise BqError(_lib.ERR_ARG, "the pool lives on a CUDA device")
            if device.index is None:
                device = torch.device("cuda", torch.cuda.current_device() if torch.cuda.is_available() else 0)
        self.layers, self.kv_heads, self.head_dim, self.page = int(layers), int(kv_heads), int(head_dim), int(page)
        self.n_pages, self.max_seqs, self.max_pages, self.device = int(n_pages), int(max_seqs), int(max_pages), device
        if self.head_dim <= 0 or self.head_dim % 32 or self.head_dim > 256:
            raise ValueError(f"head_dim={head_dim} must be a multiple of 32 up to 256")
        if not 16 <= self.page <= 4096 or self.page & (self.page - 1):
            raise ValueError(f"page={page} must be a power of two from 16 to 4096 positions")
        if min(self.layers, self.kv_heads, self.n_pages, self.max_seqs, self.max_pages) <= 0:
            raise ValueError("layers, kv_heads, n_pages, max_seqs and max_pages must be positive")
        if self.max_seqs > 8192 or self.max_pages * self.page > 1 << 30 or self.n_pages >= 1 << 30:
            raise ValueError("a pool holds at most 8192 sequences of 2^30 positions, in fewer than 2^30 pages")
        self._index = device.index or 0
        self._lib = lib = _lib.init(self._index)
        self._pool = _lib.Kv4Pool(None, None, None, None, None, self.n_pages, self.max_seqs, self.max_pages, self.layers, self.kv_heads,
                                  self.head_dim, self.page)
        self._p = C.byref(self._pool)
        self.page_bytes = int(lib.bq_kv4_page_bytes(self._p))
        if pages is None:
            pages = torch.empty((self.n_pages, self.page_bytes), dtype=torch.uint8, device=device)
            tables = torch.full((self.max_seqs, self.max_pages), -1, dtype=torch.int32, device=device)
            lens = torch.zeros(self.max_seqs, dtype=torch.int32, device=device)
            refs = torch.zeros(self.n_pages, dtype=torch.int32, device=device)
        elif pages.numel() != self.n_pages * self.page_bytes:
            raise ValueError(f"{self.n_pages} pages take {self.n_pages * self.page_bytes} bytes, got {pages.numel()}")
        self.pages, self.tables, self.lens, self.refs = pages, tables, lens, refs
        self._work = torch.empty(int(lib.bq_kv4_work_bytes(self._p)) // 4, dtype=torch.int32, device=device)
        p = self._pool
        p.pages, p.tables, p.lens, p.refs, p.work = (t.data_ptr() for t in (pages, tables, lens, refs, self._work))
        self.changes = 0                     # calls that may have changed the sequences, replays of captured ones apart
        self._attn_ints = {}                 # scratch of an attention call by (heads, dtype, sequences, rows)

    # ---- arguments --------------------------------------------------------------------------------------------------
    def _ints(self, t, what: str):
        """-> int32 CUDA tensor on the pool's device (a sequence of ints is copied there)."""
        if not isinstance(t, torch.Tensor):
            if self.device.type != "cuda":
                return torch.tensor(t, dtype=torch.int32)
            if torch.cuda.is_current_stream_capturing():
                raise BqError(_lib.ERR_STATE, f"{what} must be an int32 tensor on {self.device} during stream capture")
            return torch.tensor(t, dtype=torch.int32, pin_memory=True).to(self.device, non_blocking=True)      # the host does not wait
        if t.dtype is not torch.int32 or t.device != self.device or t.dim() != 1:
            raise BqError(_lib.ERR_ARG, f"{what} must be a 1-D int32 tensor on {self.device}")
        return t if t.is_contiguous() else t.contiguous()

    def _stream(self) -> int:
        if torch.cuda.current_device() != self._index:
            raise BqError(_lib.ERR_STATE, f"the pool is on {self.device}, the current device is {torch.cuda.current_device()}")
        return _raw_stream(self._index)

    def _batch(self, slots, pos, starts):
        """-> (slots, pos, starts) on the device, their addresses, B; the tensors are to be kept until the call is made."""
        pos = self._ints(pos, "pos")
        B = pos.numel()
        at_slots = at_starts = None
        if slots is not None:
            slots = self._ints(slots, "slots")
            if slots.numel() != B:
                raise ValueError(f"{slots.numel()} slots for {B} positions")
            at_slots = slots.data_ptr()
        if starts is not None:
            starts = self._ints(starts, "starts")
            if starts.numel() != B + 1:
                raise ValueError(f"starts must have one entry more than pos ({B}), got {starts.numel()}")
            at_starts = starts.data_ptr()
        return (slots, pos, starts), at_slots, pos.data_ptr(), at_starts, B

    @staticmethod
    def _ptr(t):
        return None if t is None else t.data_ptr()

    def _rows(self, x, heads: int, what: str):
        """[n_rows, heads, head_dim] whose rows are dense (a slice of a fused projection is; anything else is copied)."""
        if x.device != self.device:
            raise BqError(_lib.ERR_ARG, f"{what} must be a CUDA tensor on {self.device}")
        if x.dtype not in _DT:
            raise TypeError(f"{what} must be float32 or bfloat16, got {x.dtype}")
        D = self.head_dim
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != D:
            raise ValueError(f"{what} must be [n_rows, {heads}, {D}], got {tuple(shape)}")
        dense = heads * D
        s0, s1, s2 = x.stride()
        if shape[0] <= 1:
            s0 = dense
        if s0 < dense or s0 & 7 or s2 != 1 or (s1 != D and heads > 1) or x.data_ptr() & 15:
            x, s0 = x.clone(memory_format=torch.contiguous_format), dense
        return x, s0

    # ---- pages --------------------------------------------------------------------------------------------------------
    def extend(self, slots=None, starts=None, batch: int | None = None):
        """Room for every sequence's new rows (starts None: one each) -> pos int32 [B], the length before, -1 where fewer pages
        were left than the sequence needs (later ones of the batch are served all the same).  `batch` has to give B when both are None."""
        if slots is None and starts is None and batch is None:
            raise ValueError("extend needs slots, starts or batch")
        if slots is not None:
            slots = self._ints(slots, "slots")
        if starts is not None:
            starts = self._ints(starts, "starts")
            if starts.numel() == 0:
                raise ValueError("starts must have one entry more than there are sequences")
        B = slots.numel() if slots is not None else starts.numel() - 1 if starts is not None else int(batch)
        if starts is not None and starts.numel() != B + 1:
            raise ValueError(f"starts must have one entry more than slots ({B}), got {starts.numel()}")
        self.changes += 1
        pos = self.lens.new_empty(B)
        _lib.check(self._lib.bq_kv4_extend(self._p, self._ptr(slots), self._ptr(starts), B, pos.data_ptr(), self._stream()))
        return pos

    def fork(self, src, dst) -> None:
        """Sequence dst[i] becomes a copy of src[i] that shares its pages; what it held before is given up."""
        src, dst = self._ints(src, "src"), self._ints(dst, "dst")
        if src.numel() != dst.numel():
            raise ValueError(f"{src.numel()} sources for {dst.numel()} destinations")
        self.changes += 1
        _lib.check(self._lib.bq_kv4_fork(self._p, src.data_ptr(), dst.data_ptr(), src.numel(), self._stream()))

    def free(self, slots) -> None:
        """Empties sequences; pages that no other sequence holds become free."""
        slots = self._ints(slots, "slots")
        self.changes += 1
        _lib.check(self._lib.bq_kv4_free(self._p, slots.data_ptr(), slots.numel(), self._stream()))

    def compact(self, to: "PagedKV4") -> "PagedKV4":
        """Moves a copy of all live pages, in ascending order, and the sequences into pool `to`; returns it.  How many pages are
        live is known on the device alone: if `to` has fewer, it stays as it was and BQ_ERR_STATE is recorded in the
        status word (bq_status_poll)."""
        if to.device != self.device:
            raise BqError(_lib.ERR_ARG, f"both pools must be on {self.device}")
        to.changes += 1
        _lib.check(self._lib.bq_kv4_compact(self._p, to._p, self._stream()))
        return to

    # ---- rows ---------------------------------------------------------------------------------------------------------
    def append(self, layer: int, k, v, slots, pos, starts=None) -> None:
        """Quantise rows k, v [n_rows, kv_heads, head_dim] (fp32 or bf16) into their positions."""
        keep, at_slots, at_pos, at_starts, B = self._batch(slots, pos, starts)
        k, ldk = self._rows(k, self.kv_heads, "k")
        v, ldv = self._rows(v, self.kv_heads, "v")
        if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
            raise ValueError("k and v must have the same type and number of rows")
        _lib.check(self._lib.bq_kv4_append(self._p, int(layer), k.data_ptr(), v.data_ptr(), ldk, ldv, _DT[k.dtype], at_slots, at_pos,
                                           at_starts, B, k.shape[0], self._stream()))

    def rope_append(self, layer: int, qkv, heads: int, rope_base: float, slots, pos, starts=None, q_out=None, dtype=torch.bfloat16):
        """qkv fp32 [n_rows, (heads + 2 kv_heads) head_dim] of a fused projection: rotates q and k by each row's position,
        quantises k and v into the pages -> q [n_rows, heads, head_dim] in `dtype` (or q_out).  Rows of refused sequences, or
        of none, are not written: as allocated, or as they were in q_out."""
        keep, at_slots, at_pos, at_starts, B = self._batch(slots, pos, starts)
        if q_out is None and dtype not in _DT:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        if not qkv.is_cuda or qkv.device != self.device or qkv.dtype != torch.float32 or not qkv.is_contiguous():
            raise BqError(_lib.ERR_ARG, f"qkv must be a contiguous fp32 tensor on {self.device}")
        width = (heads + 2 * self.kv_heads) * self.head_dim
        if qkv.dim() != 2 or qkv.shape[1] != width:
            raise ValueError(f"qkv must be [n_rows, {width}], got {tuple(qkv.shape)}")
        if q_out is None:
            q_out = torch.empty((qkv.shape[0], heads, self.head_dim), dtype=dtype, device=self.device)
        elif (q_out.dtype not in _DT or q_out.device != self.device or not q_out.is_contiguous()
              or q_out.numel() != qkv.shape[0] * heads * self.head_dim):
            raise ValueError("q_out must be a contiguous fp32 or bf16 tensor of n_rows * heads * head_dim elements on the pool's device")
        _lib.check(self._lib.bq_kv4_rope_append(self._p, int(layer), qkv.data_ptr(), q_out.data_ptr(), int(heads), float(rope_base),
                                                _DT[q_out.dtype], at_slots, at_pos, at_starts, B, qkv.shape[0], self._stream()))
        return q_out

    def gather(self, layer: int, slots, pos, starts=None, rows: int | None = None, dtype=torch.float32):
        """What the pages hold (code * scale) of the positions that the rows stand for -> k, v [n_rows, kv_heads, head_dim];
        where `starts` is given, `rows` has to say how many they are (it is on the device).  Rows of refused sequences, or of none, are left as allocated."""
        keep, at_slots, at_pos, at_starts, B = self._batch(slots, pos, starts)
        if dtype not in _DT:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        if starts is not None and rows is None:
            raise ValueError("gather with starts needs rows, the number of rows they stand for")
        n_rows = int(rows) if starts is not None else B
        shape = (n_rows, self.kv_heads, self.head_dim)
        k, v = self.lens.new_empty(shape, dtype=dtype), self.lens.new_empty(shape, dtype=dtype)
        _lib.check(self._lib.bq_kv4_gather(self._p, int(layer), k.data_ptr(), v.data_ptr(), _DT[dtype], at_slots, at_pos, at_starts, B, n_rows,
                                           self._stream()))
        return k, v

    def attention(self, layer: int, q, slots, pos, starts=None, out=None):
        """softmax(q . K^T / sqrt(head_dim)) . V for rows q [n_rows, heads, head_dim] (fp32 or bf16) of the sequences, each
        row over the positions up to its own -> [n_rows, heads, head_dim].  Rows of refused sequences are zero; rows behind
        the last sequence are left as they were."""
        keep, at_slots, at_pos, at_starts, B = self._batch(slots, pos, starts)
        if q.dim() != 3 or q.shape[1] % self.kv_heads:
            raise ValueError(f"q must be [n_rows, heads, head_dim] with a multiple of {self.kv_heads} heads, got {tuple(q.shape)}")
        heads = q.shape[1]
        q, ldq = self._rows(q, heads, "q")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.dtype != q.dtype or out.device != self.device or not out.is_contiguous() or out.shape != q.shape:
            raise ValueError("out must be a contiguous tensor like q")
        dt = _DT[q.dtype]
        sizes = (heads, dt, B, q.shape[0])
        need = self._attn_ints.get(sizes)
        if need is None:
            if len(self._attn_ints) >= 256:              # a server's chunks come in any size
                self._attn_ints.clear()
            need = self._attn_ints[sizes] = int(self._lib.bq_kv4_attention_work_bytes(self._p, *sizes)) // 4
        work = self.refs.new_empty(need)                       # of this call alone: calls may overlap
        _lib.check(self._lib.bq_kv4_attention(self._p, int(layer), q.data_ptr(), ldq, out.data_ptr(), heads, dt, at_slots, at_pos, at_starts, B,
                                              q.shape[0], work.data_ptr(), self._stream()))
        return out
