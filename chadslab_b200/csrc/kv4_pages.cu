// Pages of the 4-bit KV cache: allocation (extend, with the copy of a shared page that is about to be written), sharing
// (fork), release (free) and moving into another pool (compact).  All bookkeeping stays on the device - page tables,
// lengths and reference counts - so that the calls can sit in a captured graph between decode steps.
//
// The plans (which page goes where) are made by one CTA and are deterministic: pages are given out lowest number first, in
// batch order.  The bytes are moved by a second, grid-wide kernel that reads the plan.
#include "kv4.cuh"

namespace bq {

constexpr int KP_THREADS = 1024;
constexpr int KP_LARGE = 1 << 20;                         // pages: 1024 such needs fit into 31 bits
constexpr int KP_PER = 16;                                // reference counts a thread looks at per pass (four 16-byte loads)

// ---- workspace (int32) -------------------------------------------------------------------------------------------------
//   [0] number of page copies of the plan (-1: refused)       [1..31] unused
//   list   n_pages              free pages found / live pages in ascending order
//   place  n_pages              compact: the new number of every page (-1: free)
//   pairs  2 * max_seqs         extend: copies (from, to); its per-sequence needs before that
//   rows   max_seqs * (max_pages + 1)   fork: length and table row of every pair, as they were before the call
struct KpWork {
  int32_t *head, *list, *place, *pairs, *rows;
};
static __host__ __device__ KpWork kp_work(int32_t* w, int64_t n_pages, int max_seqs) {
  KpWork k;
  k.head = w;
  k.list = w + 32;
  k.place = k.list + n_pages;
  k.pairs = k.place + n_pages;
  k.rows = k.pairs + 2 * (int64_t)max_seqs;
  return k;
}
static int64_t kp_work_ints(const bq_kv4_pool* p) {
  return 32 + 2 * p->n_pages + 2 * (int64_t)p->max_seqs + (int64_t)p->max_seqs * ((int64_t)p->max_pages + 1);
}

struct KpPool {
  int32_t *tables, *lens, *refs, *work;
  int64_t n_pages;
  int max_seqs, max_pages, page_log2;
};

// inclusive sum over the block; *total = the block's sum.  `red` holds 32 ints of shared memory.
__device__ __forceinline__ int kp_scan(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  __syncthreads();                                   // red may still be read from the previous call
  if (lane == 31) red[warp] = v;
  __syncthreads();
  int w = red[lane];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, w, off);
    if (lane >= off) w += o;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return v + (warp > 0 ? before : 0);
}

// Lists the pages whose reference count is zero (LIVE false) or not (LIVE true), ascending, until `want` of them are
// found; returns how many were.  `place` (optional) receives each page's position in the list, -1 for the others.
template <bool LIVE>
__device__ int kp_list(const int32_t* refs, int64_t n_pages, int want, int32_t* list, int32_t* place, int* red) {
  int found = 0;
  for (int64_t base = 0; base < n_pages && found < want; base += KP_THREADS * KP_PER) {
    const int64_t i0 = base + (int64_t)threadIdx.x * KP_PER;
    int32_t r[KP_PER];
    if (i0 + KP_PER <= n_pages) {
#pragma unroll
      for (int j = 0; j < KP_PER / 4; ++j) {
        const int4 q = reinterpret_cast<const int4*>(refs + i0)[j];
        r[4 * j] = q.x; r[4 * j + 1] = q.y; r[4 * j + 2] = q.z; r[4 * j + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < KP_PER; ++j) r[j] = i0 + j < n_pages ? refs[i0 + j] : (LIVE ? 0 : 1);
    }
    int n = 0;
#pragma unroll
    for (int j = 0; j < KP_PER; ++j) n += (r[j] > 0) == LIVE;
    int total;
    int at = found + kp_scan(n, red, &total) - n;
#pragma unroll
    for (int j = 0; j < KP_PER; ++j) {
      const bool hit = (r[j] > 0) == LIVE;
      if (hit && at < want) list[at] = (int32_t)(i0 + j);
      if (place && i0 + j < n_pages) place[i0 + j] = hit ? at : -1;
      at += hit;
    }
    found += total;
  }
  return found < want ? found : want;
}

// One CTA.  need(b) = pages that sequence b lacks for n more rows, one more if its last page is partly filled and shared.
__global__ void __launch_bounds__(KP_THREADS) kv4_extend_kernel(KpPool p, const int32_t* slots, const int32_t* starts,
                                                                int B, int32_t* pos_out, int* status) {
  extern __shared__ int owner[];                     // first batch entry that names a slot
  __shared__ int red[32];
  __shared__ int s_copies, s_large;
  pdl_launch_dependents();
  pdl_wait();
  const KpWork w = kp_work(p.work, p.n_pages, p.max_seqs);
  const int64_t room = (int64_t)p.max_pages << p.page_log2;
  const int page = 1 << p.page_log2;
  for (int i = threadIdx.x; i < p.max_seqs; i += KP_THREADS) owner[i] = B;
  if (threadIdx.x == 0) s_copies = s_large = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < B; b += KP_THREADS) {
    const int s = slots ? slots[b] : b;
    if ((unsigned)s < (unsigned)p.max_seqs) atomicMin(&owner[s], b);
  }
  __syncthreads();
  // what each sequence lacks; pairs[2 b] = pages, pairs[2 b + 1] = pages of the sequences before it (-1: refused)
  int64_t total = 0;
  for (int b0 = 0; b0 < B; b0 += KP_THREADS) {
    const int b = b0 + (int)threadIdx.x;
    int need = 0, ok = 0;
    if (b < B) {
      const int s = slots ? slots[b] : b;
      const int64_t n = starts ? (int64_t)starts[b + 1] - starts[b] : 1;
      if ((unsigned)s < (unsigned)p.max_seqs && owner[s] == b && n >= 0) {
        const int64_t len = p.lens[s];
        ok = len >= 0 && len + n <= room;
        if (ok && n > 0) {
          const int had = (int)((len + page - 1) >> p.page_log2), has = (int)((len + n + page - 1) >> p.page_log2);
          need = has - had;
          if (len & (page - 1)) {
            const int last = p.tables[(int64_t)s * p.max_pages + had - 1];
            if ((unsigned)last >= (uint64_t)p.n_pages) { ok = 0; need = 0; }
            else need += p.refs[last] > 1;
          }
        }
      }
      if (!ok) *(volatile int*)status = (int)BQ_ERR_ARG;
    }
    // what a call asks for can pass 2^31 pages even if the pool cannot: needs of 2^20 and more take the pass below
    if (need > KP_LARGE) s_large = 1;
    const int sum = need < KP_LARGE ? need : KP_LARGE;
    int chunk;
    const int64_t before = total + kp_scan(sum, red, &chunk) - sum;
    if (b < B) {
      w.pairs[2 * b] = need;
      w.pairs[2 * b + 1] = !ok ? -1 : before < p.n_pages ? (int)before : (int)p.n_pages;
    }
    total += chunk;
  }
  __syncthreads();
  if (s_large) total = p.n_pages + 1;
  int found = 0;
  if (total > 0) found = kp_list<false>(p.refs, p.n_pages, (int)(total < p.n_pages ? total : p.n_pages), w.list, nullptr, red);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  if (total > found) {
    // Not all can be served.  A sequence that needs more than is left is refused and changes nothing; the ones behind it
    // have what it did not get.
    if (threadIdx.x < 32) {
      int taken = 0;
      for (int b0 = 0; b0 < B; b0 += 32) {
        const int b = b0 + lane, need = b < B ? w.pairs[2 * b] : 0;
        int at = b < B ? w.pairs[2 * b + 1] : -1;
        for (int j = 0; j < 32; ++j) {
          const int n = __shfl_sync(0xffffffffu, at >= 0 ? need : 0, j);
          const bool fits = n <= found - taken;
          if (lane == j && at >= 0) at = fits ? taken : -1;
          if (fits) taken += n;
        }
        if (b < B) w.pairs[2 * b + 1] = at;
      }
    }
    __syncthreads();
  }
  for (int b0 = 0; b0 < B; b0 += KP_THREADS / 32) {
    const int b = b0 + (int)(threadIdx.x >> 5);
    int from = -1, to = -1;
    if (b < B) {
      const int need = w.pairs[2 * b], at = w.pairs[2 * b + 1];
      if (at < 0) {
        if (lane == 0) pos_out[b] = -1;
      } else {
        const int s = slots ? slots[b] : b;
        const int n = starts ? starts[b + 1] - starts[b] : 1;
        const int len = p.lens[s];
        const int had = (len + page - 1) >> p.page_log2, has = (int)(((int64_t)len + n + page - 1) >> p.page_log2);
        const int cow = need - (has - had);                              // 0 or 1
        int32_t* row = p.tables + (int64_t)s * p.max_pages + had - cow;
        if (cow) { from = row[0]; to = w.list[at]; }
        __syncwarp();
        for (int j = lane; j < need; j += 32) {
          const int id = w.list[at + j];
          row[j] = id;
          p.refs[id] = 1;
        }
        __syncwarp();
        if (lane == 0) {
          pos_out[b] = len;
          p.lens[s] = len + n;
          if (cow) atomicSub(&p.refs[from], 1);
        }
      }
    }
    // pairs of the plan overwrite the needs of sequences that every warp has read already
    __syncthreads();
    if (to >= 0 && lane == 0) {
      const int c = atomicAdd(&s_copies, 1);
      w.pairs[2 * c] = from;
      w.pairs[2 * c + 1] = to;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) w.head[0] = s_copies;
}

// ---- moving bytes ------------------------------------------------------------------------------------------------------
// Copies `head[0]` pages of page_bytes (a multiple of 16): from pairs (from, to), or, with COMPACT, page list[i] of the
// source to page i of the destination, and then the tables, lengths and reference counts of the destination.
constexpr int KC_THREADS = 256;
constexpr int KC_UNROLL = 8;
constexpr int KC_CHUNK = KC_THREADS * KC_UNROLL * 16;              // bytes of one work unit: 32 KB
template <bool COMPACT>
__global__ void __launch_bounds__(KC_THREADS) kv4_copy_kernel(KpPool p, const uint8_t* src, uint8_t* dst,
                                                              int64_t page_bytes, KpPool q) {
  pdl_launch_dependents();
  pdl_wait();
  const KpWork w = kp_work(p.work, p.n_pages, p.max_seqs);
  const int n = w.head[0];
  if (n < 0) return;                                                  // the plan was refused
  const int64_t per = (page_bytes + KC_CHUNK - 1) / KC_CHUNK;
  for (int64_t u = blockIdx.x; u < n * per; u += gridDim.x) {
    const int64_t i = u / per, off = (u - i * per) * KC_CHUNK;
    const int64_t from = COMPACT ? w.list[i] : w.pairs[2 * i], to = COMPACT ? i : w.pairs[2 * i + 1];
    const uint8_t* s = src + from * page_bytes + off;
    uint8_t* d = dst + to * page_bytes + off;
    const int64_t left = page_bytes - off;
    uint4 v[KC_UNROLL];
#pragma unroll
    for (int j = 0; j < KC_UNROLL; ++j) {
      const int at = (j * KC_THREADS + (int)threadIdx.x) * 16;
      if (at < left) v[j] = kv4_load16(s + at);
    }
#pragma unroll
    for (int j = 0; j < KC_UNROLL; ++j) {
      const int at = (j * KC_THREADS + (int)threadIdx.x) * 16;
      if (at < left) *reinterpret_cast<uint4*>(d + at) = v[j];
    }
  }
  if (COMPACT) {
    const int64_t t0 = blockIdx.x * (int64_t)KC_THREADS + threadIdx.x, step = (int64_t)gridDim.x * KC_THREADS;
    const int64_t entries = (int64_t)p.max_seqs * p.max_pages;
    for (int64_t i = t0; i < entries; i += step) {
      const int id = p.tables[i];
      q.tables[i] = (unsigned)id < (uint64_t)p.n_pages ? w.place[id] : -1;
    }
    for (int64_t i = t0; i < q.n_pages; i += step) q.refs[i] = i < n ? p.refs[w.list[i]] : 0;
    for (int64_t i = t0; i < p.max_seqs; i += step) q.lens[i] = p.lens[i];
  }
}

__global__ void __launch_bounds__(KP_THREADS) kv4_compact_plan_kernel(KpPool p, int64_t room, int* status) {
  __shared__ int red[32];
  pdl_launch_dependents();
  pdl_wait();
  const KpWork w = kp_work(p.work, p.n_pages, p.max_seqs);
  const int live = kp_list<true>(p.refs, p.n_pages, (int)p.n_pages, w.list, w.place, red);
  if (threadIdx.x == 0) {
    w.head[0] = live <= room ? live : -1;
    if (live > room) *(volatile int*)status = (int)BQ_ERR_STATE;
  }
}

// ---- fork / free ---------------------------------------------------------------------------------------------------------
constexpr int KF_THREADS = 128;
__device__ __forceinline__ int kp_pages_of(const KpPool& p, int len) {
  const int64_t n = ((int64_t)(len > 0 ? len : 0) + (1 << p.page_log2) - 1) >> p.page_log2;
  return (int)(n < p.max_pages ? n : p.max_pages);
}
// gives up n pages of a table row; the threads are `first`, `first` + `step`, ...
__device__ __forceinline__ void kp_release(const KpPool& p, int32_t* row, int n, int first, int step, int* status) {
  for (int j = first; j < n; j += step) {
    const int id = row[j];
    if ((unsigned)id < (uint64_t)p.n_pages) atomicSub(&p.refs[id], 1);
    else *(volatile int*)status = (int)BQ_ERR_ARG;
    row[j] = -1;
  }
}
// First half of a fork: every source is read, and its pages counted once more, before any destination changes.
// `later`: the destination occurs again behind this pair (the last pair counts).
__device__ __forceinline__ void kp_fork_read(const KpPool& p, int s, int d, bool later, int32_t* keep, int first, int step, int* status) {
  const bool ok = (unsigned)s < (unsigned)p.max_seqs && (unsigned)d < (unsigned)p.max_seqs;
  if (!ok || later) {
    if (first == 0) {
      keep[0] = -1;
      if (!ok) *(volatile int*)status = (int)BQ_ERR_ARG;
    }
    return;
  }
  const int len = p.lens[s] > 0 ? p.lens[s] : 0, np = kp_pages_of(p, len);
  const int32_t* row = p.tables + (int64_t)s * p.max_pages;
  for (int j = first; j < np; j += step) {
    const int id = row[j];
    keep[1 + j] = id;
    if ((unsigned)id < (uint64_t)p.n_pages) atomicAdd(&p.refs[id], 1);
    else *(volatile int*)status = (int)BQ_ERR_ARG;
  }
  if (first == 0) keep[0] = len;
}
__global__ void __launch_bounds__(KF_THREADS) kv4_fork_read_kernel(KpPool p, const int32_t* src, const int32_t* dst, int n, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const KpWork w = kp_work(p.work, p.n_pages, p.max_seqs);
  const int i = blockIdx.x, d = dst[i];
  int later = 0;
  for (int j = i + 1 + (int)threadIdx.x; j < n; j += KF_THREADS) later |= dst[j] == d;
  later = __syncthreads_or(later);
  kp_fork_read(p, src[i], d, later, w.rows + (int64_t)i * (p.max_pages + 1), threadIdx.x, KF_THREADS, status);
}
__global__ void __launch_bounds__(KF_THREADS) kv4_fork_write_kernel(KpPool p, const int32_t* dst, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const KpWork w = kp_work(p.work, p.n_pages, p.max_seqs);
  const int32_t* keep = w.rows + (int64_t)blockIdx.x * (p.max_pages + 1);
  const int len = keep[0];
  if (len < 0) return;
  const int d = dst[blockIdx.x];
  int32_t* row = p.tables + (int64_t)d * p.max_pages;
  kp_release(p, row, kp_pages_of(p, p.lens[d]), threadIdx.x, KF_THREADS, status);
  __syncthreads();
  const int np = kp_pages_of(p, len);
  for (int j = threadIdx.x; j < np; j += KF_THREADS) row[j] = keep[1 + j];
  if (threadIdx.x == 0) p.lens[d] = len;
}
// Both halves by one CTA, a warp per pair, for up to KF_PAIRS pairs of KF_ONE table entries in all: it saves a launch (free +
// fork + extend of three pairs 11.7 -> 10.8 us on the device; 56 pairs, two rounds of the warps, 17.3 -> 18.1)
constexpr int KF_PAIRS = 32;
constexpr int64_t KF_ONE = 8192;
__global__ void __launch_bounds__(KP_THREADS) kv4_fork_kernel(KpPool p, const int32_t* src, const int32_t* dst, int n, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const KpWork w = kp_work(p.work, p.n_pages, p.max_seqs);
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += KP_THREADS / 32) {
    const int d = dst[i];
    int later = 0;
    for (int j = i + 1 + lane; j < n; j += 32) later |= dst[j] == d;
    kp_fork_read(p, src[i], d, __any_sync(0xffffffffu, later), w.rows + (int64_t)i * (p.max_pages + 1), lane, 32, status);
  }
  __syncthreads();
  for (int i = threadIdx.x >> 5; i < n; i += KP_THREADS / 32) {
    const int32_t* keep = w.rows + (int64_t)i * (p.max_pages + 1);
    const int len = keep[0];
    if (len < 0) continue;
    const int d = dst[i];
    int32_t* row = p.tables + (int64_t)d * p.max_pages;
    kp_release(p, row, kp_pages_of(p, p.lens[d]), lane, 32, status);
    __syncwarp();
    const int np = kp_pages_of(p, len);
    for (int j = lane; j < np; j += 32) row[j] = keep[1 + j];
    if (lane == 0) p.lens[d] = len;
  }
}
__global__ void __launch_bounds__(KF_THREADS) kv4_free_kernel(KpPool p, const int32_t* slots, int* status) {
  __shared__ int s_len;
  pdl_launch_dependents();
  pdl_wait();
  const int s = slots[blockIdx.x];
  if ((unsigned)s >= (unsigned)p.max_seqs) {
    if (threadIdx.x == 0) *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  if (threadIdx.x == 0) s_len = atomicExch(&p.lens[s], 0);      // a slot named twice: one of the two finds it empty
  __syncthreads();
  kp_release(p, p.tables + (int64_t)s * p.max_pages, kp_pages_of(p, s_len), threadIdx.x, KF_THREADS, status);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
int kv4_check(const bq_kv4_pool* p, const char* what) {
  const std::string w(what);
  if (device_id() < 0) return fail(BQ_ERR_STATE, "bq_init() has not been called");
  if (!p) return fail(BQ_ERR_ARG, w + ": null pool");
  if (p->head_dim <= 0 || p->head_dim % GROUP || p->head_dim > 256)
    return fail(BQ_ERR_ARG, w + ": head_dim must be a multiple of 32 up to 256");
  if (p->page < KV4_ROWS || p->page > 4096 || (p->page & (p->page - 1)))
    return fail(BQ_ERR_ARG, w + ": page must be a power of two from 16 to 4096 positions");
  if (p->layers <= 0 || p->kv_heads <= 0 || p->layers > 65536 || p->kv_heads > 65536)
    return fail(BQ_ERR_ARG, w + ": layers and kv_heads must be positive");
  if (p->n_pages <= 0 || p->n_pages >= (int64_t)1 << 30) return fail(BQ_ERR_ARG, w + ": n_pages must be in [1, 2^30)");
  if (p->max_seqs <= 0 || p->max_seqs > KV4_MAX_SEQS) return fail(BQ_ERR_ARG, w + ": max_seqs must be in [1, 8192]");
  if (p->max_pages <= 0 || (int64_t)p->max_pages * p->page > (int64_t)1 << 30)
    return fail(BQ_ERR_ARG, w + ": a sequence holds at most 2^30 positions");
  if (!p->pages || !p->tables || !p->lens || !p->refs || !p->work) return fail(BQ_ERR_ARG, w + ": null pointer in the pool");
  if ((reinterpret_cast<uintptr_t>(p->pages) | reinterpret_cast<uintptr_t>(p->refs) | reinterpret_cast<uintptr_t>(p->work)) & 15)
    return fail(BQ_ERR_ARG, w + ": pages, refs and work must be 16-byte aligned");
  if (kv4_misaligned(4, p->tables, p->lens)) return fail(BQ_ERR_ARG, w + ": tables and lens must be aligned to their elements");
  int cur = -1;
  BQ_CUDA(cudaGetDevice(&cur));
  if (cur != device_id()) return fail(BQ_ERR_STATE, w + ": the current device is not the one bq_init() selected");
  return BQ_OK;
}
static int ilog2(int v) { int n = 0; while ((1 << n) < v) ++n; return n; }
static int64_t kv4_page_bytes(const bq_kv4_pool* p) {
  return (int64_t)p->layers * p->kv_heads * (p->page / KV4_ROWS) * kv4_block_bytes(p->head_dim);
}
int kv4_view(const bq_kv4_pool* p, int layer, const char* what, Kv4View* v) {
  int rc = kv4_check(p, what);
  if (rc) return rc;
  if (layer < 0 || layer >= p->layers) return fail(BQ_ERR_ARG, std::string(what) + ": no such layer");
  v->pages = static_cast<uint8_t*>(p->pages);
  v->tables = p->tables;
  v->n_pages = p->n_pages;
  v->page_bytes = kv4_page_bytes(p);
  v->layer_off = (int64_t)layer * (v->page_bytes / p->layers);
  v->max_seqs = p->max_seqs; v->max_pages = p->max_pages; v->Hkv = p->kv_heads; v->D = p->head_dim; v->page_log2 = ilog2(p->page);
  return BQ_OK;
}
static KpPool kp_pool(const bq_kv4_pool* p) {
  return KpPool{p->tables, p->lens, p->refs, p->work, p->n_pages, p->max_seqs, p->max_pages, ilog2(p->page)};
}
static unsigned copy_grid(int64_t most_pages, int64_t page_bytes) {
  const int64_t units = most_pages * ((page_bytes + KC_CHUNK - 1) / KC_CHUNK), most = (int64_t)sm_count() * 8;
  return (unsigned)(units < 1 ? 1 : units < most ? units : most);
}

}  // namespace bq

using namespace bq;

extern "C" {

int64_t bq_kv4_page_bytes(const bq_kv4_pool* p) {
  if (!p || p->layers <= 0 || p->kv_heads <= 0 || p->page < KV4_ROWS || p->head_dim <= 0) return 0;
  return kv4_page_bytes(p);
}
int64_t bq_kv4_work_bytes(const bq_kv4_pool* p) {
  if (!p || p->n_pages <= 0 || p->max_seqs <= 0 || p->max_pages <= 0) return 0;
  return kp_work_ints(p) * (int64_t)sizeof(int32_t);
}

int bq_kv4_extend(const bq_kv4_pool* p, const int32_t* slots, const int32_t* starts, int64_t B, int32_t* pos_out, void* stream) {
  int rc = kv4_check(p, "bq_kv4_extend");
  if (rc) return rc;
  if (B < 0 || B > p->max_seqs) return fail(BQ_ERR_ARG, "bq_kv4_extend: more sequences than the pool holds");
  if (B == 0) return BQ_OK;
  if (!pos_out) return fail(BQ_ERR_ARG, "bq_kv4_extend: null pointer");
  if (kv4_misaligned(4, slots, starts, pos_out)) return fail(BQ_ERR_ARG, "bq_kv4_extend: slots, starts and pos_out must be aligned to their elements");
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t bytes = kv4_page_bytes(p);
  BQ_CUDA(launch_chain(kv4_extend_kernel, dim3(1), dim3(KP_THREADS), (size_t)p->max_seqs * sizeof(int), s, 1, kp_pool(p), slots, starts, (int)B,
                       pos_out, status_word()));
  BQ_CUDA(launch_chain(kv4_copy_kernel<false>, dim3(copy_grid(B, bytes)), dim3(KC_THREADS), 0, s, 1, kp_pool(p), (const uint8_t*)p->pages,
                       (uint8_t*)p->pages, bytes, kp_pool(p)));
  count_launch(2);
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

int bq_kv4_fork(const bq_kv4_pool* p, const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  int rc = kv4_check(p, "bq_kv4_fork");
  if (rc) return rc;
  if (n < 0 || n > p->max_seqs) return fail(BQ_ERR_ARG, "bq_kv4_fork: more pairs than the pool holds sequences");
  if (n == 0) return BQ_OK;
  if (!src || !dst) return fail(BQ_ERR_ARG, "bq_kv4_fork: null pointer");
  if (kv4_misaligned(4, src, dst)) return fail(BQ_ERR_ARG, "bq_kv4_fork: src and dst must be aligned to their elements");
  cudaStream_t s = (cudaStream_t)stream;
  if (n <= KF_PAIRS && n * p->max_pages <= KF_ONE) {
    BQ_CUDA(launch_chain(kv4_fork_kernel, dim3(1), dim3(KP_THREADS), 0, s, 1, kp_pool(p), src, dst, (int)n, status_word()));
    count_launch();
    BQ_CUDA(cudaGetLastError());
    return BQ_OK;
  }
  BQ_CUDA(launch_chain(kv4_fork_read_kernel, dim3((unsigned)n), dim3(KF_THREADS), 0, s, 1, kp_pool(p), src, dst, (int)n, status_word()));
  BQ_CUDA(launch_chain(kv4_fork_write_kernel, dim3((unsigned)n), dim3(KF_THREADS), 0, s, 1, kp_pool(p), dst, status_word()));
  count_launch(2);
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

int bq_kv4_free(const bq_kv4_pool* p, const int32_t* slots, int64_t n, void* stream) {
  int rc = kv4_check(p, "bq_kv4_free");
  if (rc) return rc;
  if (n < 0 || n > p->max_seqs) return fail(BQ_ERR_ARG, "bq_kv4_free: more slots than the pool holds sequences");
  if (n == 0) return BQ_OK;
  if (!slots) return fail(BQ_ERR_ARG, "bq_kv4_free: null pointer");
  if (kv4_misaligned(4, slots)) return fail(BQ_ERR_ARG, "bq_kv4_free: slots must be aligned to its elements");
  BQ_CUDA(launch_chain(kv4_free_kernel, dim3((unsigned)n), dim3(KF_THREADS), 0, (cudaStream_t)stream, 1, kp_pool(p), slots, status_word()));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

int bq_kv4_compact(const bq_kv4_pool* p, const bq_kv4_pool* to, void* stream) {
  int rc = kv4_check(p, "bq_kv4_compact");
  if (rc || (rc = kv4_check(to, "bq_kv4_compact (destination)"))) return rc;
  if (p->layers != to->layers || p->kv_heads != to->kv_heads || p->head_dim != to->head_dim || p->page != to->page ||
      p->max_seqs != to->max_seqs || p->max_pages != to->max_pages)
    return fail(BQ_ERR_ARG, "bq_kv4_compact: the pools may differ in their number of pages only");
  if (p->pages == to->pages || p->tables == to->tables || p->lens == to->lens || p->refs == to->refs)
    return fail(BQ_ERR_ARG, "bq_kv4_compact: the destination must be another pool");
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t bytes = kv4_page_bytes(p);
  BQ_CUDA(launch_chain(kv4_compact_plan_kernel, dim3(1), dim3(KP_THREADS), 0, s, 1, kp_pool(p), to->n_pages, status_word()));
  BQ_CUDA(launch_chain(kv4_copy_kernel<true>, dim3(copy_grid(p->n_pages, bytes)), dim3(KC_THREADS), 0, s, 1, kp_pool(p), (const uint8_t*)p->pages,
                       (uint8_t*)to->pages, bytes, kp_pool(to)));
  count_launch(2);
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

}  // extern "C"
