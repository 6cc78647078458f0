// Rows in and out of the 4-bit KV cache: append (quantise rows into their blocks), the same with the rotary embedding of a
// fused q|k|v projection in front, and gather (back to rows).
//
// Two warps handle K or V of one (16-position block, head), half the rows each, row by row: a lane owns eight neighbouring dimensions (one or two
// 16-byte loads), four lanes a group, so the absmax takes two exchanges for the whole row, whatever head_dim.  The eight
// codes of a lane and of its neighbour share eight bytes (elements e and e + 8 of a 16-wide tile): one exchange pairs them.
// A block that the call fills completely is put together in shared memory and leaves as 16-byte stores; otherwise the bytes
// of its rows are stored one by one (a decode step has one row per block, and other rows' bytes must stay).
// Bound: launch latency for a decode step; for prompts the instructions of the quantiser.
#include "kv4.cuh"

namespace bq {

constexpr int KR_WARPS = 8;
constexpr int KR_THREADS = KR_WARPS * 32;
constexpr int KR_TASKS = KR_WARPS / 2;                 // two warps share a task: (block, head, K or V)
__device__ __forceinline__ void kr_pair_sync(int pair) { asm volatile("bar.sync %0, 64;" ::"r"(pair + 1) : "memory"); }

// The place of a work item: rows r_lo .. r_hi - 1 of block `blk` of one sequence; row r is row first + r of the call's rows
struct KrItem {
  int slot, blk, r_lo, r_hi, first, pos0;
  bool live;
};
__device__ __forceinline__ KrItem kr_item(const Kv4View& v, const int32_t* slots, const int32_t* pos, const int32_t* starts, int B, int64_t T,
                                          int item, int* status) {
  KrItem it;
  const int b = starts ? kv4_item_seq(starts, B, item) : item;
  const Kv4Seq s = kv4_seq(v, slots, pos, starts, b, T, status);
  it.live = false;
  if (s.n <= 0 || s.pos < 0) return it;
  it.slot = s.slot;
  it.blk = (s.pos >> 4) + (starts ? item - kv4_item_base(starts, b) : 0);
  it.pos0 = it.blk * KV4_ROWS;
  it.r_lo = max(0, s.pos - it.pos0);
  it.r_hi = min(KV4_ROWS, s.pos + s.n - it.pos0);
  it.first = s.row0 - s.pos + it.pos0;                // may be negative; row r >= r_lo is not
  it.live = it.blk >= (s.pos >> 4) && it.r_lo < it.r_hi;
  return it;
}

// Eight neighbouring elements of a row, from a row of the call ...
template <typename T> struct KrPlain {
  const T* base;                                       // row 0 of the block, this head
  int64_t ld;
  bool vec;                                            // rows are 16-byte aligned
  __device__ __forceinline__ void eight(int r, int d, float* x) const {
    const T* p = base + r * ld + d;
    if (vec) {
      load8<T>(p, x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = to_float<T>(p[j]);
    }
  }
};
// ... or of the fp32 projection output, rotated by the angles of row r (the roundings of rope_kv_append_kernel)
template <typename T> struct KrRope {
  const float* base;
  int64_t ld;
  const float *cs, *sn;                                // [16][D / 2]
  int D;
  bool rotate;
  __device__ __forceinline__ void eight(int r, int d, float* x) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = rope_elem_of<T>(base + r * ld, d + j, D, cs + r * (D / 2), sn + r * (D / 2), rotate);
  }
};

// code + 8 of x: rint(x / scale).  The product with the reciprocal is off by less than 2^-20 of a step, so only next to a
// border between two codes is the quotient itself needed.
__device__ __forceinline__ uint32_t kr_nibble(float x, float s, float inv) {
  const float y = x * inv;
  float f = rintf(y);
  if (fabsf(fabsf(y - f) - 0.5f) < 1e-5f) f = rintf(__fdiv_rn(x, s));
  return (uint32_t)((int)fminf(fmaxf(f, -7.0f), 7.0f) + 8);
}
// Byte of the codes that holds elements e and e + 8 (e < 8) of tile `tile` of group G at position r
__device__ __forceinline__ int kr_byte(bool values, int r, int G, int tile, int e) {
  return G * 256 + 4 * tile + (r >> 3) + (values ? (e * 4 + ((r & 7) >> 1)) * 8 + 2 * (r & 1) : ((r & 7) * 4 + (e >> 1)) * 8 + 2 * (e & 1));
}
__device__ __forceinline__ int kr_scale(bool values, int r, int G, int NG) {
  return values ? G * 16 + ((r & 7) >> 1) * 4 + (r >> 3) * 2 + (r & 1) : r * NG + G;
}
// Quantises rows r_lo .. r_hi - 1 of a block into `to`: its codes and scales in global memory, or a copy in shared memory.
// 256 / D rows at a time; the next ones are on their way while these are quantised.
template <typename SRC>
__device__ __forceinline__ void kr_quantise(const SRC& src, uint8_t* to, bool values, int D, int r_lo, int r_hi) {
  const int lane = threadIdx.x & 31, NG = D / GROUP, per = D / 8, rows = 32 / per, sub = lane / per, l = lane - sub * per;
  const int G = l >> 2, tile = (l >> 1) & 1;
  __half* scales = reinterpret_cast<__half*>(to + 256 * NG);
  auto load = [&](int r, float* x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.0f;
    if (sub < rows && r < r_hi) src.eight(r, l * 8, x);
  };
  float next[8];
  load(r_lo + sub, next);
  for (int r0 = r_lo; r0 < r_hi; r0 += rows) {
    const int r = r0 + sub;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = next[j];
    load(r + rows, next);
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = kv4_absmax(amax, x[j]);
    amax = kv4_absmax(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = kv4_absmax(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const __half sh = kv4_scale(amax);
    const float s = __half2float(sh), inv = s > 0.0f ? 1.0f / s : 0.0f;
    uint32_t mine = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine |= kr_nibble(x[j], s, inv) << (4 * j);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
    if (sub >= rows || r >= r_hi) continue;
    // the even lane (elements 0-7 of the tile) has the low nibbles; each lane stores four of the eight bytes
    const uint32_t low = l & 1 ? other : mine, high = l & 1 ? mine : other;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = ((j + G) & 3) * 2 + (l & 1);                         // (groups start at different banks)
      to[kr_byte(values, r, G, tile, e)] = (uint8_t)(((low >> (4 * e)) & 15u) | (((high >> (4 * e)) & 15u) << 4));
    }
    if ((l & 3) == 0) scales[kr_scale(values, r, G, NG)] = sh;
  }
}
// the same by a pair of warps: through `stage` (288 * NG bytes of shared memory of the pair's own) if the whole block is written
template <typename SRC>
__device__ __forceinline__ void kr_append(const SRC& src, uint8_t* blk, uint8_t* stage, bool values, int D, int r_lo, int r_hi) {
  const int pair = threadIdx.x >> 6, half = (threadIdx.x >> 5) & 1;
  if (r_hi - r_lo < KV4_ROWS) {
    const int mid = (r_lo + r_hi + 1) >> 1;
    kr_quantise(src, blk, values, D, half ? mid : r_lo, half ? r_hi : mid);
    return;
  }
  kr_quantise(src, stage, values, D, half * 8, half * 8 + 8);
  kr_pair_sync(pair);
  for (int e = (threadIdx.x & 63) * 16; e < 288 * (D / GROUP); e += 1024)
    *reinterpret_cast<uint4*>(blk + e) = *reinterpret_cast<const uint4*>(stage + e);
}
constexpr int KR_STAGE = 288 * 8;                      // of the largest head_dim

// grid: (items, tasks by pairs of warps); a task is (head, K or V)
template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv4_append_kernel(Kv4View v, const T* k, const T* val, int64_t ldk,
                                                                int64_t ldv, const int32_t* slots,
                                                                const int32_t* pos, const int32_t* starts, int B,
                                                                int64_t n_rows, int* status, bool vec) {
  __shared__ __align__(16) uint8_t stage[KR_TASKS][KR_STAGE];
  pdl_launch_dependents();
  pdl_wait();
  const KrItem it = kr_item(v, slots, pos, starts, B, n_rows, blockIdx.x, status);
  const int pair = threadIdx.x >> 6, task = blockIdx.y * KR_TASKS + pair;
  if (!it.live || task >= 2 * v.Hkv) return;
  const int h = task >> 1;
  uint8_t* blk = v.block(v.tables + (int64_t)it.slot * v.max_pages, it.blk, h);
  if (!blk) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  const bool values = task & 1;
  const int64_t ld = values ? ldv : ldk;
  kr_append(KrPlain<T>{(values ? val : k) + (int64_t)it.first * ld + (int64_t)h * v.D, ld, vec}, blk + (values ? kv4_v_off(v.D) : 0), stage[pair],
            values, v.D, it.r_lo, it.r_hi);
}

// The same behind a fused projection: qkv fp32 [n_rows][(Hq + 2 Hkv) * D].  Tasks 0 .. 2 Hkv - 1 are the heads' K and V,
// the others one query head each (rotated into q_out).
template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv4_rope_append_kernel(Kv4View v, const float* qkv, T* q_out, int Hq,
                                                                     float rope_base, const int32_t* slots,
                                                                     const int32_t* pos, const int32_t* starts, int B,
                                                                     int64_t n_rows, int* status) {
  extern __shared__ float s_ang[];                     // cos [16][D / 2], sin [16][D / 2]
  __shared__ __align__(16) uint8_t stage[KR_TASKS][KR_STAGE];
  pdl_launch_dependents();
  pdl_wait();
  const KrItem it = kr_item(v, slots, pos, starts, B, n_rows, blockIdx.x, status);
  if (!it.live) return;
  const int D = v.D, half = D / 2;
  float *cs = s_ang, *sn = s_ang + KV4_ROWS * half;
  for (int e = threadIdx.x; e < (it.r_hi - it.r_lo) * half; e += KR_THREADS) {
    const int r = it.r_lo + e / half, j = e % half;
    const float inv = 1.0f / powf(rope_base, (float)(2 * j) / (float)D);
    sincosf((float)(it.pos0 + r) * inv, &sn[r * half + j], &cs[r * half + j]);
  }
  __syncthreads();
  const int task = blockIdx.y * KR_TASKS + (threadIdx.x >> 6);
  if (task >= 2 * v.Hkv + Hq) return;
  const int64_t ld = (int64_t)(Hq + 2 * v.Hkv) * D;
  const float* rows = qkv + (int64_t)it.first * ld;
  if (task >= 2 * v.Hkv) {
    const int h = task - 2 * v.Hkv;
    for (int e = threadIdx.x & 63; e < (it.r_hi - it.r_lo) * D; e += 64) {
      const int r = it.r_lo + e / D, d = e % D;
      q_out[((int64_t)(it.first + r) * Hq + h) * D + d] =
          from_float<T>(rope_elem_of<T>(rows + r * ld + (int64_t)h * D, d, D, cs + r * half, sn + r * half, true));
    }
    return;
  }
  const int h = task >> 1;
  uint8_t* blk = v.block(v.tables + (int64_t)it.slot * v.max_pages, it.blk, h);
  if (!blk) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  const bool values = task & 1;
  kr_append(KrRope<T>{rows + (int64_t)(Hq + (values ? v.Hkv : 0) + h) * D, ld, cs, sn, D, !values}, blk + (values ? kv4_v_off(D) : 0),
            stage[threadIdx.x >> 6], values, D, it.r_lo, it.r_hi);
}

template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv4_gather_kernel(Kv4View v, T* k, T* val, const int32_t* slots,
                                                                const int32_t* pos, const int32_t* starts, int B,
                                                                int64_t n_rows, int* status, bool vec) {
  __shared__ __align__(16) uint8_t all[KR_TASKS][KR_STAGE];
  pdl_launch_dependents();
  pdl_wait();
  const KrItem it = kr_item(v, slots, pos, starts, B, n_rows, blockIdx.x, status);
  const int pair = threadIdx.x >> 6, task = blockIdx.y * KR_TASKS + pair;
  if (!it.live || task >= 2 * v.Hkv) return;
  const int h = task >> 1, D = v.D, NG = D / GROUP, lane = threadIdx.x & 31;
  const bool values = task & 1;
  const uint8_t* blk = v.block(v.tables + (int64_t)it.slot * v.max_pages, it.blk, h);
  if (!blk) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  if (values) blk += kv4_v_off(D);
  uint8_t* stage = all[pair];
#pragma unroll
  for (int e = (threadIdx.x & 63) * 16; e < KR_STAGE; e += 1024)
    if (e < 288 * NG) *reinterpret_cast<uint4*>(stage + e) = *reinterpret_cast<const uint4*>(blk + e);
  kr_pair_sync(pair);
  const int per = D / 8, rows = 32 / per, sub = lane / per, l = lane - sub * per;       // 256 / D rows at a time
  if (sub >= rows) return;
  const int G = l >> 2, tile = (l >> 1) & 1, shift = 4 * (l & 1);
  const __half* scales = reinterpret_cast<const __half*>(stage + 256 * NG);
  const int64_t ld = (int64_t)v.Hkv * D;
  T* out = (values ? val : k) + (int64_t)it.first * ld + (int64_t)h * D + l * 8;
  for (int r = it.r_lo + ((threadIdx.x >> 5) & 1) * rows + sub; r < it.r_hi; r += 2 * rows) {
    const float s = __half2float(scales[kr_scale(values, r, G, NG)]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)((int)((stage[kr_byte(values, r, G, tile, e)] >> shift) & 15) - 8) * s;
    if (vec) {
      store8<T>(out + r * ld, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) out[r * ld + e] = from_float<T>(x[e]);
    }
  }
}

// work items that cover every block which n_rows rows of B sequences can touch (kv4_item_base)
static int64_t kr_items(int64_t B, int64_t n_rows, bool ragged) { return ragged ? (n_rows >> 4) + 2 * B : B; }
static int kr_check(const bq_kv4_pool* p, int64_t B, int64_t n_rows, const int32_t* slots, const int32_t* starts, const int32_t* pos, int dtype,
                    const char* what) {
  const std::string w(what);
  if (dtype != BQ_DT_F32 && dtype != BQ_DT_BF16) return fail(BQ_ERR_ARG, w + ": dtype must be BQ_DT_F32 or BQ_DT_BF16");
  if (B < 0 || B > p->max_seqs) return fail(BQ_ERR_ARG, w + ": more sequences than the pool holds");
  if (n_rows < 0 || n_rows > (int64_t)1 << 30 || (!starts && n_rows != B))
    return fail(BQ_ERR_ARG, w + ": bad number of rows (one per sequence without row ranges)");
  if (B && !pos) return fail(BQ_ERR_ARG, w + ": null pointer");
  if (kv4_misaligned(4, slots, starts, pos)) return fail(BQ_ERR_ARG, w + ": slots, pos and starts must be aligned to their elements");
  return BQ_OK;
}

}  // namespace bq

using namespace bq;

extern "C" {

int bq_kv4_append(const bq_kv4_pool* p, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int dtype, const int32_t* slots,
                  const int32_t* pos, const int32_t* starts, int64_t B, int64_t n_rows, void* stream) {
  Kv4View view;
  int rc = kv4_view(p, layer, "bq_kv4_append", &view);
  if (rc || (rc = kr_check(p, B, n_rows, slots, starts, pos, dtype, "bq_kv4_append"))) return rc;
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!k || !v) return fail(BQ_ERR_ARG, "bq_kv4_append: null pointer");
  const int64_t row = (int64_t)p->kv_heads * p->head_dim;
  const uintptr_t size = dtype == BQ_DT_F32 ? 4 : 2;
  const uintptr_t align = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  if (ldk < row || ldv < row || (align & (size - 1))) return fail(BQ_ERR_ARG, "bq_kv4_append: rows overlap or are not aligned to their elements");
  const bool vec = ((align | (uintptr_t)ldk * size | (uintptr_t)ldv * size) & 15) == 0;
  const dim3 grid((unsigned)kr_items(B, n_rows, starts != nullptr), (unsigned)((2 * p->kv_heads + KR_TASKS - 1) / KR_TASKS));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BQ_DT_F32)
    BQ_CUDA(launch_chain(kv4_append_kernel<float>, grid, dim3(KR_THREADS), 0, s, 1, view, (const float*)k, (const float*)v, ldk, ldv, slots, pos,
                         starts, (int)B, n_rows, status_word(), vec));
  else
    BQ_CUDA(launch_chain(kv4_append_kernel<__nv_bfloat16>, grid, dim3(KR_THREADS), 0, s, 1, view, (const __nv_bfloat16*)k,
                         (const __nv_bfloat16*)v, ldk, ldv, slots, pos, starts, (int)B, n_rows, status_word(), vec));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

int bq_kv4_rope_append(const bq_kv4_pool* p, int layer, const float* qkv, void* q_out, int Hq, float rope_base, int dtype, const int32_t* slots,
                       const int32_t* pos, const int32_t* starts, int64_t B, int64_t n_rows, void* stream) {
  Kv4View view;
  int rc = kv4_view(p, layer, "bq_kv4_rope_append", &view);
  if (rc || (rc = kr_check(p, B, n_rows, slots, starts, pos, dtype, "bq_kv4_rope_append"))) return rc;
  if (Hq <= 0 || Hq > 65536 || Hq % p->kv_heads)
    return fail(BQ_ERR_ARG, "bq_kv4_rope_append: query heads must be a multiple of the KV heads, 65536 at most");
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!qkv || !q_out) return fail(BQ_ERR_ARG, "bq_kv4_rope_append: null pointer");
  if (kv4_misaligned(4, qkv) || kv4_misaligned(dtype == BQ_DT_F32 ? 4 : 2, q_out))
    return fail(BQ_ERR_ARG, "bq_kv4_rope_append: qkv and q_out must be aligned to their elements");
  const dim3 grid((unsigned)kr_items(B, n_rows, starts != nullptr), (unsigned)((2 * p->kv_heads + Hq + KR_TASKS - 1) / KR_TASKS));
  const size_t smem = (size_t)KV4_ROWS * p->head_dim * sizeof(float);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BQ_DT_F32)
    BQ_CUDA(launch_chain(kv4_rope_append_kernel<float>, grid, dim3(KR_THREADS), smem, s, 1, view, qkv, (float*)q_out, Hq, rope_base, slots, pos,
                         starts, (int)B, n_rows, status_word()));
  else
    BQ_CUDA(launch_chain(kv4_rope_append_kernel<__nv_bfloat16>, grid, dim3(KR_THREADS), smem, s, 1, view, qkv, (__nv_bfloat16*)q_out, Hq,
                         rope_base, slots, pos, starts, (int)B, n_rows, status_word()));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

int bq_kv4_gather(const bq_kv4_pool* p, int layer, void* k, void* v, int dtype, const int32_t* slots, const int32_t* pos, const int32_t* starts,
                  int64_t B, int64_t n_rows, void* stream) {
  Kv4View view;
  int rc = kv4_view(p, layer, "bq_kv4_gather", &view);
  if (rc || (rc = kr_check(p, B, n_rows, slots, starts, pos, dtype, "bq_kv4_gather"))) return rc;
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!k || !v) return fail(BQ_ERR_ARG, "bq_kv4_gather: null pointer");
  if (kv4_misaligned(dtype == BQ_DT_F32 ? 4 : 2, k, v)) return fail(BQ_ERR_ARG, "bq_kv4_gather: k and v must be aligned to their elements");
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  const dim3 grid((unsigned)kr_items(B, n_rows, starts != nullptr), (unsigned)((2 * p->kv_heads + KR_TASKS - 1) / KR_TASKS));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BQ_DT_F32)
    BQ_CUDA(launch_chain(kv4_gather_kernel<float>, grid, dim3(KR_THREADS), 0, s, 1, view, (float*)k, (float*)v, slots, pos, starts, (int)B,
                         n_rows, status_word(), vec));
  else
    BQ_CUDA(launch_chain(kv4_gather_kernel<__nv_bfloat16>, grid, dim3(KR_THREADS), 0, s, 1, view, (__nv_bfloat16*)k, (__nv_bfloat16*)v, slots,
                         pos, starts, (int)B, n_rows, status_word(), vec));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

}  // extern "C"
