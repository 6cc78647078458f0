// Rows in and out of the 4-bit KV cache: append (quantise rows into their blocks), the same with the rotary embedding of a
// fused q|k|v projection in front, and gather (back to rows).
//
// One warp handles K or V of one (16-position block, head).  It works in the fragment order of the block (kv4.cuh): for K a
// lane holds eight dimensions of two positions per group and the absmax of a group is a maximum over the four lanes of a
// quad; for V it holds four dimensions of four positions and the maximum runs over the eight quads.  A block that the call
// fills completely is stored as whole words, otherwise each position's bytes are stored by themselves.
#include "kv4.cuh"

namespace bq {

constexpr int KR_WARPS = 8;
constexpr int KR_THREADS = KR_WARPS * 32;

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

// two neighbouring elements of a row
__device__ __forceinline__ float2 kr_load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 kr_load2(const __nv_bfloat16* p) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
// Where a warp's rows come from: element d of row r of the block.
template <typename T> struct KrPlain {
  const T* base;                                       // row 0 of the block, this head
  int64_t ld;
  __device__ __forceinline__ float one(int r, int d) const { return to_float<T>(base[r * ld + d]); }
  __device__ __forceinline__ float2 two(int r, int d) const { return kr_load2(base + r * ld + d); }
};
// ... of the fp32 projection output, rotated by the angles of row r (the roundings of rope_kv_append_kernel)
template <typename T> struct KrRope {
  const float* base;
  int64_t ld;
  const float *cs, *sn;                                // [16][D / 2]
  int D;
  bool rotate;
  __device__ __forceinline__ float one(int r, int d) const {
    return rope_elem<T>(base + r * ld, d, D, cs + r * (D / 2), sn + r * (D / 2), rotate);
  }
  __device__ __forceinline__ float2 two(int r, int d) const { return make_float2(one(r, d), one(r, d + 1)); }
};

template <typename SRC>
__device__ __forceinline__ void kr_append_k(const SRC& src, uint8_t* blk, int NG, int r_lo, int r_hi) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool in0 = g >= r_lo && g < r_hi, in1 = g + 8 >= r_lo && g + 8 < r_hi, whole = r_lo == 0 && r_hi == KV4_ROWS;
  __half* scales = reinterpret_cast<__half*>(blk + 256 * NG);
  for (int G = 0; G < NG; ++G) {
    float x[2][8];                                     // [row g / g + 8][tile][2t, 2t + 1, 2t + 8, 2t + 9]
    float amax[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 p = make_float2(0.0f, 0.0f);
        if (u ? in1 : in0) p = src.two(g + 8 * u, G * 32 + j * 8 + 2 * t);
        x[u][2 * j] = p.x; x[u][2 * j + 1] = p.y;
        amax[u] = kv4_absmax(amax[u], kv4_absmax(p.x, p.y));
      }
      amax[u] = kv4_absmax(amax[u], __shfl_xor_sync(0xffffffffu, amax[u], 1));
      amax[u] = kv4_absmax(amax[u], __shfl_xor_sync(0xffffffffu, amax[u], 2));
    }
    uint32_t w[2] = {0u, 0u};                          // the lane's words of the two tiles
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const __half sh = kv4_scale(amax[u]);
      const float s = __half2float(sh);
      if (t == 0 && (u ? in1 : in0)) scales[(g + 8 * u) * NG + G] = sh;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)                    // e = 2 * (high k) + odd
          w[i] |= kv4_nibble(x[u][i * 4 + e], s) << (8 * u + 16 * (e & 1) + 4 * (e >> 1));
    }
    uint8_t* at = blk + G * 256 + lane * 8;
    if (whole) {
      *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (u ? in1 : in0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            at[i * 4 + u] = (uint8_t)(w[i] >> (8 * u));
            at[i * 4 + 2 + u] = (uint8_t)(w[i] >> (16 + 8 * u));
          }
        }
    }
  }
}

template <typename SRC>
__device__ __forceinline__ void kr_append_v(const SRC& src, uint8_t* blk, int NG, int r_lo, int r_hi) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool whole = r_lo == 0 && r_hi == KV4_ROWS;
  __half* scales = reinterpret_cast<__half*>(blk + 256 * NG);
  for (int G = 0; G < NG; ++G) {
    uint32_t w[2] = {0u, 0u};
    __half sh[4];
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {                      // byte j of a word: position 2t + 8 (j & 1) + (j >> 1)
      const int r = 2 * t + 8 * (j & 1) + (j >> 1);
      in[j] = r >= r_lo && r < r_hi;
      float x[4], amax = 0.0f;                         // dimensions g, g + 8 of the two tiles
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = in[j] ? src.one(r, G * 32 + e * 8 + g) : 0.0f;
        amax = kv4_absmax(amax, x[e]);
      }
      amax = kv4_absmax(amax, __shfl_xor_sync(0xffffffffu, amax, 4));
      amax = kv4_absmax(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
      amax = kv4_absmax(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
      sh[j] = kv4_scale(amax);
      const float s = __half2float(sh[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e >> 1] |= kv4_nibble(x[e], s) << (8 * j + 4 * (e & 1));
    }
    uint8_t* at = blk + G * 256 + lane * 8;
    if (whole) {
      *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in[j]) {
          at[j] = (uint8_t)(w[0] >> (8 * j));
          at[4 + j] = (uint8_t)(w[1] >> (8 * j));
        }
    }
    if (g == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {                    // scale order: low even, low odd, high even, high odd position
        const int o = 2 * (j & 1) + (j >> 1);
        if (in[j]) scales[G * 16 + t * 4 + o] = sh[j];
      }
    }
  }
}

// grid: (items, heads by warps); a warp takes (head, K or V)
template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv4_append_kernel(Kv4View v, const T* __restrict__ k, const T* __restrict__ val, int64_t ldk,
                                                                int64_t ldv, const int32_t* __restrict__ slots,
                                                                const int32_t* __restrict__ pos, const int32_t* __restrict__ starts, int B,
                                                                int64_t n_rows, int* __restrict__ status) {
  pdl_launch_dependents();
  pdl_wait();
  const KrItem it = kr_item(v, slots, pos, starts, B, n_rows, blockIdx.x, status);
  const int task = blockIdx.y * KR_WARPS + (threadIdx.x >> 5);
  if (!it.live || task >= 2 * v.Hkv) return;
  const int h = task >> 1;
  uint8_t* blk = v.block(v.tables + (int64_t)it.slot * v.max_pages, it.blk, h);
  if (!blk) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  const int NG = v.D / GROUP;
  if (!(task & 1)) kr_append_k(KrPlain<T>{k + (int64_t)it.first * ldk + (int64_t)h * v.D, ldk}, blk, NG, it.r_lo, it.r_hi);
  else kr_append_v(KrPlain<T>{val + (int64_t)it.first * ldv + (int64_t)h * v.D, ldv}, blk + kv4_v_off(v.D), NG, it.r_lo, it.r_hi);
}

// The same behind a fused projection: qkv fp32 [n_rows][(Hq + 2 Hkv) * D].  Tasks 0 .. 2 Hkv - 1 are the heads' K and V,
// the others one query head each (rotated into q_out).
template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv4_rope_append_kernel(Kv4View v, const float* __restrict__ qkv, T* __restrict__ q_out, int Hq,
                                                                     float rope_base, const int32_t* __restrict__ slots,
                                                                     const int32_t* __restrict__ pos, const int32_t* __restrict__ starts, int B,
                                                                     int64_t n_rows, int* __restrict__ status) {
  extern __shared__ float s_ang[];                     // cos [16][D / 2], sin [16][D / 2]
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
  const int task = blockIdx.y * KR_WARPS + (threadIdx.x >> 5);
  if (task >= 2 * v.Hkv + Hq) return;
  const int64_t ld = (int64_t)(Hq + 2 * v.Hkv) * D;
  const float* rows = qkv + (int64_t)it.first * ld;
  if (task >= 2 * v.Hkv) {
    const int h = task - 2 * v.Hkv;
    for (int e = threadIdx.x & 31; e < (it.r_hi - it.r_lo) * D; e += 32) {
      const int r = it.r_lo + e / D, d = e % D;
      q_out[((int64_t)(it.first + r) * Hq + h) * D + d] =
          from_float<T>(rope_elem<T>(rows + r * ld + (int64_t)h * D, d, D, cs + r * half, sn + r * half, true));
    }
    return;
  }
  const int h = task >> 1;
  uint8_t* blk = v.block(v.tables + (int64_t)it.slot * v.max_pages, it.blk, h);
  if (!blk) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  const int NG = D / GROUP;
  if (!(task & 1)) kr_append_k(KrRope<T>{rows + (int64_t)(Hq + h) * D, ld, cs, sn, D, true}, blk, NG, it.r_lo, it.r_hi);
  else kr_append_v(KrRope<T>{rows + (int64_t)(Hq + v.Hkv + h) * D, ld, cs, sn, D, false}, blk + kv4_v_off(D), NG, it.r_lo, it.r_hi);
}

// code * scale of one nibble of a word
__device__ __forceinline__ float kr_value(uint32_t w, int shift, float s) { return (float)((int)((w >> shift) & 15u) - 8) * s; }

template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv4_gather_kernel(Kv4View v, T* __restrict__ k, T* __restrict__ val, const int32_t* __restrict__ slots,
                                                                const int32_t* __restrict__ pos, const int32_t* __restrict__ starts, int B,
                                                                int64_t n_rows, int* __restrict__ status) {
  pdl_launch_dependents();
  pdl_wait();
  const KrItem it = kr_item(v, slots, pos, starts, B, n_rows, blockIdx.x, status);
  const int task = blockIdx.y * KR_WARPS + (threadIdx.x >> 5);
  if (!it.live || task >= 2 * v.Hkv) return;
  const int h = task >> 1, D = v.D, NG = D / GROUP;
  const uint8_t* blk = v.block(v.tables + (int64_t)it.slot * v.max_pages, it.blk, h);
  if (!blk) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    return;
  }
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t ld = (int64_t)v.Hkv * D;
  T* out = ((task & 1) ? val : k) + (int64_t)it.first * ld + (int64_t)h * D;
  if (task & 1) blk += kv4_v_off(D);
  const __half* scales = reinterpret_cast<const __half*>(blk + 256 * NG);
  for (int G = 0; G < NG; ++G) {
    const uint2 w2 = *reinterpret_cast<const uint2*>(blk + G * 256 + lane * 8);
    const uint32_t w[2] = {w2.x, w2.y};
    if (!(task & 1)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = g + 8 * u;
        if (r < it.r_lo || r >= it.r_hi) continue;
        const float s = __half2float(scales[r * NG + G]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            T* o = out + r * ld + G * 32 + i * 16 + hi * 8 + 2 * t;
            o[0] = from_float<T>(kr_value(w[i], 8 * u + 4 * hi, s));
            o[1] = from_float<T>(kr_value(w[i], 16 + 8 * u + 4 * hi, s));
          }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 2 * t + 8 * (j & 1) + (j >> 1);
        if (r < it.r_lo || r >= it.r_hi) continue;
        const float s = __half2float(scales[G * 16 + t * 4 + 2 * (j & 1) + (j >> 1)]);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[r * ld + G * 32 + e * 8 + g] = from_float<T>(kr_value(w[e >> 1], 8 * j + 4 * (e & 1), s));
      }
    }
  }
}

// work items that cover every block which n_rows rows of B sequences can touch (kv4_item_base)
static int64_t kr_items(int64_t B, int64_t n_rows, bool ragged) { return ragged ? (n_rows >> 4) + 2 * B : B; }
static int kr_check(const bq_kv4_pool* p, int64_t B, int64_t n_rows, const int32_t* starts, const int32_t* pos, int dtype, const char* what) {
  const std::string w(what);
  if (dtype != BQ_DT_F32 && dtype != BQ_DT_BF16) return fail(BQ_ERR_ARG, w + ": dtype must be BQ_DT_F32 or BQ_DT_BF16");
  if (B < 0 || B > p->max_seqs) return fail(BQ_ERR_ARG, w + ": more sequences than the pool holds");
  if (n_rows < 0 || n_rows > (int64_t)1 << 30 || (!starts && n_rows != B))
    return fail(BQ_ERR_ARG, w + ": bad number of rows (one per sequence without row ranges)");
  if (B && !pos) return fail(BQ_ERR_ARG, w + ": null pointer");
  return BQ_OK;
}

}  // namespace bq

using namespace bq;

extern "C" {

int bq_kv4_append(const bq_kv4_pool* p, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int dtype, const int32_t* slots,
                  const int32_t* pos, const int32_t* starts, int64_t B, int64_t n_rows, void* stream) {
  Kv4View view;
  int rc = kv4_view(p, layer, "bq_kv4_append", &view);
  if (rc || (rc = kr_check(p, B, n_rows, starts, pos, dtype, "bq_kv4_append"))) return rc;
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!k || !v) return fail(BQ_ERR_ARG, "bq_kv4_append: null pointer");
  const int64_t row = (int64_t)p->kv_heads * p->head_dim;
  const uintptr_t pair = dtype == BQ_DT_F32 ? 7 : 3;
  if (ldk < row || ldv < row || (ldk & 1) || (ldv & 1) || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & pair))
    return fail(BQ_ERR_ARG, "bq_kv4_append: rows must be aligned to two elements, an even number of elements apart and not overlap");
  const dim3 grid((unsigned)kr_items(B, n_rows, starts != nullptr), (unsigned)((2 * p->kv_heads + KR_WARPS - 1) / KR_WARPS));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BQ_DT_F32)
    BQ_CUDA(launch_chain(kv4_append_kernel<float>, grid, dim3(KR_THREADS), 0, s, 1, view, (const float*)k, (const float*)v, ldk, ldv, slots, pos,
                         starts, (int)B, n_rows, status_word()));
  else
    BQ_CUDA(launch_chain(kv4_append_kernel<__nv_bfloat16>, grid, dim3(KR_THREADS), 0, s, 1, view, (const __nv_bfloat16*)k,
                         (const __nv_bfloat16*)v, ldk, ldv, slots, pos, starts, (int)B, n_rows, status_word()));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

int bq_kv4_rope_append(const bq_kv4_pool* p, int layer, const float* qkv, void* q_out, int Hq, float rope_base, int dtype, const int32_t* slots,
                       const int32_t* pos, const int32_t* starts, int64_t B, int64_t n_rows, void* stream) {
  Kv4View view;
  int rc = kv4_view(p, layer, "bq_kv4_rope_append", &view);
  if (rc || (rc = kr_check(p, B, n_rows, starts, pos, dtype, "bq_kv4_rope_append"))) return rc;
  if (Hq <= 0 || Hq % p->kv_heads) return fail(BQ_ERR_ARG, "bq_kv4_rope_append: query heads must be a multiple of the KV heads");
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!qkv || !q_out) return fail(BQ_ERR_ARG, "bq_kv4_rope_append: null pointer");
  const dim3 grid((unsigned)kr_items(B, n_rows, starts != nullptr), (unsigned)((2 * p->kv_heads + Hq + KR_WARPS - 1) / KR_WARPS));
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
  if (rc || (rc = kr_check(p, B, n_rows, starts, pos, dtype, "bq_kv4_gather"))) return rc;
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!k || !v) return fail(BQ_ERR_ARG, "bq_kv4_gather: null pointer");
  const dim3 grid((unsigned)kr_items(B, n_rows, starts != nullptr), (unsigned)((2 * p->kv_heads + KR_WARPS - 1) / KR_WARPS));
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BQ_DT_F32)
    BQ_CUDA(launch_chain(kv4_gather_kernel<float>, grid, dim3(KR_THREADS), 0, s, 1, view, (float*)k, (float*)v, slots, pos, starts, (int)B,
                         n_rows, status_word()));
  else
    BQ_CUDA(launch_chain(kv4_gather_kernel<__nv_bfloat16>, grid, dim3(KR_THREADS), 0, s, 1, view, (__nv_bfloat16*)k, (__nv_bfloat16*)v, slots,
                         pos, starts, (int)B, n_rows, status_word()));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

}  // extern "C"
