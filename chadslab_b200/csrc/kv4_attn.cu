// Attention over the paged 4-bit KV cache.
//   o[i, h] = sum_p softmax_p(q[i, h] . K[p] / sqrt(D)) V[p],   p <= position of row i
// One CTA per (row, query head); its warps take the positions in turn with a running maximum and sum, and meet in shared
// memory.
#include "kv4.cuh"

namespace bq {

constexpr int KA_WARPS = 4;
constexpr int KA_THREADS = KA_WARPS * 32;

template <typename T>
__global__ void __launch_bounds__(KA_THREADS) kv4_attention_kernel(Kv4View v, const T* __restrict__ q, int64_t ldq, T* __restrict__ out, int Hq,
                                                                   const int32_t* __restrict__ slots, const int32_t* __restrict__ pos,
                                                                   const int32_t* __restrict__ starts, int B, int64_t n_rows,
                                                                   int* __restrict__ status) {
  __shared__ float s_m[KA_WARPS], s_l[KA_WARPS], s_o[KA_WARPS][256];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.y, hq = blockIdx.x, D = v.D, NG = D / GROUP, h = hq / (Hq / v.Hkv);
  int b = row;
  if (starts) {                                        // the sequence of this row: the last that starts at or before it
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (starts[mid] <= row) lo = mid; else hi = mid;
    }
    b = lo;
  }
  const Kv4Seq s = kv4_seq(v, slots, pos, starts, b, n_rows, status);
  if (row < s.row0 || row >= s.row0 + s.n) return;     // behind the last sequence
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int end = s.pos < 0 ? 0 : s.pos + (row - s.row0) + 1;
  float qv[8], acc[8], m = -INFINITY, l = 0.0f;
  for (int G = 0; G < 8; ++G) {
    qv[G] = G < NG ? to_float<T>(q[(int64_t)row * ldq + (int64_t)hq * D + G * 32 + lane]) * rsqrtf((float)D) : 0.0f;
    acc[G] = 0.0f;
  }
  const int e = lane & 15, tile = lane >> 4;
  for (int p = warp; p < end; p += KA_WARPS) {
    const uint8_t* blk = v.block(v.tables + (int64_t)s.slot * v.max_pages, p >> 4, h);
    if (!blk) {
      *(volatile int*)status = (int)BQ_ERR_ARG;
      continue;
    }
    const int r = p & 15;
    const __half* ks = reinterpret_cast<const __half*>(blk + kv4_kscale_off(D));
    const __half* vs = reinterpret_cast<const __half*>(blk + kv4_vscale_off(D));
    float dot = 0.0f;
    for (int G = 0; G < NG; ++G) {
      const uint8_t byte = blk[G * 256 + ((r & 7) * 4 + (e & 7) / 2) * 8 + tile * 4 + (r >> 3) + 2 * (e & 1)];
      dot += qv[G] * ((float)((byte >> (4 * (e >> 3))) & 15) - 8.0f) * __half2float(ks[r * NG + G]);
    }
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float nm = fmaxf(m, dot), corr = __expf(m - nm), w = __expf(dot - nm);
    l = l * corr + w;
    for (int G = 0; G < NG; ++G) {
      const uint8_t byte = blk[kv4_v_off(D) + G * 256 + ((e & 7) * 4 + (r & 7) / 2) * 8 + tile * 4 + (r >> 3) + 2 * (r & 1)];
      acc[G] = acc[G] * corr + w * ((float)((byte >> (4 * (e >> 3))) & 15) - 8.0f) * __half2float(vs[G * 16 + (r & 7) / 2 * 4 + (r >> 3) * 2 + (r & 1)]);
    }
    m = nm;
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  for (int G = 0; G < NG; ++G) s_o[warp][G * 32 + lane] = acc[G];
  __syncthreads();
  float gm = -INFINITY;
  for (int w = 0; w < KA_WARPS; ++w) gm = fmaxf(gm, s_m[w]);
  for (int d = threadIdx.x; d < D; d += KA_THREADS) {
    float o = 0.0f, sum = 0.0f;
    for (int w = 0; w < KA_WARPS; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.0f : __expf(s_m[w] - gm);
      o += s_o[w][d] * f;
      sum += s_l[w] * f;
    }
    out[((int64_t)row * Hq + hq) * D + d] = from_float<T>(end > 0 ? o / sum : 0.0f);
  }
}

}  // namespace bq

using namespace bq;

extern "C" {

int64_t bq_kv4_attention_work_bytes(const bq_kv4_pool* p, int Hq, int dtype) { (void)p; (void)Hq; (void)dtype; return 16; }

int bq_kv4_attention(const bq_kv4_pool* p, int layer, const void* q, int64_t ldq, void* out, int Hq, int dtype, const int32_t* slots,
                     const int32_t* pos, const int32_t* starts, int64_t B, int64_t n_rows, void* work, void* stream) {
  Kv4View view;
  int rc = kv4_view(p, layer, "bq_kv4_attention", &view);
  if (rc) return rc;
  if (dtype != BQ_DT_F32 && dtype != BQ_DT_BF16) return fail(BQ_ERR_ARG, "bq_kv4_attention: dtype must be BQ_DT_F32 or BQ_DT_BF16");
  if (Hq <= 0 || Hq % p->kv_heads) return fail(BQ_ERR_ARG, "bq_kv4_attention: query heads must be a multiple of the KV heads");
  if (B < 0 || B > p->max_seqs) return fail(BQ_ERR_ARG, "bq_kv4_attention: more sequences than the pool holds");
  if (n_rows < 0 || n_rows > 65535 || (!starts && n_rows != B))
    return fail(BQ_ERR_ARG, "bq_kv4_attention: bad number of rows (one per sequence without row ranges)");
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!q || !out || !pos || !work) return fail(BQ_ERR_ARG, "bq_kv4_attention: null pointer");
  if (ldq < (int64_t)Hq * p->head_dim) return fail(BQ_ERR_ARG, "bq_kv4_attention: rows of q overlap");
  const dim3 grid((unsigned)Hq, (unsigned)n_rows);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BQ_DT_F32)
    BQ_CUDA(launch_chain(kv4_attention_kernel<float>, grid, dim3(KA_THREADS), 0, s, 1, view, (const float*)q, ldq, (float*)out, Hq, slots, pos,
                         starts, (int)B, n_rows, status_word()));
  else
    BQ_CUDA(launch_chain(kv4_attention_kernel<__nv_bfloat16>, grid, dim3(KA_THREADS), 0, s, 1, view, (const __nv_bfloat16*)q, ldq,
                         (__nv_bfloat16*)out, Hq, slots, pos, starts, (int)B, n_rows, status_word()));
  count_launch();
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

}  // extern "C"
