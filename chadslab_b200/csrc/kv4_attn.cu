// Attention over the paged 4-bit KV cache: entry points, and the variants of the head dimensions without a file of their own
// (32, 96, 160, 192, 224: eight columns whatever the number of query heads).
#include "kv4_attn.cuh"

namespace bq {

template <> int ka_pick<float, 2>(const KaArgs& a, int64_t cols, cudaStream_t s);
template <> int ka_pick<__nv_bfloat16, 2>(const KaArgs& a, int64_t cols, cudaStream_t s);
template <> int ka_pick<float, 4>(const KaArgs& a, int64_t cols, cudaStream_t s);
template <> int ka_pick<__nv_bfloat16, 4>(const KaArgs& a, int64_t cols, cudaStream_t s);
template <> int ka_pick<float, 8>(const KaArgs& a, int64_t cols, cudaStream_t s);
template <> int ka_pick<__nv_bfloat16, 8>(const KaArgs& a, int64_t cols, cudaStream_t s);
template <typename T, int NG> int ka_pick(const KaArgs& a, int64_t cols, cudaStream_t s) { (void)cols; return ka_launch<T, NG, 8>(a, s); }

template <typename T> static int ka_run(const KaArgs& a, int64_t cols, cudaStream_t s) {
  switch (a.v.D / GROUP) {
    case 1: return ka_pick<T, 1>(a, cols, s);
    case 2: return ka_pick<T, 2>(a, cols, s);
    case 3: return ka_pick<T, 3>(a, cols, s);
    case 4: return ka_pick<T, 4>(a, cols, s);
    case 5: return ka_pick<T, 5>(a, cols, s);
    case 6: return ka_pick<T, 6>(a, cols, s);
    case 7: return ka_pick<T, 7>(a, cols, s);
    default: return ka_pick<T, 8>(a, cols, s);
  }
}

// columns of an average sequence and KV head: any variant is right for any number, this decides which is fast
static int64_t ka_columns(int64_t B, int64_t n_rows, int rep, int dtype) { return (n_rows + B - 1) / B * rep * (dtype == BQ_DT_F32 ? 2 : 1); }

}  // namespace bq

using namespace bq;

extern "C" {

int64_t bq_kv4_attention_work_bytes(const bq_kv4_pool* p, int Hq, int dtype, int64_t B, int64_t n_rows) {
  if (!p || p->head_dim <= 0 || p->kv_heads <= 0 || Hq <= 0 || B <= 0 || n_rows < 0) return 0;
  int64_t part = kv4_chunk_part_bytes(p->head_dim);
  if (!kv4_chunk_supported(p->head_dim, dtype, B, p->kv_heads, ka_columns(B, n_rows, Hq / p->kv_heads, dtype))) {
    const int64_t width = KA_MAX_WIDTH / (dtype == BQ_DT_F32 ? 2 : 1);
    int64_t runs = (int64_t)sm_count() * KA_MAX_TEAMS;
    if (runs > KA_MAX_RUNS) runs = KA_MAX_RUNS;
    part = runs * 2 * width * (p->head_dim + 4) * (int64_t)sizeof(float);
  }
  return KA_MAX_RUNS * 8 * (int64_t)sizeof(int) + part;
}

int bq_kv4_attention(const bq_kv4_pool* p, int layer, const void* q, int64_t ldq, void* out, int Hq, int dtype, const int32_t* slots,
                     const int32_t* pos, const int32_t* starts, int64_t B, int64_t n_rows, void* work, void* stream) {
  KaArgs a = {};
  int rc = kv4_view(p, layer, "bq_kv4_attention", &a.v);
  if (rc) return rc;
  if (dtype != BQ_DT_F32 && dtype != BQ_DT_BF16) return fail(BQ_ERR_ARG, "bq_kv4_attention: dtype must be BQ_DT_F32 or BQ_DT_BF16");
  if (Hq <= 0 || Hq % p->kv_heads) return fail(BQ_ERR_ARG, "bq_kv4_attention: query heads must be a multiple of the KV heads");
  if (B < 0 || B > p->max_seqs) return fail(BQ_ERR_ARG, "bq_kv4_attention: more sequences than the pool holds");
  const int rep = Hq / p->kv_heads;
  if (n_rows < 0 || n_rows * rep > (int64_t)1 << 29 || (!starts && n_rows != B))
    return fail(BQ_ERR_ARG, "bq_kv4_attention: bad number of rows (one per sequence without row ranges)");
  if (B == 0 || n_rows == 0) return BQ_OK;
  if (!q || !out || !pos || !work) return fail(BQ_ERR_ARG, "bq_kv4_attention: null pointer");
  if (kv4_misaligned(4, slots, starts, pos)) return fail(BQ_ERR_ARG, "bq_kv4_attention: slots, pos and starts must be aligned to their elements");
  const uintptr_t pair = dtype == BQ_DT_F32 ? 7 : 3;
  if (ldq < (int64_t)Hq * p->head_dim || (ldq & 1) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & pair) ||
      (reinterpret_cast<uintptr_t>(work) & 15))
    return fail(BQ_ERR_ARG, "bq_kv4_attention: rows of q and out must be aligned to two elements, those of q an even number of "
                            "elements apart and not overlap; "
                            "work must be 16-byte aligned");
  a.q = q; a.out = out; a.cut = static_cast<int*>(work); a.part = reinterpret_cast<float*>(a.cut + KA_MAX_RUNS * 8);
  a.ldq = ldq; a.n_rows = n_rows;
  a.slots = slots; a.pos = pos; a.starts = starts; a.status = status_word();
  a.B = (int)B; a.Hq = Hq; a.rep = rep;
  const int64_t cols = ka_columns(B, n_rows, rep, dtype);
  if (kv4_chunk_supported(p->head_dim, dtype, B, p->kv_heads, cols)) return kv4_chunk(a, (cudaStream_t)stream);
  return dtype == BQ_DT_F32 ? ka_run<float>(a, cols, (cudaStream_t)stream) : ka_run<__nv_bfloat16>(a, cols, (cudaStream_t)stream);
}

}  // extern "C"
