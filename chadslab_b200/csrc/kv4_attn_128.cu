// Attention over the 4-bit KV cache, head_dim 128: the narrowest variant that holds a sequence's columns
// (see kv4_attn.cuh); more than eight go eight at a time, as at head_dim 256.
#include "kv4_attn.cuh"

namespace bq {

template <typename T> static int pick(const KaArgs& a, int64_t cols, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (cols <= 1) return ka_launch<T, 4, 1>(a, s);
  if (cols <= 2) return ka_launch<T, 4, 2>(a, s);
  if (cols <= 4) return ka_launch<T, 4, 4>(a, s);
  return ka_launch<T, 4, 8>(a, s);
}
template <> int ka_pick<float, 4>(const KaArgs& a, int64_t cols, cudaStream_t s) { return pick<float>(a, cols, s); }
template <> int ka_pick<__nv_bfloat16, 4>(const KaArgs& a, int64_t cols, cudaStream_t s) { return pick<__nv_bfloat16>(a, cols, s); }

}  // namespace bq
