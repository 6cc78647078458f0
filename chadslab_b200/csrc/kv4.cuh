// Paged 4-bit KV cache: the layout of a block and what its kernels share.
//
// A pool is pages[n_pages][layers][kv_heads][page / 16][KV4_BLOCK(D)] bytes.  A block holds 16 consecutive positions of one
// head in one layer, NG = D / 32 quantisation groups:
//   K codes  256 * NG bytes | K scales 32 * NG bytes | V codes 256 * NG bytes | V scales 32 * NG bytes
// Codes are stored as mma.sync.m16n8k16 A fragments, one 32-bit word per lane and 16 x 16 tile, the two tiles of a group
// side by side (a lane's 8 bytes): attention reads them with one conflict-free 8-byte load per lane and group, and a word
// unpacks into the four fragment registers r0 = w & 0x000F000F, r1 = w & 0x00F000F0, r2, r3 = the same of w >> 8.
//   K tile: row = position (g, g + 8), k = dimension.   r0 = (g, low k), r1 = (g, high k), r2 = (g + 8, low), r3 = (g + 8, high)
//   V tile: row = dimension (g, g + 8), k = position.   r0 = (g, low k), r1 = (g + 8, low k), r2 = (g, high), r3 = (g + 8, high)
// In both the nibbles of one position fill whole bytes, so that appending a position never reads what is there.
// A nibble n = code + 8 in bits 0-3 (r0, r2) is the fp16 subnormal n * 2^-24, in bits 4-7 (r1, r3) n * 2^-20, and with the
// exponent of 1024 or-ed in 1024 + n or 1024 + 16 n.
#pragma once
#include "common.cuh"

namespace bq {

constexpr int KV4_MAX_SEQS = 8192;        // per pool: the batch calls resolve slots that occur twice in shared memory
constexpr int KV4_ROWS = 16;              // positions of a block
constexpr int KV4_GROUP_BYTES = 576;      // a block's bytes per group: 2 * (256 + 32)
__host__ __device__ constexpr int kv4_block_bytes(int D) { return KV4_GROUP_BYTES * (D / GROUP); }
__host__ __device__ constexpr int kv4_kscale_off(int D) { return 256 * (D / GROUP); }
__host__ __device__ constexpr int kv4_v_off(int D) { return 288 * (D / GROUP); }
__host__ __device__ constexpr int kv4_vscale_off(int D) { return 544 * (D / GROUP); }

// What the kernels read of a pool, and the layer they work on
struct Kv4View {
  uint8_t* pages;
  const int32_t* tables;
  int64_t n_pages, page_bytes, layer_off;
  int max_seqs, max_pages, Hkv, D, page_log2;
  __device__ __forceinline__ int page_blocks_log2() const { return page_log2 - 4; }
  // block `blk` (position / 16) of a sequence with table row `row`, head h; nullptr: the table holds no such page
  __device__ __forceinline__ uint8_t* block(const int32_t* row, int blk, int h) const {
    const int pb = page_blocks_log2();
    const int id = row[blk >> pb];
    if ((unsigned)id >= (uint64_t)n_pages) return nullptr;
    return pages + (int64_t)id * page_bytes + layer_off +
           ((int64_t)h * (1 << pb) + (blk & ((1 << pb) - 1))) * kv4_block_bytes(D);
  }
};

int kv4_check(const bq_kv4_pool* p, const char* what);                     // kv4_pages.cu: 0, or BQ_ERR_* with the message set
int kv4_view(const bq_kv4_pool* p, int layer, const char* what, Kv4View* out);
// element addresses: a pointer that is not a multiple of its elements' size would fault on the device
inline bool kv4_misaligned(size_t size, const void* a, const void* b = nullptr, const void* c = nullptr) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & (size - 1)) != 0;
}

#ifdef __CUDACC__
// The kernels of the cache may start before the kernel that wrote their inputs has finished (pdl_wait orders them), so nothing
// here is declared __restrict__ or read through the non-coherent path: that is for memory nobody writes while a kernel lives.
__device__ __forceinline__ uint4 kv4_load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// The rows of one sequence of a batch call.  n < 0: refused (bad ranges, recorded in the status word); pos < 0: skipped.
struct Kv4Seq {
  int slot, row0, n, pos;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4View& v, const int32_t* slots, const int32_t* pos, const int32_t* starts, int b,
                                          int64_t T, int* status) {
  Kv4Seq s;
  s.slot = slots ? slots[b] : b;
  s.row0 = starts ? starts[b] : b;
  s.n = starts ? starts[b + 1] - s.row0 : 1;
  s.pos = pos[b];
  const bool rows_ok = s.row0 >= 0 && s.n >= 0 && (int64_t)s.row0 + s.n <= T;
  const bool place_ok = (unsigned)s.slot < (unsigned)v.max_seqs && s.pos + (int64_t)s.n <= ((int64_t)v.max_pages << v.page_log2);
  if (!rows_ok || !place_ok) {
    *(volatile int*)status = (int)BQ_ERR_ARG;
    if (!rows_ok) s.n = 0;
    s.pos = -1;
  }
  return s;
}
// The sequence that work item `item` belongs to, where sequence b owns the items from (starts[b] >> 4) + 2 b on: enough of
// them for every 16-position block that its rows can touch.  All lanes of the warp take part.
__device__ __forceinline__ int kv4_item_base(const int32_t* starts, int b) { return (starts[b] >> 4) + 2 * b; }
__device__ __forceinline__ int kv4_item_seq(const int32_t* starts, int B, int item) {
  int lo = 0, n = B;                       // the answer is in [lo, lo + n)
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int b = lo + lane * step;
    const bool le = b < lo + n && (lane == 0 || kv4_item_base(starts, b) <= item);
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
    n = min(step, lo + n - (lo + last * step));
    lo += last * step;
  }
  return lo;
}
// scale and code of one group: scale = fp16(min(absmax * (1/7), 65504)), code = clip(rint(x / scale), +-7).  The weight
// quantiser's rule but for two things: absmax is multiplied by the fp32 reciprocal of 7, and a NaN makes its whole group NaN
// instead of vanishing in the maximum.  The reciprocal is what torch computes for a CUDA tensor divided by the number 7 (a
// quotient would differ from it in the last bit of about one scale in 10^4): a cache written by torch code has the same bytes.
__device__ __forceinline__ float kv4_absmax(float a, float b) {       // fmaxf that keeps NaN (bits of |x| order like |x|)
  const uint32_t x = __float_as_uint(a) & 0x7FFFFFFFu, y = __float_as_uint(b) & 0x7FFFFFFFu;
  return __uint_as_float(x > y ? x : y);
}
__device__ __forceinline__ __half kv4_scale(float amax) {
  const float s = __fmul_rn(amax, 1.0f / 7.0f);
  return __float2half_rn(s > 65504.0f ? 65504.0f : s);
}
#endif

}  // namespace bq
