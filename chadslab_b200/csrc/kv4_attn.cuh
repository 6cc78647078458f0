// Attention over the paged 4-bit KV cache on the warp-level tensor path (mma.sync m16n8k16, fp16 in, fp32 accumulate).
//   o[i, h] = sum_p softmax_p(q[i, h] . K[p] / sqrt(D)) V[p],   p <= position of row i
//
// Bound: HBM.  A position costs 1.125 D bytes per KV head; the kernel streams them once per column tile, a column being
// one (row, query head) of the KV head, and everything else stays in registers and shared memory.
//
// Codes to operands.  The codes lie in fragment order (kv4.cuh): a lane's 32-bit word is its whole A fragment of a 16 x 16
// tile, one mask (and a shift for half of them) away from four pairs of codes.
//   * Values, and keys of fp32 rows: w & 0x000F000F | 0x6400.. is a pair of fp16 numbers 1024 + n (n = code + 8), w &
//     0x00F000F0 | 0x6400.. a pair 1024 + 16 n; one packed subtraction leaves the code, or 16 times the code, exactly.
//   * Keys of bf16 rows: w & 0x000F000F IS a pair of fp16 subnormals n * 2^-24, w & 0x00F000F0 a pair n * 2^-20, and the +8 is
//     taken off by starting the accumulator at -8 * sum q: five integer instructions for eight codes and nothing else.  The
//     matrix unit aligns products by their exponents, which for a subnormal lie above its leading bit: a sum is good to about
//     2^-17 of its largest term instead of 2^-24 (measured: fp32 rows lost their last bits to it).  A score needs no more
//     for a bf16 result; for the values the start would be many times the result of a long context.
// What carries 16 times as much (the high half of a tile's dimensions for keys, rows 8-15 for values) meets q / 16, or is
// divided by 16 at the end.  A key group's scale multiplies its sum in fp32; the scale of (position, group) of the values
// multiplies the weight before it becomes the B operand.
// q is scaled per column by a power of two so that fp16 holds it exactly (bf16 has 8 bits); fp32 rows take two columns, the
// value and its remainder times 2^11 (22 bits), and so do their weights.
//
// Few columns (one query head per KV head: one).  m16n8k16 has 8 columns, so NC < 8 columns leave room for up to 8 / NC groups
// side by side: column n = group * NC + c of the B operand is zero outside its group's dimensions, one accumulator tile then holds
// 8 / NC groups' sums, each still apart for its scale; weights times scales of 8 / NC groups share one B fragment likewise.
//
// Softmax runs in the exp2 domain with a reference R per column that lags behind the maximum: weights are 2^(s - R), R = max -
// A, and R moves only when a weight would exceed 2^(A + 4) (A = 11: weights up to 2^15, 2^-24 is the smallest fp16).  A
// drops when weight * scale overflows, i.e. for values far above one.  Weights end at 2^(A + 4): where scores are so large that
// fp32 has steps of 16 and more (2^27), R cannot be set closer to their maximum; it is rounded down.
//
// Small values.  As long as no value scale was above 1/16, the scales of a step are raised in the stage by a power of two
// (ka_raise): the products would lose in fp16's subnormals what the weights still hold.  What weights and products lose is
// then at most 2^-31.9 of the largest weight times the largest value per position, however small the values are.  Looking at
// the first step's scales costs 1 to 2 % (64 x 2048 positions x 16 heads of 256: 101.5 -> 103.7 us, ragged batch 66.0 -> 67.1),
// raising those of every step a quarter (values around 0.01: 105 -> 131 us; 32 / 4 heads of 128 28 -> 32).
//
// Work.  The tiles (128 positions, or 64 where two steps of 32 per warp do not fit into shared memory) of all (sequence, KV
// head, column tile) segments form one list that is cut into equal runs, one per team of four warps: ragged batches and few
// long sequences fill the machine alike.  The teams of an SM (two to four) are one CTA: as CTAs of their own some found no
// contiguous registers beside the preceding kernel's and started when the others were done, which doubled the kernel's time
// (8 of 444 late: 169 us for 100 us of work).  A warp takes 32 (16) positions of every tile through its own ring of bulk copies
// (no barrier between warps inside a segment).  A segment that lies in one run is finished there; one that is cut leaves
// partial states in the caller's scratch, which a second kernel merges in run order.  Every result has one order of additions:
// repeated calls give the same bits.
//
// Measured (device time of graph replays; short loops, in long ones the power cap lowers the clock): 64 x 2048 positions x 16
// heads of 256 105 us = 5.75 TB/s (calls in a loop of seconds 121), ragged batch of 96 up to 8000 positions with 32 / 4 heads
// of 128 68.5 us = 3.3 TB/s, two contexts of 131072 with the same heads 46.4 us = 3.25 TB/s (eight columns per position block:
// bound by its instructions, 342 per block).
#pragma once
#include "kv4.cuh"
#include "kv4_ring.h"

namespace bq {

constexpr int KA_WARPS = 4;                           // of a team: the warps that work on one run
constexpr int KA_THREADS = KA_WARPS * 32;
constexpr uint64_t KA_WAIT_NS = 2000000000ull;        // bound of the wait for a copy; a warp runs into it once, and once more for
                                                      // all that is still under way when it leaves

// x / d for 0 <= x < 2^31
struct KaDiv {
  uint32_t mul, shift, d;
  __device__ __forceinline__ int operator()(int x) const { return (int)((__umulhi(mul, (uint32_t)x) + (uint32_t)x) >> shift); }
};
inline KaDiv ka_div(uint32_t d) {
  uint32_t s = 0;
  while (((uint64_t)1 << s) < d) ++s;
  return KaDiv{(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1), s, d};
}

struct KaArgs {
  Kv4View v;
  const void* q;
  void* out;
  float* part;                                        // [runs][2][HC * (D + 4)]: outputs, then (reference, sum) pairs
  int* cut;                                           // [runs][8]: the segment that a run begins and does not finish
  int64_t ldq, n_rows;
  const int32_t *slots, *pos, *starts;
  int* status;
  int B, Hq, rep;
  KaDiv by_rep, by_row;                               // query heads of a KV head; columns of a row: those times sl
  int width_log2, sl;                                 // columns of a tile; columns per (row, head): 1, or 2 for fp32 rows
  int tile_log2;                                      // positions of a tile: 16 or 32 per warp
};

// ---- the list of tiles ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ int ka_col_tiles(const KaArgs& a, const Kv4Seq& s) {      // rows * columns of a row < 2^31
  return s.n > 0 && s.pos >= 0 ? (s.n * (int)a.by_row.d + (1 << a.width_log2) - 1) >> a.width_log2 : 0;
}
__device__ __forceinline__ int ka_end(const KaArgs& a, const Kv4Seq& s, int ct) {      // positions that column tile ct sees
  const int rows = a.by_row(((ct + 1) << a.width_log2) - 1) + 1;
  return s.pos + (rows < s.n ? rows : s.n);
}
__device__ __forceinline__ int ka_tiles(const KaArgs& a, const Kv4Seq& s, int ct) {
  return (ka_end(a, s, ct) + (1 << a.tile_log2) - 1) >> a.tile_log2;
}
// Tiles of one KV head of each lane's sequence.  A sequence with many column tiles is summed by the whole warp.
__device__ __forceinline__ int64_t ka_head_tiles(const KaArgs& a, const Kv4Seq& s) {
  const int lane = threadIdx.x & 31, cts = ka_col_tiles(a, s);
  int64_t n = 0;
  if (cts <= 4)
    for (int ct = 0; ct < cts; ++ct) n += ka_tiles(a, s, ct);
  for (unsigned many = __ballot_sync(0xffffffffu, cts > 4); many; many &= many - 1) {
    const int src = __ffs(many) - 1;
    Kv4Seq o = {};
    o.n = __shfl_sync(0xffffffffu, s.n, src);
    o.pos = __shfl_sync(0xffffffffu, s.pos, src);
    const int all = __shfl_sync(0xffffffffu, cts, src);
    int64_t sum = 0;
    for (int ct = lane; ct < all; ct += 32) sum += ka_tiles(a, o, ct);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == src) n = sum;
  }
  return n;
}
// The column tile that holds tile *rem of one KV head; *rem becomes the tile within it.
__device__ __forceinline__ int ka_find_col_tile(const KaArgs& a, const Kv4Seq& s, int* rem) {
  const int lane = threadIdx.x & 31, cts = ka_col_tiles(a, s);
  int r = *rem, ct0 = 0;
  if (cts > 1) {
    for (;; ct0 += 32) {
      const int n = ct0 + lane < cts ? ka_tiles(a, s, ct0 + lane) : 0;
      int upto = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto > r);
      if (past || ct0 + 32 >= cts) {
        const int l = past ? __ffs(past) - 1 : 31;
        r -= __shfl_sync(0xffffffffu, upto - n, l);
        ct0 += l;
        break;
      }
      r -= __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  *rem = r;
  return ct0;
}
__device__ __forceinline__ Kv4Seq ka_seq(const KaArgs& a, int b) { return kv4_seq(a.v, a.slots, a.pos, a.starts, b, a.n_rows, a.status); }

// barrier of a team (1 + its number; 0 is the CTA's)
__device__ __forceinline__ void ka_sync(int team) { asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(KA_THREADS) : "memory"); }
__device__ __forceinline__ bool ka_sync_or(int team, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "bar.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(team + 1), "n"(KA_THREADS), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

struct KaPlace { int b, h, ct, tile; };               // a tile of the list
struct KaScan {
  int64_t part[KA_WARPS];
  int b, rem;
};
// inclusive sum of v over the team, *total = the sum of all
__device__ __forceinline__ int64_t ka_scan(int64_t v, KaScan* sc, int team, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % KA_WARPS;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  ka_sync(team);
  if (lane == 31) sc->part[warp] = v;
  ka_sync(team);
  int64_t t = 0;
#pragma unroll
  for (int w = 0; w < KA_WARPS; ++w) {
    if (w < warp) v += sc->part[w];
    t += sc->part[w];
  }
  *total = t;
  return v;
}
// Length of the list and of a run, and the place of the first tile of run `run` (false: the list ends before it).
template <typename T>
static __device__ bool ka_locate(const KaArgs& a, int runs, int run, int team, KaScan* sc, KaPlace* at, int* total, int* per) {
  const int tid = threadIdx.x % KA_THREADS;
  int64_t sum = 0, mine = 0, upto = 0, chunk;
  for (int b0 = 0; b0 < a.B; b0 += KA_THREADS) {
    const int b = b0 + tid;
    Kv4Seq s = {};
    if (b < a.B) s = ka_seq(a, b);
    mine = ka_head_tiles(a, s) * a.v.Hkv;
    upto = ka_scan(mine, sc, team, &chunk);
    sum += chunk;
    // rows of refused sequences are zero: the runs share them
    if (ka_sync_or(team, s.pos < 0 && s.n > 0))
      for (int j = 0; j < KA_THREADS && b0 + j < a.B; ++j) {
        if ((b0 + j) % runs != run) continue;
        const Kv4Seq z = ka_seq(a, b0 + j);
        if (z.pos >= 0) continue;
        const int64_t n = (int64_t)z.n * a.Hq * a.v.D;
        T* o = static_cast<T*>(a.out) + (int64_t)z.row0 * a.Hq * a.v.D;
        for (int64_t e = tid; e < n; e += KA_THREADS) o[e] = from_float<T>(0.0f);
      }
  }
  if (sum > 0x7FFFFFFF) {                              // weeks of work: not taken on
    *(volatile int*)a.status = (int)BQ_ERR_UNSUPPORTED;
    return false;
  }
  *total = (int)sum;
  *per = (int)(((unsigned)sum + runs - 1) / (unsigned)runs);
  const int64_t lo = (int64_t)run * *per;
  if (lo >= sum) return false;
  int64_t before = 0;
  for (int b0 = 0; b0 < a.B; b0 += KA_THREADS) {
    if (a.B > KA_THREADS) {                           // otherwise the sums of the loop above are still there
      const int b = b0 + tid;
      Kv4Seq s = {};
      if (b < a.B) s = ka_seq(a, b);
      mine = ka_head_tiles(a, s) * a.v.Hkv;
      upto = ka_scan(mine, sc, team, &chunk);
    }
    const int64_t from = before + upto - mine;
    if (lo >= from && lo < from + mine) { sc->b = b0 + tid; sc->rem = (int)(lo - from); }
    before += chunk;
    if (lo < before) break;
  }
  ka_sync(team);
  at->b = sc->b;
  int rem = sc->rem;
  const Kv4Seq s = ka_seq(a, at->b);
  const int head = __shfl_sync(0xffffffffu, (int)ka_head_tiles(a, s), 0);
  at->h = rem / head;
  rem -= at->h * head;
  at->ct = ka_find_col_tile(a, s, &rem);
  at->tile = rem;
  return true;
}

// ---- copies ----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ka_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ka_bar_init(uint32_t bar) { asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void ka_bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ka_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool ka_bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint64_t ka_now() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
static __device__ __noinline__ bool ka_bar_wait_long(uint32_t bar, uint32_t parity, uint64_t t0) {
  if (t0 == 0) t0 = ka_now();
  do {
    for (int i = 0; i < 1024; ++i)
      if (ka_bar_test(bar, parity)) return true;
  } while (ka_now() - t0 < KA_WAIT_NS);
  return false;
}
// lane 0 polls, the warp follows; false: the copy did not arrive in time (counted from t0, 0: from now)
__device__ __forceinline__ bool ka_bar_wait(uint32_t bar, uint32_t parity, int lane, uint64_t t0 = 0) {
  bool ok = true;
  if (lane == 0 && !ka_bar_test(bar, parity)) ok = ka_bar_wait_long(bar, parity, t0);
  return __all_sync(0xffffffffu, ok);
}

// ---- arithmetic --------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ka_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ka_mma_new(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {      // d = A x B
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t ka_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ka_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ka_min(float a, float b) {              // NaN stays
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint32_t ka_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 ka_half2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ uint32_t ka_pack(float lo, float hi) { return ka_bits(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ uint32_t ka_mul2(uint32_t a, uint32_t b) { return ka_bits(__hmul2(ka_half2(a), ka_half2(b))); }
__device__ __forceinline__ uint32_t ka_sub2(uint32_t a, uint32_t b) { return ka_bits(__hsub2(ka_half2(a), ka_half2(b))); }
// codes of the low / high nibble of bytes 0 and 2 as fp16, the latter times 16: 1032 = 0x6408, 1152 = 0x6480
__device__ __forceinline__ uint32_t ka_code(uint32_t w) { return ka_sub2(lop3_and_or(w, 0x000F000Fu, 0x64006400u), 0x64086408u); }
__device__ __forceinline__ uint32_t ka_code16(uint32_t w) { return ka_sub2(lop3_and_or(w, 0x00F000F0u, 0x64006400u), 0x64806480u); }
__device__ __forceinline__ float2 ka_q2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 ka_q2(const __nv_bfloat16* p) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ void ka_store2(float* p, float x, float y) { *reinterpret_cast<float2*>(p) = make_float2(x, y); }
__device__ __forceinline__ void ka_store2(__nv_bfloat16* p, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
}
constexpr float KA_LO = 1.0f / 2048.0f;               // weight of the second column of an fp32 row

// `vlim`: a power of two that no value scale so far exceeds, from 2^-15 on; 1 once there was one above 1/16.  Scales are raised by 1 / vlim.
constexpr float KA_VLIM0 = 1.0f / 32768.0f;
constexpr float KA_ORDINARY = 1.0f / 16.0f;
__device__ __forceinline__ float ka_vlim(float vlim, float top) {
  if (top <= vlim) return vlim;
  return top > KA_ORDINARY ? 1.0f : __uint_as_float((__float_as_uint(top) + 0x007FFFFFu) & 0x7F800000u);
}
__device__ __forceinline__ float ka_inverse(float two_to_the_k) { return __uint_as_float(0x7F000000u - __float_as_uint(two_to_the_k)); }
// Two value scales of a block, words of the layout (word w of a block: positions r, r + 1 of w % 8), those of positions
// `live` and behind replaced by zero
__device__ __forceinline__ uint32_t ka_live_scales(uint32_t x, int w, int live) {
  const int r = (w >> 1 & 3) * 2 + 8 * (w & 1);
  return (r < live ? x & 0x0000FFFFu : 0u) | (r + 1 < live ? x & 0xFFFF0000u : 0u);
}
// Whether one of the first value scales of a block (D / 32 * 8 words of them) is above 1/16: a warp's first look
template <int D> __device__ __forceinline__ bool ka_ordinary(const uint8_t* blk, int live) {
  const int w = (threadIdx.x & 31) % (D / GROUP * 8);
  const uint32_t x = ka_live_scales(*reinterpret_cast<const uint32_t*>(blk + kv4_vscale_off(D) + w * 4), w, live);
  return __any_sync(0xffffffffu, __hgt2_mask(ka_half2(x), __floats2half2_rn(KA_ORDINARY, KA_ORDINARY)) != 0u);
}
// Raises the value scales of `blocks` blocks (`live` positions) in a warp's stage; returns the new vlim
template <int D, int BLK>
__device__ __forceinline__ float ka_raise(uint8_t* stage, int blocks, int live, float vlim) {
  constexpr int WORDS = D / GROUP * 8;
  const int lane = threadIdx.x & 31;
  auto at = [&](int e) { return reinterpret_cast<uint32_t*>(stage + e / WORDS * BLK + kv4_vscale_off(D) + e % WORDS * 4); };
  auto scales = [&](int e) { return ka_live_scales(*at(e), e % WORDS, live - e / WORDS * KV4_ROWS); };
  __half2 top2 = __floats2half2_rn(0.0f, 0.0f);
  for (int e = lane; e < blocks * WORDS; e += 32) top2 = __hmax2(top2, ka_half2(scales(e)));
  float top = fmaxf(__low2float(top2), __high2float(top2));
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  vlim = ka_vlim(vlim, top);
  if (vlim == 1.0f) return vlim;
  const uint32_t up = ka_pack(ka_inverse(vlim), ka_inverse(vlim));
  for (int e = lane; e < blocks * WORDS; e += 32) *at(e) = ka_mul2(scales(e), up);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before the copy that will fill the stage again
  __syncwarp();
  return vlim;
}

// ---- variants ------------------------------------------------------------------------------------------------------------------
template <typename T, int NG, int NC> struct KaCfg {
  static constexpr int SL = sizeof(T) == 4 ? 2 : 1;
  static constexpr int D = NG * GROUP;
  static constexpr int GP = 8 / NC < NG ? 8 / NC : NG; // groups side by side in a fragment
  static_assert(NG % GP == 0, "whole fragments");
  static constexpr int NF = NG / GP;
  static constexpr int W = NC;                        // columns of a tile
  static constexpr int HC = W / SL;
  static_assert(W % SL == 0, "an fp32 row takes two columns");
  static constexpr int J = NC == 1 || SL == 2 ? 1 : 2;  // different (row, head) pairs among a lane's two columns
  static constexpr bool SUBNORMAL = SL == 1;          // keys as fp16 subnormals
  static constexpr int BLK = kv4_block_bytes(D);
  static constexpr int QG = NG % 4 == 0 ? NG / 4 : 1;  // groups that are merged over the warps at a time
  static constexpr int OSTR = QG * 32 + 4;            // row pitch of the merge buffer: a quad's columns hit different banks
  // teams of an SM, by the registers that a thread needs: 8 NG accumulators, 4 NG of q, and with eight columns 4 NG more for
  // starts and weights.  One team more at the price of spills is slower: 32 / 4 heads of 128 take 79 us with four teams of
  // 128 registers (200 bytes spilled) and 70 with three of 168 (ragged batch of 96).  That was measured with eight columns; with
  // two and four the same rule leaves 16 to 112 bytes spilled, which is not measured against fewer teams
  static constexpr int TEAMS = NG <= (NC == 8 ? 3 : 4) ? 4 : NG <= (NC == 8 ? 5 : 8) ? 3 : 2;
  static constexpr int FIXED = KA_WARPS * HC * OSTR * 4 + 2 * KA_WARPS * W * 4 + HC * 12 + (int)sizeof(KaScan) + 128;
  // a warp's step, one stage of its ring: two blocks if the ring then has two stages, else one
  static constexpr int ROOM = (232448 / TEAMS - FIXED) / KA_WARPS;
  static constexpr int STEP = ROOM / (2 * BLK + 8) >= 2 ? 2 : 1;
  static constexpr int TILE = KA_WARPS * STEP * KV4_ROWS;
  static constexpr int STAGE = STEP * BLK;
  static constexpr int STAGES = ROOM / (STAGE + 8) >= 4 ? 4 : ROOM / (STAGE + 8);
  static_assert(STAGES >= 2, "the ring needs two stages");
  static constexpr int SMEM = (KA_WARPS * STAGES * (STAGE + 8) + FIXED) / 128 * 128;      // of a team
  static constexpr int U = NF * NG <= 16 ? STEP : 1;  // blocks whose scores and weights are held at a time
};

template <typename T, int NG, int NC>
__global__ void __launch_bounds__((KaCfg<T, NG, NC>::TEAMS * KA_THREADS), 1) kv4_attention_kernel(const __grid_constant__ KaArgs a) {
  using C = KaCfg<T, NG, NC>;
  constexpr int D = C::D, SL = C::SL, GP = C::GP, NF = C::NF, W = C::W, HC = C::HC, S = C::STAGES, U = C::U, STEP = C::STEP, TILE = C::TILE, J = C::J;
  extern __shared__ __align__(128) uint8_t smem_all[];
  const int team = threadIdx.x / KA_THREADS, tid = threadIdx.x % KA_THREADS;
  const int run = team * gridDim.x + blockIdx.x, runs = gridDim.x * C::TEAMS;      // few runs: one per SM first
  uint8_t* smem = smem_all + team * C::SMEM;
  // [warps][S][STAGE] ring | [warps][S] barriers | merge buffer | reference and sum of every warp and column | scan
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + KA_WARPS * S * C::STAGE);
  float* s_o = reinterpret_cast<float*>(bars + KA_WARPS * S);  // [warps][HC][OSTR]
  float* s_ref = s_o + KA_WARPS * HC * C::OSTR;
  float* s_sum = s_ref + KA_WARPS * W;
  KaScan* scan = reinterpret_cast<KaScan*>(s_sum + KA_WARPS * W);
  int64_t* s_to = reinterpret_cast<int64_t*>(scan + 1);
  float* s_div = reinterpret_cast<float*>(s_to + HC);
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % KA_WARPS, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * S * C::STAGE;
  const uint32_t bar0 = ka_smem(bars + warp * S);
  if (lane < S) ka_bar_init(bar0 + lane * 8);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();
  ka_sync(team);

  int* cut = a.cut + (int64_t)run * 8;
  if (tid == 0) cut[0] = -1;
  KaPlace at;
  int total, per;
  if (!ka_locate<T>(a, runs, run, team, scan, &at, &total, &per)) return;
  const int lo = run * per;
  int left = total - lo < per ? total - lo : per;              // tiles of this run that are still to do

  Kv4Seq seq = ka_seq(a, at.b);
  int end = ka_end(a, seq, at.ct), tiles = (end + TILE - 1) / TILE;
  int cts = ka_col_tiles(a, seq);
  Kv4Ring<S> copies;
  const int pb = a.v.page_blocks_log2();
  const int32_t* row = a.v.tables + (int64_t)seq.slot * a.v.max_pages;
  // One lane requests this warp's blocks of a tile into stage `st`; `blocks` = blocks of the segment
  auto request = [&](const int32_t* row, int h, int tile, int blocks, int st) {
    const uint32_t bar = bar0 + st * 8, dst = ka_smem(ring + st * C::STAGE);
    const int b0 = (tile * KA_WARPS + warp) * STEP, n = blocks - b0 < STEP ? blocks - b0 : STEP;
    ka_bar_expect(bar, n * C::BLK);
    auto load = [&](int blk, int count, uint32_t to) {
      uint32_t id = (uint32_t)row[blk >> pb];
      if (id >= (uint64_t)a.v.n_pages) {                       // no such page: recorded, the result is undefined
        *(volatile int*)a.status = (int)BQ_ERR_ARG;
        id = 0;
      }
      const uint32_t in = ((uint32_t)h << pb) + (blk & ((1 << pb) - 1));
      ka_bulk_load(to, a.v.pages + (int64_t)id * a.v.page_bytes + (a.v.layer_off + (int64_t)in * C::BLK), count * C::BLK, bar);
    };
    if (STEP == 1 || pb > 0) load(b0, n, dst);                 // a page holds them all
    else
      for (int j = 0; j < n; ++j) load(b0 + j, 1, dst + j * C::BLK);
  };
  // The ring is empty: the first steps of a piece, one lane each
  auto fill = [&](const int32_t* row, int h, int first, int steps, int blocks) {
    const int n = copies.room(steps);
    if (lane < n) request(row, h, first + lane, blocks, copies.stage(lane));
    copies.requested(n);
    return n;
  };
  int first = at.tile;
  int last = tiles - first < left ? tiles : first + left;         // this piece: tiles first .. last - 1
  int blocks = (end + KV4_ROWS - 1) / KV4_ROWS;
  auto my_steps = [&]() {                                      // tiles of the piece in which this warp has a block
    const int full = (blocks - warp * STEP + KA_WARPS * STEP - 1) / (KA_WARPS * STEP);
    const int n = (full < last ? full : last) - first;
    return n > 0 ? n : 0;
  };
  int mine = my_steps();                                       // steps of this piece: all, and requested
  int ahead = fill(row, at.h, first, mine, blocks);

  while (true) {
    // ---- the columns: q as B fragments ------------------------------------------------------------------------------------
    uint32_t bq[2 * NG][2];
    float start[NF][2], kappa[2];
    int vis[2];
    const int cols = seq.n * a.rep * SL;
    {
      const int c = NC < 8 ? g % NC : g, gi = NC < 8 ? g / NC : 0;
      const int col = at.ct * W + c, rh = col / SL, i = a.by_rep(rh);
      const bool ok = col < cols;
      const T* qp = static_cast<const T*>(a.q) + (ok ? (int64_t)(seq.row0 + i) * a.ldq + (int64_t)(at.h * a.rep + rh - i * a.rep) * D : 0) + 2 * t;
      // this lane's groups are f * GP + gi; the loads are all under way before the first is used
      float2 x[NF][4];
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int k = 0; k < 4; ++k) x[f][k] = ok && gi < GP ? ka_q2(qp + (f * GP + gi) * 32 + k * 8) : make_float2(0.0f, 0.0f);
      float big = 0.0f;
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int k = 0; k < 4; ++k) big = fmaxf(big, fmaxf(fabsf(x[f][k].x), fabsf(x[f][k].y)));
#pragma unroll
      for (int off = 1; off < 32; off <<= 1)
        if (off < 4 || off >= 4 * NC) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
      int k2 = 13 - ((int)(__float_as_uint(big) >> 23) - 127);          // big * 2^k2 is in [2^13, 2^14)
      k2 = k2 > 100 ? 100 : k2 < -114 ? -114 : k2;
      const float up = __uint_as_float((uint32_t)(127 + k2) << 23);
      // queries past 2^113: scores of that size are all or nothing, so they may come out 2^-14 of what they are
      k2 = k2 < -100 ? -100 : k2;
      const bool second = SL == 2 && (col & 1);
      float sum[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        sum[f] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // k = 2 * tile + (high k): the high half meets codes that carry 16 times as much
          const float m = (k & 1) ? up * 0.0625f : up;
          float2 z = make_float2(x[f][k].x * m, x[f][k].y * m);
          if (second) {
            z.x = (z.x - __half2float(__float2half_rn(z.x))) * 2048.0f;
            z.y = (z.y - __half2float(__float2half_rn(z.y))) * 2048.0f;
          }
          const __half2 hx = __floats2half2_rn(z.x, z.y);
          if (C::SUBNORMAL) {
            const float2 back = __half22float2(hx);
            sum[f] += (back.x + back.y) * ((k & 1) ? 16.0f : 1.0f);
          }
#pragma unroll
          for (int o = 0; o < GP; ++o) bq[2 * (f * GP + o) + (k >> 1)][k & 1] = GP == 1 || o == gi ? ka_bits(hx) : 0u;
        }
      }
      // what the accumulator layout needs of columns 2t and 2t + 1
      const float kap = __uint_as_float((uint32_t)(127 - k2) << 23) * ((C::SUBNORMAL ? 16777216.0f : 1.0f) * 1.4426950408889634f) * rsqrtf((float)D);
      const int see = ok ? seq.pos + i : 0x7FFFFFFF;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        kappa[j] = __shfl_sync(0xffffffffu, kap, (2 * t + j) * 4);
        vis[j] = __shfl_sync(0xffffffffu, see, (2 * t + j) * 4);
      }
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        float z = sum[f];
        z += __shfl_xor_sync(0xffffffffu, z, 1);
        z += __shfl_xor_sync(0xffffffffu, z, 2);
        z *= -8.0f / 16777216.0f;                              // (SUBNORMAL; else there is nothing to take off)
#pragma unroll
        for (int j = 0; j < 2; ++j) start[f][j] = __shfl_sync(0xffffffffu, z, (2 * t + j) * 4);
      }
    }
    const int all_see = seq.pos + a.by_row(at.ct * W);        // every column sees positions up to here

    // ---- the positions ----------------------------------------------------------------------------------------------------
    float acc[2 * NG][4], ref[2], l[2];
    float A = 11.0f;
    float vlim = KA_VLIM0;                                     // acc carries the 1 / vlim of the scales
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      // a column without a row has no weight anywhere: it must not take part in the search for a reference
      ref[j] = vis[j] == 0x7FFFFFFF ? 3.0e38f : -3.0e38f;
      l[j] = 0.0f;
    }
    for (int i = 0; i < mine; ++i) {
      // a copy that does not arrive: recorded; this warp takes no further part but in the merges
      if (!copies.arrived([&](int st, uint32_t parity) { return ka_bar_wait(bar0 + st * 8, parity, lane); })) {
        *(volatile int*)a.status = (int)BQ_ERR_TIMEOUT;
        break;
      }
      uint8_t* stage = ring + copies.take * C::STAGE;
      const int step0 = ((first + i) * KA_WARPS + warp) * STEP * KV4_ROWS;
      if (vlim < 1.0f) {
        const float was = vlim;
        const int live = end - step0;
        vlim = ka_ordinary<D>(stage, live) ? 1.0f : ka_raise<D, C::BLK>(stage, live <= KV4_ROWS ? 1 : STEP, live, was);
        const float lower = was * ka_inverse(vlim);
#pragma unroll
        for (int x = 0; x < 2 * NG; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[x][j] *= lower;
      }
#pragma unroll 1
      for (int u0 = 0; u0 < STEP; u0 += U) {
        if (U == 1 && u0 && step0 + KV4_ROWS >= end) break;    // no second block
        const uint8_t* blk0 = stage + u0 * C::BLK;
        const int p0 = step0 + u0 * KV4_ROWS;
        // scores
        float s[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint8_t* blk = blk0 + u * C::BLK;
          uint2 kq0, kq1;
#pragma unroll
          for (int f = 0; f < NF; ++f) {
            float c[4];
            if (C::SUBNORMAL) {
              c[0] = c[2] = start[f][0];
              c[1] = c[3] = start[f][1];
            }
#pragma unroll
            for (int gi = 0; gi < GP; ++gi) {
              const int G = f * GP + gi;
              const uint2 w2 = *reinterpret_cast<const uint2*>(blk + G * 256 + lane * 8);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w = h ? w2.y : w2.x, x = w >> 8;
                uint32_t r0, r1, r2, r3;
                if (C::SUBNORMAL) {
                  r0 = w & 0x000F000Fu; r1 = w & 0x00F000F0u; r2 = x & 0x000F000Fu; r3 = x & 0x00F000F0u;
                } else {
                  r0 = ka_code(w); r1 = ka_code16(w); r2 = ka_code(x); r3 = ka_code16(x);
                }
                if (!C::SUBNORMAL && gi == 0 && h == 0) ka_mma_new(c, r0, r2, r1, r3, bq[2 * G][0], bq[2 * G][1]);
                else ka_mma(c, r0, r2, r1, r3, bq[2 * G + h][0], bq[2 * G + h][1]);
              }
            }
            // scales of rows g and g + 8: of the column's group, or (NC == 1) of the two columns' groups
            const __half* ks = reinterpret_cast<const __half*>(blk + kv4_kscale_off(D));
            float2 k0, k1;
            if (NC == 1) {
              const int G = f * GP + (2 * t < GP ? 2 * t : 0);         // columns past the groups hold zeros
              k0 = __half22float2(*reinterpret_cast<const __half2*>(ks + g * NG + G));
              k1 = __half22float2(*reinterpret_cast<const __half2*>(ks + (g + 8) * NG + G));
            } else if (NC == 8 && NG % 4 == 0) {               // four groups by one load per row
              if (f % 4 == 0) {
                kq0 = *reinterpret_cast<const uint2*>(ks + g * NG + f);
                kq1 = *reinterpret_cast<const uint2*>(ks + (g + 8) * NG + f);
              }
              const float2 x0 = __half22float2(ka_half2(f % 4 < 2 ? kq0.x : kq0.y)), x1 = __half22float2(ka_half2(f % 4 < 2 ? kq1.x : kq1.y));
              k0.x = k0.y = f % 2 ? x0.y : x0.x;
              k1.x = k1.y = f % 2 ? x1.y : x1.x;
            } else {
              const int at_col = 2 * t / NC, G = f * GP + (at_col < GP ? at_col : 0);
              k0.x = k0.y = __half2float(ks[g * NG + G]);
              k1.x = k1.y = __half2float(ks[(g + 8) * NG + G]);
            }
            s[u][0] = f ? fmaf(k0.x, c[0], s[u][0]) : k0.x * c[0];
            s[u][1] = f ? fmaf(k0.y, c[1], s[u][1]) : k0.y * c[1];
            s[u][2] = f ? fmaf(k1.x, c[2], s[u][2]) : k1.x * c[2];
            s[u][3] = f ? fmaf(k1.y, c[3], s[u][3]) : k1.y * c[3];
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float* z = s[u];
          if (NC == 1) {
            z[0] += z[1];
            z[2] += z[3];
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              z[j] += __shfl_xor_sync(0xffffffffu, z[j], 1);
              z[j] += __shfl_xor_sync(0xffffffffu, z[j], 2);
              z[j + 1] = z[j];
            }
          } else if (NC < 8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (NC == 2) z[j] += __shfl_xor_sync(0xffffffffu, z[j], 1);
              z[j] += __shfl_xor_sync(0xffffffffu, z[j], 2);
            }
          }
          if (SL == 2) {
            z[0] = z[1] = z[0] + z[1] * KA_LO;
            z[2] = z[3] = z[2] + z[3] * KA_LO;
          }
        }
        const bool masked = p0 + U * KV4_ROWS - 1 > all_see;   // positions past the end, or past a column's own
        if (masked) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if ((J == 2 || !(j & 1)) && p0 + u * KV4_ROWS + g + (j >> 1) * 8 > vis[j & 1]) s[u][j] = -INFINITY;
        }
        // weights; wv = weight * scale of the values, the B fragments of the second product
        float p[U][4];
        uint32_t wv[U][NF][2];
#pragma unroll 1
        for (int tries = 0;; ++tries) {
          float high = -INFINITY;
          __half2 top = __floats2half2_rn(0.0f, 0.0f);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint8_t* vsc = blk0 + u * C::BLK + kv4_vscale_off(D) + (g / NC < GP ? g / NC : 0) * 32 + t * 8;
            {
              float* w = p[u];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (J == 1 && (j & 1)) { w[j] = w[j - 1]; continue; }
                w[j] = fmaf(s[u][j], kappa[j & 1], -ref[j & 1]);
                high = fmaxf(high, w[j]);
                w[j] = ka_exp2(ka_min(w[j], A + 4.0f));
              }
              uint32_t m0, m1;                                 // rows g, g + 8: columns 2t, 2t + 1
              if (SL == 1) {
                m0 = ka_pack(w[0], w[1]);
                m1 = ka_pack(w[2], w[3]);
              } else {
                const float h0 = __half2float(__float2half_rn(w[0])), h1 = __half2float(__float2half_rn(w[2]));
                m0 = ka_pack(h0, (w[0] - h0) * 2048.0f);
                m1 = ka_pack(h1, (w[2] - h1) * 2048.0f);
              }
              m0 = ka_transpose(m0);                           // column g: positions 2t, 2t + 1
              m1 = ka_transpose(m1);                           //           positions 2t + 8, 2t + 9
              if (SL == 1) {
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                  const uint2 vs = *reinterpret_cast<const uint2*>(vsc + f * GP * 32);
                  wv[u][f][0] = ka_mul2(m0, vs.x);
                  wv[u][f][1] = ka_mul2(m1, vs.y);
                }
                if (masked) {                                  // a scale behind the last position can be anything: no weight, no product
                  const uint32_t live0 = __hne2_mask(ka_half2(m0), __floats2half2_rn(0.0f, 0.0f));
                  const uint32_t live1 = __hne2_mask(ka_half2(m1), __floats2half2_rn(0.0f, 0.0f));
#pragma unroll
                  for (int f = 0; f < NF; ++f) { wv[u][f][0] &= live0; wv[u][f][1] &= live1; }
                }
#pragma unroll
                for (int f = 0; f < NF; ++f) top = __hmax2(top, __hmax2(ka_half2(wv[u][f][0]), ka_half2(wv[u][f][1])));
              } else {
                // the partner lane holds the other half of the same weight: 22 bits times the scale, split again
                const uint32_t o0 = __shfl_xor_sync(0xffffffffu, m0, 4), o1 = __shfl_xor_sync(0xffffffffu, m1, 4);
                const bool odd = g & 1;
                const float2 a0 = __half22float2(ka_half2(odd ? o0 : m0)), b0 = __half22float2(ka_half2(odd ? m0 : o0));
                const float2 a1 = __half22float2(ka_half2(odd ? o1 : m1)), b1 = __half22float2(ka_half2(odd ? m1 : o1));
                const float w4[4] = {a0.x + b0.x * KA_LO, a0.y + b0.y * KA_LO, a1.x + b1.x * KA_LO, a1.y + b1.y * KA_LO};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                  const uint2 vs = *reinterpret_cast<const uint2*>(vsc + f * GP * 32);
                  const float2 va = __half22float2(ka_half2(vs.x)), vb = __half22float2(ka_half2(vs.y));
                  const float v4[4] = {va.x, va.y, vb.x, vb.y};
                  float z[4];
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    z[j] = w4[j] == 0.0f ? 0.0f : w4[j] * v4[j];
                    const float h = __half2float(__float2half_rn(z[j]));
                    if (h > 60000.0f) top = __floats2half2_rn(65504.0f, 65504.0f);
                    z[j] = odd ? (z[j] - h) * 2048.0f : h;
                  }
                  wv[u][f][0] = ka_pack(z[0], z[1]);
                  wv[u][f][1] = ka_pack(z[2], z[3]);
                }
              }
            }
          }
          const bool large = fmaxf(__low2float(top), __high2float(top)) > 60000.0f;
          if (!__any_sync(0xffffffffu, high > A + 4.0f || large) || tries == 8) break;
          // The reference moves up to the maximum so far; if after that a weight times its scale leaves fp16, all weights become
          // 16 times smaller.
          if (tries && !__any_sync(0xffffffffu, large)) break;        // (the limit above holds the weights)
          const float drop = tries ? 4.0f : 0.0f;
          A -= drop;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (J == 1 && j) {
                ref[1] = ref[0];
                continue;
              }
              float m = -INFINITY;
#pragma unroll
              for (int u = 0; u < U; ++u) m = fmaxf(m, fmaxf(s[u][j], s[u][j + 2]));
              m = __fmul_rd(m, kappa[j]);
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              const float r = fmaxf(ref[j] + drop, m - A), corr = ka_exp2(ref[j] - r);
              ref[j] = r;
              l[j] *= corr;
#pragma unroll
              for (int x = 0; x < 2 * NG; ++x) {
                acc[x][j] *= corr; acc[x][j + 2] *= corr;
                if (J == 1) { acc[x][1] *= corr; acc[x][3] *= corr; }
              }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          l[0] += p[u][0] + p[u][2];
          if (J == 2) l[1] += p[u][1] + p[u][3];
        }
        // Values.  The matrix unit truncates its sums, which over a long context adds up to a bias of 2^-25 per step: fp32 rows
        // add a step's sum to the accumulators themselves, rounded to nearest (4096 positions and more: 3.5e-6 -> 3e-7 off).
        if (SL == 2) {
#pragma unroll
          for (int G = 0; G < NG; ++G) {
            float sum[2][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const uint2 w2 = *reinterpret_cast<const uint2*>(blk0 + u * C::BLK + kv4_v_off(D) + G * 256 + lane * 8);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w = h ? w2.y : w2.x, x = w >> 8;
                const uint32_t r0 = ka_code(w), r1 = ka_code16(w), r2 = ka_code(x), r3 = ka_code16(x);
                if (u == 0) ka_mma_new(sum[h], r0, r1, r2, r3, wv[u][G / GP][0], wv[u][G / GP][1]);
                else ka_mma(sum[h], r0, r1, r2, r3, wv[u][G / GP][0], wv[u][G / GP][1]);
              }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[2 * G + h][j] += sum[h][j];
          }
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int G = 0; G < NG; ++G) {
              const uint2 w2 = *reinterpret_cast<const uint2*>(blk0 + u * C::BLK + kv4_v_off(D) + G * 256 + lane * 8);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w = h ? w2.y : w2.x, x = w >> 8;
                const uint32_t r0 = ka_code(w), r1 = ka_code16(w), r2 = ka_code(x), r3 = ka_code16(x);
                ka_mma(acc[2 * G + h], r0, r1, r2, r3, wv[u][G / GP][0], wv[u][G / GP][1]);
              }
            }
        }
      }
      copies.consumed();
      __syncwarp();                                            // the stage has been read by every lane
      if (ahead < mine) {
        if (lane == 0) request(row, at.h, first + ahead, blocks, copies.put);
        copies.requested(1);
        ++ahead;
      }
    }

    // ---- where this run goes next: its first copies travel while this piece is merged ------------------------------------------
    const KaPlace was = at;
    const Kv4Seq was_seq = seq;
    const bool begins = first == 0, ends = last == tiles;
    const int was_last = last, was_tiles = tiles;
    left -= last - first;
    if (left > 0) {
      if (++at.ct >= cts) {
        at.ct = 0;
        if (++at.h >= a.v.Hkv) {
          at.h = 0;
          cts = 0;
          while (cts == 0 && ++at.b < a.B) {                   // left > 0: there is one
            seq = ka_seq(a, at.b);
            cts = ka_col_tiles(a, seq);
          }
          if (cts == 0) left = 0;                              // (unless the batch changed under the call)
          row = a.v.tables + (int64_t)seq.slot * a.v.max_pages;
        }
      }
    }
    if (left > 0) {
      end = ka_end(a, seq, at.ct);
      tiles = (end + TILE - 1) / TILE;
      first = 0;
      last = tiles < left ? tiles : left;
      blocks = (end + KV4_ROWS - 1) / KV4_ROWS;
      mine = copies.dead ? 0 : my_steps();
      ahead = fill(row, at.h, 0, mine, blocks);
    }

    // ---- the four warps' states become one ---------------------------------------------------------------------------------------
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float z = l[j];
        z += __shfl_xor_sync(0xffffffffu, z, 4);
        z += __shfl_xor_sync(0xffffffffu, z, 8);
        z += __shfl_xor_sync(0xffffffffu, z, 16);
        const int n = 2 * t + j;
        if (g == 0 && n < NC) {
          s_ref[warp * W + n] = ref[j];
          s_sum[warp * W + n] = z;
        }
      }
    ka_sync(team);
    float corr[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = (NC < 8 ? (2 * t + j) % NC : 2 * t + j);
        float r = s_ref[c];
#pragma unroll
        for (int w = 1; w < KA_WARPS; ++w) r = fmaxf(r, s_ref[w * W + c]);
        corr[j] = ka_exp2(ref[j] - r) * vlim * (SL == 2 && j ? KA_LO : 1.0f);
      }
    // (row, head) hc = column hc * SL of the tile: its reference and sum, and where its output goes
    float* part = a.part + ((int64_t)run * 2 + (begins ? 1 : 0)) * (HC * (D + 4));
    const bool whole = begins && ends;
    if (tid < HC) {
      const int hc = tid, c = hc * SL, rh = was.ct * HC + hc;
      float r = s_ref[c], z = 0.0f;
#pragma unroll
      for (int w = 1; w < KA_WARPS; ++w) r = fmaxf(r, s_ref[w * W + c]);
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) z += s_sum[w * W + c] * ka_exp2(s_ref[w * W + c] - r);
      if (!whole) { part[HC * D + 2 * hc] = r; part[HC * D + 2 * hc + 1] = z; }
      s_div[hc] = whole ? z : 1.0f;
      const int i = a.by_rep(rh);
      s_to[hc] = !whole ? (int64_t)hc * D : i < was_seq.n ? ((int64_t)(was_seq.row0 + i) * a.Hq + was.h * a.rep + rh - i * a.rep) * D : -1;
    }
    if (begins && !ends && tid == 0) {                 // the merge starts from here: it begins at the end of this run
      const int begin = lo + per - was_last;
      cut[1] = was_seq.row0; cut[2] = was_seq.n; cut[3] = was.h; cut[4] = was.ct;
      cut[0] = (begin + was_tiles - 1) / per;                  // the last run that holds a piece of it
    }
    // QG groups at a time: every warp leaves its sums, all threads add the four in order and store
#pragma unroll
    for (int G0 = 0; G0 < NG; G0 += C::QG) {
      constexpr int QD = C::QG * 32, QSTR = C::OSTR;
#pragma unroll
        for (int G = G0; G < G0 + C::QG; ++G) {
          const int n0 = 2 * t;                                // this lane's columns n0, n0 + 1; group G % GP owns NC of them
          if (NC < 8 && (NC == 1 ? (n0 >> 1) != (G % GP) >> 1 : n0 / NC != G % GP)) continue;
          const int c0 = (NC < 8 ? n0 % NC : n0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* x = acc[2 * G + h];
            float* o = s_o + (warp * HC + c0 / SL) * QSTR + (G - G0) * 32 + h * 16 + g;
            if (SL == 2) {
              o[0] = x[0] * corr[0] + x[1] * corr[1];
              o[8] = (x[2] * corr[0] + x[3] * corr[1]) * 0.0625f;
            } else if (NC == 1) {
              o[0] = (G & 1 ? x[1] : x[0]) * corr[0];
              o[8] = (G & 1 ? x[3] : x[2]) * (corr[0] * 0.0625f);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                o[j * QSTR] = x[j] * corr[j];
                o[j * QSTR + 8] = x[j + 2] * (corr[j] * 0.0625f);
              }
            }
          }
        }
      ka_sync(team);
#pragma unroll
      for (int e0 = 0; e0 < HC * QD; e0 += KA_THREADS * 2) {   // two dimensions per thread
        const int e = e0 + 2 * tid;
        if (e >= HC * QD) break;
        const int hc = e / QD, d = e % QD;
        float2 o = *reinterpret_cast<const float2*>(s_o + hc * QSTR + d);
#pragma unroll
        for (int w = 1; w < KA_WARPS; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(s_o + (w * HC + hc) * QSTR + d);
          o.x += v.x; o.y += v.y;
        }
        const int64_t to = s_to[hc];
        if (whole) {
          const float z = s_div[hc];
          if (to >= 0) ka_store2(static_cast<T*>(a.out) + to + G0 * 32 + d, o.x / z, o.y / z);
        } else {
          *reinterpret_cast<float2*>(part + to + G0 * 32 + d) = o;
        }
      }
      ka_sync(team);
    }
    if (left <= 0) break;
  }
  if (copies.dead) {                                           // do not leave with copies in flight
    const uint64_t t0 = ka_now();
    copies.drain([&](int st, uint32_t parity) { return ka_bar_wait(bar0 + st * 8, parity, lane, t0); });
  }
}

// Segments that were cut, merged in run order.  grid: (runs, (row, head) pairs of a tile); a run that begins a segment and
// does not finish it has left its place in `cut`, the others have nothing to do.  Few pieces: a warp per pair; many: a CTA per
// pair, whose threads share the pieces (two contexts of 131072 positions with 32 / 4 heads of 128 have 56; one warp would read them one by one).
constexpr int KA_MERGE_THREADS = 256, KA_MAX_RUNS = 1024, KA_FEW = 4;
template <typename T>
__global__ void __launch_bounds__(KA_MERGE_THREADS) kv4_attention_merge_kernel(const __grid_constant__ KaArgs a) {
  __shared__ float s_f[KA_MAX_RUNS], s_red[KA_MERGE_THREADS / 32][2];
  __shared__ float4 s_o[KA_MERGE_THREADS];
  pdl_launch_dependents();
  pdl_wait();
  const int run = blockIdx.x, HC = (1 << a.width_log2) / a.sl, D = a.v.D, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int* cut = a.cut + (int64_t)run * 8;
  const int last = cut[0];
  if (last < 0) return;
  const int row0 = cut[1], n = cut[2], h = cut[3];
  const int64_t slot = (int64_t)HC * (D + 4);
  const int pieces = last - run + 1;
  // piece 0 is this run's second state, piece j > 0 the first state of run run + j
  const float* p0 = a.part + ((int64_t)run * 2 + 1) * slot;
  const float* p1 = a.part + (int64_t)run * 2 * slot;
  if (pieces <= KA_FEW) {
    for (int hc = blockIdx.y * (KA_MERGE_THREADS / 32) + warp; hc < HC; hc += gridDim.y * (KA_MERGE_THREADS / 32)) {
      const int rh = cut[4] * HC + hc;
      if (rh >= n * a.rep) break;
      // lane j looks after piece j
      const float* st = (lane ? p1 + 2 * lane * slot : p0) + HC * D + 2 * hc;
      float r = lane < pieces ? st[0] : -INFINITY, z = lane < pieces ? st[1] : 0.0f;
      float top = r;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float f = lane < pieces ? ka_exp2(r - top) : 0.0f;
      z *= f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) z += __shfl_xor_sync(0xffffffffu, z, off);
      const float inv = 1.0f / z;
      const int i = rh / a.rep;
      T* out = static_cast<T*>(a.out) + ((int64_t)(row0 + i) * a.Hq + h * a.rep + rh - i * a.rep) * D;
      for (int d0 = 0; d0 < D; d0 += 128) {
        const int d = d0 + lane * 4;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int j = 0; j < pieces; ++j) {
          const float w = __shfl_sync(0xffffffffu, f, j);
          if (d >= D) continue;
          const float4 v = *reinterpret_cast<const float4*>((j ? p1 + 2 * j * slot : p0) + hc * D + d);
          o.x += v.x * w; o.y += v.y * w; o.z += v.z * w; o.w += v.w * w;
        }
        if (d < D) {
          ka_store2(out + d, o.x * inv, o.y * inv);
          ka_store2(out + d + 2, o.z * inv, o.w * inv);
        }
      }
    }
    return;
  }
  for (int hc = blockIdx.y; hc < HC; hc += gridDim.y) {
    const int rh = cut[4] * HC + hc;
    if (rh >= n * a.rep) break;
    if (hc != (int)blockIdx.y) __syncthreads();                 // the buffers are free again
    float r = -INFINITY;
    for (int j = threadIdx.x; j < pieces; j += KA_MERGE_THREADS) r = fmaxf(r, (j ? p1 + 2 * j * slot : p0)[HC * D + 2 * hc]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, off));
    if (lane == 0) s_red[warp][0] = r;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KA_MERGE_THREADS / 32; ++w) r = fmaxf(r, s_red[w][0]);
    float z = 0.0f;
    for (int j = threadIdx.x; j < pieces; j += KA_MERGE_THREADS) {
      const float* st = (j ? p1 + 2 * j * slot : p0) + HC * D + 2 * hc;
      const float f = ka_exp2(st[0] - r);
      s_f[j] = f;
      z += st[1] * f;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) z += __shfl_xor_sync(0xffffffffu, z, off);
    if (lane == 0) s_red[warp][1] = z;
    __syncthreads();
    z = 0.0f;
#pragma unroll
    for (int w = 0; w < KA_MERGE_THREADS / 32; ++w) z += s_red[w][1];
    // a thread sums four dimensions over every slices-th piece
    const int quads = D / 4, slices = KA_MERGE_THREADS / quads, q = threadIdx.x % quads, sl = threadIdx.x / quads;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (sl < slices) {
#pragma unroll 4
      for (int j = sl; j < pieces; j += slices) {
        const float4 v = *reinterpret_cast<const float4*>((j ? p1 + 2 * j * slot : p0) + hc * D + q * 4);
        const float f = s_f[j];
        o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
      }
    }
    s_o[threadIdx.x] = o;
    __syncthreads();
    if (sl == 0) {
      const int used = slices < pieces ? slices : pieces;
      for (int k = 1; k < used; ++k) {
        const float4 v = s_o[k * quads + q];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      }
      T* out = static_cast<T*>(a.out) + ((int64_t)(row0 + rh / a.rep) * a.Hq + h * a.rep + rh % a.rep) * D + q * 4;
      const float inv[4] = {o.x / z, o.y / z, o.z / z, o.w / z};
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = from_float<T>(inv[j]);
    }
  }
}

constexpr int KA_MAX_TEAMS = 4, KA_MAX_WIDTH = 8;      // of any variant

template <typename T, int NG, int NC>
int ka_launch(KaArgs a, cudaStream_t s) {
  using C = KaCfg<T, NG, NC>;
  static_assert(C::TEAMS <= KA_MAX_TEAMS && C::W <= KA_MAX_WIDTH, "the caller's scratch is sized for these");
  static bool sized = false;
  if (!sized) {
    BQ_CUDA(cudaFuncSetAttribute(kv4_attention_kernel<T, NG, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TEAMS * C::SMEM));
    sized = true;
  }
  a.by_rep = ka_div(a.rep);
  a.by_row = ka_div(a.rep * C::SL);
  a.sl = C::SL;
  for (a.width_log2 = 0; 1 << a.width_log2 < C::W;) ++a.width_log2;
  for (a.tile_log2 = 0; 1 << a.tile_log2 < C::TILE;) ++a.tile_log2;
  // a list cannot be longer than the tables allow
  const double most = (double)a.B * a.v.Hkv * (double)((((int64_t)a.v.max_pages << a.v.page_log2) + C::TILE - 1) / C::TILE) *
                      (double)((a.n_rows * a.rep * C::SL + C::W - 1) / C::W);
  int64_t grid = sm_count();
  if (grid > KA_MAX_RUNS / C::TEAMS) grid = KA_MAX_RUNS / C::TEAMS;
  if ((double)grid > most) grid = (int64_t)most;
  BQ_CUDA(launch_chain(kv4_attention_kernel<T, NG, NC>, dim3((unsigned)grid), dim3(C::TEAMS * KA_THREADS), C::TEAMS * C::SMEM, s, 1, a));
  BQ_CUDA(launch_chain(kv4_attention_merge_kernel<T>, dim3((unsigned)(grid * C::TEAMS - 1), (unsigned)C::HC), dim3(KA_MERGE_THREADS), 0, s, 1, a));
  count_launch(2);
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

// kv4_chunk.cu: many rows per sequence; cols = (row, head) pairs of an average sequence and KV head
bool kv4_chunk_supported(int D, int dtype, int64_t B, int Hkv, int64_t cols);
int64_t kv4_chunk_part_bytes(int D);
int kv4_chunk(const KaArgs& a, cudaStream_t s);

// one per head_dim (kv4_attn_*.cu): picks the variant for `cols` columns per sequence
template <typename T, int NG> int ka_pick(const KaArgs& a, int64_t cols, cudaStream_t s);

}  // namespace bq
