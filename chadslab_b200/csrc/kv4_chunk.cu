// Attention of many rows over the paged 4-bit KV cache (chunks of prompts behind cached context), bf16 rows.
//
// The decode kernel (kv4_attn.cuh) unpacks every code once per eight columns, which for a chunk is most of its work: 53
// TFLOP/s at 512 rows.  Here a CTA of eight warps holds 128 (row, query head) pairs of one KV head, unpacks a tile of 64
// positions once into shared memory as fp16 codes and all warps use it: 16 pairs are the M dimension of a warp's
// mma.sync.m16n8k16, positions (scores) or dimensions (outputs) the N dimension.
//   * The fragment words of the cache are B fragments as they lie: for keys (n = position) words r0, r1 and r2, r3 are those
//     of positions 0-7 and 8-15, for values (n = dimension) r0, r2 and r1, r3 those of dimensions 0-7 and 8-15.
//   * Codes stay whole numbers (exact in fp16).  A key group's scale multiplies its 32-dimension sum in fp32, a value's scale
//     multiplies the weight, as in the decode kernel; so do the power-of-two scaling of q, the lagging softmax reference,
//     the raising of small value scales and the list of tiles that is cut into equal runs (here one per SM) and merged.
// Bound: shared memory and its latency.  Every 512-byte B fragment is read for two matrix instructions (a warp has 16 rows; 32
// would need 256 accumulator registers at head_dim 256), which is 128 bytes per cycle and SM at the matrix pipe's full rate:
// 117 TFLOP/s at 512 rows, 8 heads on one KV head of 256; the shared-memory pipe is busy in 68 % of the cycles, the matrix pipe
// in 38 %, with two warps per scheduler to cover the rest.  Unpacking the next tile while this one is multiplied (two buffers, half the tile
// at head_dim 256) changed nothing at head_dim 128 (272 -> 270 us) and lost at 256 (132 -> 159 us).
#include "kv4_attn.cuh"

namespace bq {

constexpr int KK_WARPS = 8;
constexpr int KK_THREADS = KK_WARPS * 32;
constexpr int KK_ROWS = KK_WARPS * 16;                // (row, head) pairs of a tile
constexpr int KK_BLOCKS = 4;                          // 16-position blocks of a tile
constexpr int KK_TILE = KK_BLOCKS * KV4_ROWS;
constexpr int KK_LOST = 0x7FFFFFFF;                   // in vmax: the tile's copies did not arrive

struct KkShared {
  KaScan scan;
  KaPlace at;
  int total, per, ok;
  int vmax[2];                                        // largest value scale of a stage's tile (bits of a float), or KK_LOST
  uint64_t bar[2];
};
template <int NG> struct KkCfg {
  static constexpr int D = NG * GROUP;
  static constexpr int BLK = kv4_block_bytes(D);
  static constexpr int FRAG = KK_BLOCKS * NG * 2 * 512;         // fp16 codes of K or of V of a tile
  static constexpr int Q = KK_WARPS * 2 * NG * 512;
  static constexpr int SMEM = 2 * KK_BLOCKS * BLK + 2 * FRAG + Q + NG * KK_TILE * 4 + (int)sizeof(KkShared);
};
// (1024 + 16 n) / 16 - 72 = n - 8, exact
__device__ __forceinline__ uint32_t kk_code_high(uint32_t w) {
  return ka_bits(__hfma2(ka_half2(lop3_and_or(w, 0x00F000F0u, 0x64006400u)), ka_half2(0x2C002C00u), ka_half2(0xD480D480u)));
}

template <int NG>
__global__ void __launch_bounds__(KK_THREADS, 1) kv4_chunk_kernel(const __grid_constant__ KaArgs a) {
  using C = KkCfg<NG>;
  constexpr int D = C::D;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* raw = smem;                                           // [2][KK_BLOCKS][BLK]
  uint8_t* kf = raw + 2 * KK_BLOCKS * C::BLK;                    // [block][group][tile][lane][4 words]
  uint8_t* vf = kf + C::FRAG;
  uint8_t* qf = vf + C::FRAG;                                    // [warp][k step][lane][4 words]
  float* ks = reinterpret_cast<float*>(qf + C::Q);               // [group][position] scales of the keys
  KkShared* sh = reinterpret_cast<KkShared*>(ks + NG * KK_TILE);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t bar0 = ka_smem(sh->bar);
  if (tid == 0) {
    ka_bar_init(bar0);
    ka_bar_init(bar0 + 8);
    sh->vmax[0] = sh->vmax[1] = 0;
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait();
  const int run = blockIdx.x, runs = gridDim.x;
  int* cut = a.cut + (int64_t)run * 8;
  if (tid == 0) cut[0] = -1;
  if (warp < KA_WARPS) {                                         // the search is written for a team of four warps
    KaPlace p = {};
    int total = 0, per = 0;
    const bool ok = ka_locate<__nv_bfloat16>(a, runs, run, 0, &sh->scan, &p, &total, &per);
    if (tid == 0) { sh->at = p; sh->total = total; sh->per = per; sh->ok = ok; }
  }
  __syncthreads();
  if (!sh->ok) return;
  KaPlace at = sh->at;
  const int per = sh->per, lo = run * per;
  int left = sh->total - lo < per ? sh->total - lo : per;
  Kv4Seq seq = ka_seq(a, at.b);
  int end = ka_end(a, seq, at.ct), tiles = (end + KK_TILE - 1) / KK_TILE, cts = ka_col_tiles(a, seq);
  const int pb = a.v.page_blocks_log2();
  int first = at.tile, last = tiles - first < left ? tiles : first + left;
  const int32_t* row = a.v.tables + (int64_t)seq.slot * a.v.max_pages;
  Kv4Ring<2> copies;                                             // the same in every warp; warp 0 requests
  // a tile's blocks, one lane each
  auto request = [&](int tile, int st) {
    const int blocks = (end + KV4_ROWS - 1) / KV4_ROWS, b0 = tile * KK_BLOCKS, n = blocks - b0 < KK_BLOCKS ? blocks - b0 : KK_BLOCKS;
    if (lane == 0) ka_bar_expect(bar0 + st * 8, n * C::BLK);
    __syncwarp();
    if (lane < n) {
      const int blk = b0 + lane;
      uint32_t id = (uint32_t)row[blk >> pb];
      if (id >= (uint64_t)a.v.n_pages) {                         // no such page: recorded, the result is undefined
        *(volatile int*)a.status = (int)BQ_ERR_ARG;
        id = 0;
      }
      const uint32_t in = ((uint32_t)at.h << pb) + (blk & ((1 << pb) - 1));
      ka_bulk_load(ka_smem(raw + (st * KK_BLOCKS + lane) * C::BLK), a.v.pages + (int64_t)id * a.v.page_bytes + (a.v.layer_off + (int64_t)in * C::BLK),
                   C::BLK, bar0 + st * 8);
    }
  };
  if (warp == 0) request(first, copies.put);
  copies.requested(1);

  while (true) {
    // ---- this warp's 16 pairs: rows g and g + 8 of its A fragments ---------------------------------------------------------------
    float kappa[2];
    int vis[2];
    {
      const __nv_bfloat16* qp[2];
      float up[2];
      bool ok[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int rh = at.ct * KK_ROWS + warp * 16 + g + 8 * j, i = a.by_rep(rh);
        ok[j] = i < seq.n;
        qp[j] = static_cast<const __nv_bfloat16*>(a.q) + (ok[j] ? (int64_t)(seq.row0 + i) * a.ldq + (int64_t)(at.h * a.rep + rh - i * a.rep) * D : 0) + 2 * t;
        float big = 0.0f;
#pragma unroll 8
        for (int k = 0; k < 4 * NG; ++k) {
          const float2 x = ok[j] ? ka_q2(qp[j] + k * 8) : make_float2(0.0f, 0.0f);
          big = fmaxf(big, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        int k2 = 13 - ((int)(__float_as_uint(big) >> 23) - 127);
        k2 = k2 > 100 ? 100 : k2 < -114 ? -114 : k2;
        up[j] = __uint_as_float((uint32_t)(127 + k2) << 23);
        k2 = k2 < -100 ? -100 : k2;                              // as in the decode kernel
        kappa[j] = __uint_as_float((uint32_t)(127 - k2) << 23) * 1.4426950408889634f * rsqrtf((float)D);
        vis[j] = ok[j] ? seq.pos + i : 0x7FFFFFFF;
      }
#pragma unroll 4
      for (int k = 0; k < 2 * NG; ++k) {
        uint32_t f[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {                            // (row g, low k), (g + 8, low), (g, high), (g + 8, high)
          const int j = x & 1;
          const float2 v = ok[j] ? ka_q2(qp[j] + k * 16 + (x >> 1) * 8) : make_float2(0.0f, 0.0f);
          f[x] = ka_pack(v.x * up[j], v.y * up[j]);
        }
        *reinterpret_cast<uint4*>(qf + ((warp * 2 * NG + k) * 32 + lane) * 16) = make_uint4(f[0], f[1], f[2], f[3]);
      }
      __syncwarp();
    }
    const int all_see = seq.pos + a.by_rep(at.ct * KK_ROWS);

    float o[4 * NG][4], ref[2], l[2], A = 11.0f, vlim = KA_VLIM0;      // o carries the 1 / vlim of the scales
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      ref[j] = vis[j] == 0x7FFFFFFF ? 3.0e38f : -3.0e38f;        // a pair without a row has no weight anywhere
      l[j] = 0.0f;
    }
    for (int tile = first; tile < last; ++tile) {
      if (tile + 1 < last) {
        if (warp == 0) request(tile + 1, copies.put);
        copies.requested(1);
      }
      // a copy that does not arrive: recorded, and all warps leave behind the next barrier
      if (!copies.arrived([&](int st, uint32_t parity) { return ka_bar_wait(bar0 + st * 8, parity, lane); })) {
        *(volatile int*)a.status = (int)BQ_ERR_TIMEOUT;
        if (lane == 0) atomicMax(&sh->vmax[copies.take], KK_LOST);
      }
      const int take = copies.take;
      uint8_t* stage = raw + take * KK_BLOCKS * C::BLK;
      const int p0 = tile * KK_TILE;
      // ---- unpack: warp w takes (block, group) units -----------------------------------------------------------------------------
      float vtop = 0.0f;
#pragma unroll
      for (int u = warp; u < KK_BLOCKS * NG; u += KK_WARPS) {
        const int blk = u / NG, G = u % NG;
        const uint8_t* b = stage + blk * C::BLK;
        const uint2 kw = *reinterpret_cast<const uint2*>(b + G * 256 + lane * 8);
        const uint2 vw = *reinterpret_cast<const uint2*>(b + kv4_v_off(D) + G * 256 + lane * 8);
        uint4* kd = reinterpret_cast<uint4*>(kf + u * 1024) + lane;
        uint4* vd = reinterpret_cast<uint4*>(vf + u * 1024) + lane;
        kd[0] = make_uint4(ka_code(kw.x), kk_code_high(kw.x), ka_code(kw.x >> 8), kk_code_high(kw.x >> 8));
        kd[32] = make_uint4(ka_code(kw.y), kk_code_high(kw.y), ka_code(kw.y >> 8), kk_code_high(kw.y >> 8));
        vd[0] = make_uint4(ka_code(vw.x), ka_code(vw.x >> 8), kk_code_high(vw.x), kk_code_high(vw.x >> 8));
        vd[32] = make_uint4(ka_code(vw.y), ka_code(vw.y >> 8), kk_code_high(vw.y), kk_code_high(vw.y >> 8));
        if (lane < 16) {
          const __half* sk = reinterpret_cast<const __half*>(b + kv4_kscale_off(D));
          ks[G * KK_TILE + blk * 16 + lane] = __half2float(sk[lane * NG + G]);
          const int r = (lane >> 2) * 2 + (lane & 1) + 8 * ((lane >> 1) & 1);            // the position of value scale `lane`
          const float vs = __half2float(reinterpret_cast<const __half*>(b + kv4_vscale_off(D))[G * 16 + lane]);
          if (p0 + blk * 16 + r < end) vtop = fmaxf(vtop, vs);
        }
      }
      if (vlim < 1.0f) vtop = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)));
      if (vlim < 1.0f ? lane == 0 : vtop > 1.0f) atomicMax(&sh->vmax[take], __float_as_int(vtop));
      __syncthreads();
      const int vbits = sh->vmax[take];
      if (vbits == KK_LOST) {
        copies.dead = true;
        break;
      }
      // values above one: weights stay so far below 2^15 that their product with the largest scale does too
      const float vbig = __int_as_float(vbits);
      const float want = vbig > 1.0f ? 11.0f - (float)((__float_as_int(vbig) >> 23) - 126) : 11.0f;
      if (vlim < 1.0f) {                                         // no scale above 1/16 before this tile: see kv4_attn.cuh
        const float was = vlim;
        vlim = ka_vlim(was, vbig);
        const float lower = was * ka_inverse(vlim);
        if (tile > first) {
#pragma unroll
          for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] *= lower;
        }
        if (vlim < 1.0f) {
          constexpr int WORDS = NG * 8;
          const uint32_t up = ka_pack(ka_inverse(vlim), ka_inverse(vlim));
          for (int e = tid; e < KK_BLOCKS * WORDS; e += KK_THREADS) {
            uint32_t* p = reinterpret_cast<uint32_t*>(stage + e / WORDS * C::BLK + kv4_vscale_off(D) + e % WORDS * 4);
            *p = ka_mul2(ka_live_scales(*p, e % WORDS, end - p0 - e / WORDS * KV4_ROWS), up);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before the copy that will fill the stage again
          __syncthreads();
        }
      }
      // ---- scores: rows g, g + 8; positions 8 n + 2t, + 1 -------------------------------------------------------------------------
      float s[2 * KK_BLOCKS][4];
#pragma unroll
      for (int n = 0; n < 2 * KK_BLOCKS; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
#pragma unroll 2
      for (int G = 0; G < NG; ++G) {
        float c[2 * KK_BLOCKS][4];
#pragma unroll
        for (int n = 0; n < 2 * KK_BLOCKS; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) c[n][j] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 q = *reinterpret_cast<const uint4*>(qf + ((warp * 2 * NG + 2 * G + h) * 32 + lane) * 16);
#pragma unroll
          for (int blk = 0; blk < KK_BLOCKS; ++blk) {
            const uint4 k = *reinterpret_cast<const uint4*>(kf + ((blk * NG + G) * 2 + h) * 512 + lane * 16);
            ka_mma(c[2 * blk], q.x, q.y, q.z, q.w, k.x, k.y);
            ka_mma(c[2 * blk + 1], q.x, q.y, q.z, q.w, k.z, k.w);
          }
        }
#pragma unroll
        for (int n = 0; n < 2 * KK_BLOCKS; ++n) {
          const float2 f = *reinterpret_cast<const float2*>(ks + G * KK_TILE + n * 8 + 2 * t);
          s[n][0] = fmaf(f.x, c[n][0], s[n][0]);
          s[n][1] = fmaf(f.y, c[n][1], s[n][1]);
          s[n][2] = fmaf(f.x, c[n][2], s[n][2]);
          s[n][3] = fmaf(f.y, c[n][3], s[n][3]);
        }
      }
      const bool masked = p0 + KK_TILE - 1 > all_see;            // positions past the end, or past a pair's own
      if (masked) {
#pragma unroll
        for (int n = 0; n < 2 * KK_BLOCKS; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p0 + n * 8 + 2 * t + (j & 1) > vis[j >> 1]) s[n][j] = -INFINITY;
      }
      float high[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2 * KK_BLOCKS; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) high[j >> 1] = fmaxf(high[j >> 1], s[n][j]);
      const float low = fminf(A, want);
      if (__any_sync(0xffffffffu, fmaf(high[0], kappa[0], -ref[0]) > A + 4.0f || fmaf(high[1], kappa[1], -ref[1]) > A + 4.0f) || low < A) {
        // the reference moves up to the maximum so far (and further away from it if the values ask for that)
        const float drop = A - low;
        A = low;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float m = __fmul_rd(high[j], kappa[j]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const float r = fmaxf(ref[j] + drop, m - A), corr = ka_exp2(ref[j] - r);
          ref[j] = r;
          l[j] *= corr;
#pragma unroll
          for (int i = 0; i < 4 * NG; ++i) { o[i][2 * j] *= corr; o[i][2 * j + 1] *= corr; }
        }
      }
      uint32_t p[KK_BLOCKS][4];                                  // A fragments of the weights
#pragma unroll
      for (int n = 0; n < 2 * KK_BLOCKS; ++n) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = ka_exp2(ka_min(fmaf(s[n][j], kappa[j >> 1], -ref[j >> 1]), A + 4.0f));
          l[j >> 1] += w[j];
        }
        p[n >> 1][(n & 1) * 2] = ka_pack(w[0], w[1]);
        p[n >> 1][(n & 1) * 2 + 1] = ka_pack(w[2], w[3]);
      }
      // ---- outputs ---------------------------------------------------------------------------------------------------------------------
#pragma unroll
      for (int blk = 0; blk < KK_BLOCKS; ++blk) {
        uint32_t live[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
        if (masked) {                                            // a scale behind the last position can be anything: no weight, no product
#pragma unroll
          for (int j = 0; j < 4; ++j) live[j] = __hne2_mask(ka_half2(p[blk][j]), __floats2half2_rn(0.0f, 0.0f));
        }
#pragma unroll
        for (int G = 0; G < NG; ++G) {
          const uint2 vs = *reinterpret_cast<const uint2*>(stage + blk * C::BLK + kv4_vscale_off(D) + G * 32 + t * 8);
          const uint32_t w0 = ka_mul2(p[blk][0], vs.x) & live[0], w1 = ka_mul2(p[blk][1], vs.x) & live[1];
          const uint32_t w2 = ka_mul2(p[blk][2], vs.y) & live[2], w3 = ka_mul2(p[blk][3], vs.y) & live[3];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 v = *reinterpret_cast<const uint4*>(vf + ((blk * NG + G) * 2 + h) * 512 + lane * 16);
            ka_mma(o[G * 4 + h * 2], w0, w1, w2, w3, v.x, v.y);
            ka_mma(o[G * 4 + h * 2 + 1], w0, w1, w2, w3, v.z, v.w);
          }
        }
      }
      __syncthreads();                                           // the tile has been read by every warp
      if (tid == 0) sh->vmax[take] = 0;
      copies.consumed();
    }
    if (copies.dead) break;

    // ---- where this run goes next: its first tile travels while this piece is stored -----------------------------------------------
    const KaPlace was = at;
    const Kv4Seq was_seq = seq;
    const int was_last = last, was_tiles = tiles;
    const bool begins = first == 0, ends = last == tiles, whole = begins && ends;
    left -= last - first;
    if (left > 0) {
      if (++at.ct >= cts) {
        at.ct = 0;
        if (++at.h >= a.v.Hkv) {
          at.h = 0;
          cts = 0;
          while (cts == 0 && ++at.b < a.B) {                     // left > 0: there is one
            seq = ka_seq(a, at.b);
            cts = ka_col_tiles(a, seq);
          }
          if (cts == 0) left = 0;                                // (unless the batch changed under the call)
          row = a.v.tables + (int64_t)seq.slot * a.v.max_pages;
        }
      }
    }
    if (left > 0) {
      end = ka_end(a, seq, at.ct);
      tiles = (end + KK_TILE - 1) / KK_TILE;
      first = 0;
      last = tiles < left ? tiles : left;
      if (warp == 0) request(0, copies.put);
      copies.requested(1);
    }
    // ---- this warp's rows --------------------------------------------------------------------------------------------------------------
    float* part = a.part + ((int64_t)run * 2 + (begins ? 1 : 0)) * (KK_ROWS * (D + 4));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float z = l[j];
      z += __shfl_xor_sync(0xffffffffu, z, 1);
      z += __shfl_xor_sync(0xffffffffu, z, 2);
      const int hc = warp * 16 + g + 8 * j, rh = was.ct * KK_ROWS + hc, i = a.by_rep(rh);
      if (i >= was_seq.n) continue;
      if (whole) {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + ((int64_t)(was_seq.row0 + i) * a.Hq + was.h * a.rep + rh - i * a.rep) * D + 2 * t;
        const float inv = vlim / z;
#pragma unroll
        for (int x = 0; x < 4 * NG; ++x) ka_store2(out + x * 8, o[x][2 * j] * inv, o[x][2 * j + 1] * inv);
      } else {
#pragma unroll
        for (int x = 0; x < 4 * NG; ++x) ka_store2(part + hc * D + x * 8 + 2 * t, o[x][2 * j] * vlim, o[x][2 * j + 1] * vlim);
        if (t == 0) { part[KK_ROWS * D + 2 * hc] = ref[j]; part[KK_ROWS * D + 2 * hc + 1] = z; }
      }
    }
    if (begins && !ends && tid == 0) {                           // the merge starts from here: it begins at the end of this run
      const int begin = lo + per - was_last;
      cut[1] = was_seq.row0; cut[2] = was_seq.n; cut[3] = was.h; cut[4] = was.ct;
      cut[0] = (begin + was_tiles - 1) / per;
    }
    if (left <= 0) break;
  }
  if (warp == 0 && copies.dead) {                                // do not leave with copies in flight
    const uint64_t t0 = ka_now();
    copies.drain([&](int st, uint32_t parity) { return ka_bar_wait(bar0 + st * 8, parity, lane, t0); });
  }
}

template <int NG>
static int chunk_launch(KaArgs a, cudaStream_t s) {
  using C = KkCfg<NG>;
  static bool sized = false;
  if (!sized) {
    BQ_CUDA(cudaFuncSetAttribute(kv4_chunk_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    sized = true;
  }
  a.by_rep = ka_div(a.rep);
  a.by_row = ka_div(a.rep);
  a.sl = 1;
  a.width_log2 = 7;
  a.tile_log2 = 6;
  const unsigned grid = (unsigned)sm_count();
  BQ_CUDA(launch_chain(kv4_chunk_kernel<NG>, dim3(grid), dim3(KK_THREADS), C::SMEM, s, 1, a));
  BQ_CUDA(launch_chain(kv4_attention_merge_kernel<__nv_bfloat16>, dim3(grid - 1, KK_ROWS / 8), dim3(KA_MERGE_THREADS), 0, s, 1, a));
  count_launch(2);
  BQ_CUDA(cudaGetLastError());
  return BQ_OK;
}

// Which calls come here: head dimensions of whole, even fragments, at least 96 (row, head) pairs per sequence and KV head, and
// 48 segments of 128 of them or more, so that few are cut (a cut leaves 128 pairs' states to be merged).  Both kernels, us, at
// 8 sequences x 2048 positions, 16 heads of 256 (decode kernel / this one): 64 pairs 143 / 171, 96: 204 / 177, 256: 488 / 330;
// 32 / 4 heads of 128 (32 segments up to 128 pairs, 64 at 256): 96: 44 / 48, 128: 53 / 54, 256: 80 / 58; 8 heads on one KV
// head of 256, 256 pairs (16 segments): 51 / 67.
bool kv4_chunk_supported(int D, int dtype, int64_t B, int Hkv, int64_t cols) {
  return dtype == BQ_DT_BF16 && (D == 64 || D == 128 || D == 256) && cols >= 96 && B * Hkv * ((cols + KK_ROWS - 1) / KK_ROWS) >= 48;
}
int64_t kv4_chunk_part_bytes(int D) { return (int64_t)sm_count() * 2 * KK_ROWS * (D + 4) * (int64_t)sizeof(float); }
int kv4_chunk(const KaArgs& a, cudaStream_t s) {
  return a.v.D == 64 ? chunk_launch<2>(a, s) : a.v.D == 128 ? chunk_launch<4>(a, s) : chunk_launch<8>(a, s);
}

}  // namespace bq
