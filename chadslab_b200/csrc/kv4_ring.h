// Bookkeeping of a ring of S stages that asynchronous copies fill in order and their consumer reads in the same order.
// Plain C++ (a test runs it on the host): `wait(stage, parity)` waits for a copy with a limit and says whether it arrived.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define KV4_RING_FN __host__ __device__ __forceinline__
#else
#define KV4_RING_FN inline
#endif

namespace bq {

template <int S> struct Kv4Ring {
  int put = 0, take = 0;                               // stage to fill next, stage to read next ...
  uint32_t phase = 0;                                  // ... and the parity of its barrier
  int flying = 0;                                      // copies requested and not consumed
  bool dead = false;                                   // a copy did not arrive in time: nothing is requested or waited for any more

  // how many of `steps` copies may be requested into an empty ring; the j-th of them goes to stage(j)
  KV4_RING_FN int room(int steps) const { return dead ? 0 : steps < S ? steps : S; }
  KV4_RING_FN int stage(int j) const { return put + j >= S ? put + j - S : put + j; }
  KV4_RING_FN void requested(int n) {
    put = stage(n);
    flying += n;
  }
  // waits for the copy in stage `take`; false: it did not arrive, the stage must not be read or filled, nor this called again
  template <typename W> KV4_RING_FN bool arrived(W wait) {
    if (wait(take, phase)) return true;
    dead = true;
    return false;
  }
  KV4_RING_FN void consumed() {
    --flying;
    if (++take == S) { take = 0; phase ^= 1u; }
  }
  // before the memory is given up: the copies still under way, in order, until one does not arrive either
  template <typename W> KV4_RING_FN void drain(W wait) {
    while (flying > 0 && wait(take, phase)) consumed();
  }
};

}  // namespace bq
