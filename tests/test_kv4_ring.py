"""The ring that attention over the 4-bit cache copies through (kv4_ring.h), run on the host: order, parities, and what happens
when a copy never arrives."""
import os
import subprocess

import pytest

from conftest import ROOT

DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "kv4_ring.h"
using bq::Kv4Ring;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)

constexpr int S = STAGES;
// Barriers with one arrival per phase.  A copy arrives when somebody waits for it, unless it is the lost one.
struct Machine {
  int done[S] = {}, open[S] = {}, token[S] = {}, expired = 0, next = 0, lost;
  bool request(int st) {
    CHECK(!open[st]);                                   // never into a stage that is still being filled
    open[st] = 1;
    token[st] = next++;
    return true;
  }
  bool wait(int st, uint32_t parity) {
    if ((uint32_t)(done[st] & 1) != parity) return true;
    if (open[st] && token[st] != lost) { open[st] = 0; ++done[st]; return true; }
    ++expired;
    return false;
  }
};

int main() {
  std::mt19937 rng(1);
  for (int trial = 0; trial < 20000; ++trial) {
    Machine m;
    Kv4Ring<S> ring;
    std::vector<int> pieces(1 + rng() % 4);
    int all = 0;
    for (int& n : pieces) all += n = rng() % 9;
    m.lost = rng() % 2 ? (int)(rng() % (all + 1)) : -1;
    const bool loses = m.lost >= 0 && m.lost < all;
    auto wait = [&](int st, uint32_t parity) { return m.wait(st, parity); };
    int read = 0;
    for (int n : pieces) {
      const int mine = ring.dead ? 0 : n;
      int ahead = ring.room(mine);
      for (int j = 0; j < ahead; ++j) m.request(ring.stage(j));
      ring.requested(ahead);
      for (int i = 0; i < mine; ++i) {
        if (!ring.arrived(wait)) break;
        CHECK(m.token[ring.take] == read && !m.open[ring.take]);
        ++read;
        ring.consumed();
        if (ahead < mine) { m.request(ring.put); ring.requested(1); ++ahead; }
      }
    }
    CHECK(ring.dead == loses);
    CHECK(read == (loses ? m.lost : all));
    CHECK(m.expired == (loses ? 1 : 0));                // nobody waits again for what did not arrive
    if (!ring.dead) { CHECK(ring.flying == 0); continue; }
    ring.drain(wait);
    CHECK(m.expired == 2 && ring.flying > 0);             // once more, then the kernel leaves
    m.lost = -1;                                          // had it arrived late, all of them would be seen
    ring.drain(wait);
    CHECK(ring.flying == 0);
    for (int st = 0; st < S; ++st) CHECK(!m.open[st]);
  }
  std::puts("ok");
}
"""


@pytest.mark.parametrize("stages", [2, 3, 4])
def test_ring_order_and_lost_copies(tmp_path, stages):
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-DSTAGES={stages}", "-I", os.path.join(ROOT, "chadslab_b200", "csrc"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout
