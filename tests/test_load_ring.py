"""The ring of loads that the attention kernel over a cache in 8 or 4 bits walks (``csrc/load_ring.h``), compiled for the host:
what happens when a load does not arrive, which no test makes happen on a GPU."""

import shutil
import subprocess

import pytest

from simple_inference_autoresearch_b200.kernels import build

WALK = r"""
#include "load_ring.h"
#include <cstdio>
#include <cstdlib>
#include <vector>

// The barriers as the kernel uses them: arming one starts the phase that its load completes.
template <int STAGES>
struct Barriers {
  int lost;                                   // the load that never arrives, or -1
  std::vector<int> armed = std::vector<int>(STAGES, 0), done = std::vector<int>(STAGES, 0);
  std::vector<int> load = std::vector<int>(STAGES, -1);
  std::vector<char> waited;                   // by load
  void fail(const char* why, int at) { std::printf("%s %d\n", why, at); std::exit(1); }
  void arm(int s, int i) {
    if (s != i % STAGES) fail("a load in another stage", i);
    if (armed[s] != done[s]) fail("a barrier armed while its phase is under way, load", i);
    ++armed[s];
    load[s] = i;
    waited.push_back(0);
  }
  bool wait(int s, int parity) {
    if (armed[s] == 0) fail("a wait for a stage that was never loaded", s);
    if (((armed[s] - 1) & 1) != parity) fail("a wait for another phase, stage", s);
    waited[load[s]] = 1;
    if (load[s] != lost) done[s] = armed[s];  // it has arrived by now
    return done[s] == armed[s];
  }
};

template <int STAGES>
void walk(int loads, int lost) {
  Barriers<STAGES> b{lost};
  siar::LoadRing<STAGES> ring;
  auto wait = [&](int s, int parity) { return b.wait(s, parity); };
  int asked = 0, used = 0, after = 0;
  auto issue = [&]() {
    if (asked < loads && ring.room()) {
      if (ring.expired) ++after;
      b.arm(ring.next(), asked++);
    }
  };
  for (int s = 0; s < STAGES; ++s) issue();
  for (int i = 0; i < loads; ++i) {
    if (!ring.take(wait)) continue;           // (as a later unit of the same block asks again)
    if (b.load[ring.stage()] != i) b.fail("the wrong load taken at", i);
    ++used;
    ring.release();
    issue();
  }
  ring.drain(wait);
  const bool meets = lost >= 0 && lost < loads;
  if (used != (meets ? lost : loads)) b.fail("loads used", used);
  if (after) b.fail("loads after a wait ran out", after);
  if (ring.expired != meets) b.fail("what is reported", ring.expired);
  if (asked > used + STAGES) b.fail("loads beyond the ring", asked);
  for (int i = 0; i < asked; ++i)
    if (!b.waited[i]) b.fail("left without waiting for load", i);
}

int main() {
  for (int loads = 0; loads <= 13; ++loads)
    for (int lost = -1; lost <= loads; ++lost) {
      walk<2>(loads, lost);
      walk<4>(loads, lost);
    }
  return 0;
}
"""


def test_a_load_that_does_not_arrive_ends_the_ring(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "walk.cpp").write_text(WALK)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I", str(build.CSRC), "-o", str(tmp_path / "walk"), str(tmp_path / "walk.cpp")],
                   check=True)
    out = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_the_kernel_walks_this_ring():
    """No wait, issue or hand-back beside the ring's own: loads only where it has room, steps only for what it took, and a
    drain on the way out."""
    text = (build.CSRC / "attention_quant.cu").read_text()
    assert text.count("mbar_wait(") == 1 and "ring.take(arrived)" in text
    assert "while (l_left > 0 && ring.room())" in text
    assert text.index("ring.drain(arrived)") > text.index("store_all();")
