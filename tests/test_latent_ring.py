"""Places and barriers of the latent attention's ring (``csrc/mla_cache_ring.cuh``),
followed on the CPU in the loading warp's order."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from conftest import REPO

CSRC = os.path.join(REPO, "-kimi-linear-_b200", "csrc")

# Nothing lands or is freed sooner than the loader has waited for: what it does not
# know, is not so.  (An mbarrier of count one: arming it again before its phase is over
# is undefined; a parity wait is ambiguous unless the phase before is over.)
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "mla_cache_ring.cuh"
using namespace kda::cache;

int main(int argc, char** argv) {
  const int chunks = std::atoi(argv[1]), half = std::atoi(argv[2]), ring = std::atoi(argv[3]);
  const Ring places(ring, chunks, half);
  std::vector<int> holder(ring, -1), armed(2 * kStages, -1);   // half tiles, by place and by barrier
  int freed = -1, slot = 0;
  auto fail = [&](const char* what, int h) {
    std::printf("%s: half tile %d, tile_chunks %d half %d ring %d\n", what, h, chunks, half, ring);
    std::exit(1);
  };
  for (int k = 0; k < 64; ++k) {
    for (int h = 2 * k; h <= 2 * k + 1; ++h) {          // the loading warp arms both halves first,
      int& last = armed[half_barrier(h)];
      if (last > freed) fail("arms while the phase before may be open", h);
      if (last >= 0 && half_parity(last) == half_parity(h)) fail("parity", h);
      last = h;
    }
    for (int c = 0; c < chunks; ++c) {                  // then waits for each chunk's place
      const int need = places.held_by(k, c);
      if (need > freed) {
        if (need / 2 >= k || (need % 2 && half == chunks)) fail("waits for what is not loaded", need);
        if (need - 2 * kStages > freed) fail("waits while the phase before may be open", need);
        freed = need;
      }
      if (holder[slot] > freed) fail("loads over a chunk that may still be read", 2 * k + (c >= half));
      holder[slot] = 2 * k + (c >= half);
      slot = (slot + 1) % ring;
    }
  }
  std::puts("ok");
}
"""


# The same loader giving up at each of its waits: every half tile that it then drains is
# armed and completes with the bytes that it asked for, and none in flight is left out.
GIVE_UP = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include "mla_cache_ring.cuh"
using namespace kda::cache;

int main(int argc, char** argv) {
  const int chunks = std::atoi(argv[1]), half = std::atoi(argv[2]), ring = std::atoi(argv[3]);
  const Ring places(ring, chunks, half);
  auto fail = [&](const char* what, int h) {
    std::printf("%s: half tile %d, tile_chunks %d half %d ring %d\n", what, h, chunks, half, ring);
    std::exit(1);
  };
  int gave_up = 0;
  for (int waits = 0;; ++waits) {                       // gives up at this wait
    std::map<int, int> expected, asked;                 // chunks by half tile
    int freed = -1, left = waits, k = 0;
    bool ok = true;
    for (; k < 24 && ok; ++k) {
      expected[2 * k] = half;
      expected[2 * k + 1] = chunks - half;
      for (int c = 0; c < chunks; ++c) {
        const int need = places.held_by(k, c);
        if (need > freed) {
          if (left-- == 0) {
            for (int h = 0; h < 2; ++h) expected[2 * k + h] -= places.missing(c, h);
            ok = false;
            break;
          }
          freed = need;
        }
        ++asked[2 * k + (c >= half)];
      }
    }
    if (ok) break;                                      // fewer waits than that
    ++gave_up;
    const int first = first_in_flight(k), last = 2 * k - 1;
    if (last - first >= 2 * kStages) fail("drains a barrier twice", first);
    for (const auto& e : expected) {
      if (e.second != asked[e.first]) fail("expects other bytes than were asked for", e.first);
      if (e.first > last) fail("leaves out what is armed", e.first);
      if (e.first < first && e.first > freed && e.second) fail("leaves out what may be in flight", e.first);
    }
    for (int h = first; h <= last; ++h)
      if (!expected.count(h)) fail("drains what was never armed", h);
  }
  if (gave_up < 16) fail("too few waits", gave_up);
  std::puts("ok");
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.fail("no C++ compiler (nvcc needs one too)")
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text(PROGRAM)
    (d / "give_up.cpp").write_text(GIVE_UP)
    for name in ("ring", "give_up"):
        subprocess.run([cxx, "-std=c++17", "-O1", "-I", CSRC, "-o", str(d / name), str(d / f"{name}.cpp")],
                       check=True)
    return d


def follow(exe, codes, rope):
    """Every ring from two tiles (the least that the products need) to kRingTiles."""
    chunks, half = codes + rope, rope + (codes + 1) // 2
    for ring in range(2 * chunks, 4 * chunks + 1):
        res = subprocess.run([str(exe), str(chunks), str(half), str(ring)], capture_output=True, text=True)
        assert res.returncode == 0 and res.stdout == "ok\n", res.stdout


@pytest.mark.parametrize("rope", [0, 1])
@pytest.mark.parametrize("codes", [1, 2, 3, 4])
def test_barriers_are_armed_only_when_their_phase_is_over(codes, rope, program):
    follow(program / "ring", codes, rope)


@pytest.mark.parametrize("rope", [0, 1])
@pytest.mark.parametrize("codes", [1, 2, 3, 4])
def test_a_loader_that_gives_up_waits_for_its_copies_only(codes, rope, program):
    follow(program / "give_up", codes, rope)
