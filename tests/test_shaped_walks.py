"""What a call with a window sees of a shared prefix, and how long its walks are (ellm_amd/csrc/shaped_plan.hpp, host code)."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ellm_amd", "csrc")

HEAD = r"""
#include "shaped_plan.hpp"
#include <cstdio>
#include <cstdlib>
using namespace ellm;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)
"""


def run_probe(tmp_path, body):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(HEAD + body)
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout


def test_prefix_rows_that_a_window_hides_take_no_part_in_a_plan(tmp_path):
    run_probe(tmp_path, r"""
static void by_counting() {   // against the definition: key j of the text is seen at position p where p - j < window
  for (uint32_t prefix = 0; prefix < 40; ++prefix)
    for (uint32_t window = 0; window < 50; ++window)
      for (uint32_t first = 0; first < 50; ++first) {
        uint32_t seen = 0;
        for (uint32_t j = 0; j < prefix; ++j) seen += !window || prefix + first - j < window;
        CHECK(shaped_prefix_seen(prefix, window, first) == seen);
        for (uint32_t interval = 1; interval < 40; interval += 6)
          for (uint32_t group = 1; group <= 64; group *= 4) {
            const ShapedWalks w = shaped_walks(first, interval, group, seen, window);
            CHECK(w.own <= first + interval && w.both <= seen + first + interval && w.own <= w.both);
            const uint32_t tokens = 128 / group;   // of any tile's rows: the keys from the first's first to the last's own
            for (uint32_t t = 0; t < interval; ++t) {
              const uint32_t last = t + tokens < interval ? t + tokens : interval - 1;
              const uint32_t a = prefix + first + t, b = prefix + first + last;
              const uint32_t lo = window && a + 1 > window ? a + 1 - window : 0;
              CHECK(b + 1 - lo <= w.both);
              CHECK(b + 1 - (lo > prefix ? lo : prefix) <= w.own);
            }
          }
      }
  CHECK(shaped_prefix_seen(100000, 1, 0) == 0 && shaped_prefix_seen(100000, 0, 7) == 100000);
  CHECK(shaped_prefix_seen(100000, 0xffffffffu, 0x7fff0000u) == 100000);
}

static ShapedPlan plan(uint32_t interval, uint32_t batch, uint32_t position, uint32_t window, uint32_t prefix) {
  const uint32_t seen = shaped_prefix_seen(prefix, window, position);
  const ShapedWalks w = shaped_walks(position, interval, 8, seen, window);
  return shaped_plan(interval, batch, 4, 8, w.own, seen, 256, shaped_part_rows(interval, batch, 32, 256), window ? w.both : 0);
}
static bool same(const ShapedPlan& a, const ShapedPlan& b) {
  return a.n_split == b.n_split && a.prefix_tiles == b.prefix_tiles && a.prefix_split == b.prefix_split && a.n_part == b.n_part;
}

int main() {
  by_counting();
  // a window that ends inside the own rows: the plan without a prefix
  CHECK(same(plan(1, 2, 1999, 1000, 100000), plan(1, 2, 1999, 1000, 0)) && plan(1, 2, 1999, 1000, 100000).n_split == 8);
  CHECK(same(plan(64, 2, 1023, 1024, 32768), plan(64, 2, 1023, 1024, 0)));
  CHECK(same(plan(64, 1, 4000, 1024, 32768), plan(64, 1, 4000, 1024, 0)));
  // one that leaves a part of the prefix: the plan behind that part alone
  CHECK(same(plan(8, 2, 100, 1024, 100000), plan(8, 2, 100, 1024, 923)) && plan(8, 2, 100, 1024, 100000).prefix_tiles);
  // walks over both parts are no longer than the window lets them be
  const ShapedPlan p = plan(256, 1, 0, 4096, 100000);
  CHECK(!p.prefix_tiles && same(p, shaped_plan(256, 1, 4, 8, 4096 + 17, 0, 256, shaped_part_rows(256, 1, 32, 256))));
  printf("done\n");
  return 0;
}
""")


def test_a_short_prefix_ahead_of_long_uneven_own_rows_is_not_walked(tmp_path):
    run_probe(tmp_path, r"""
int main() {
  // sequences, K/V heads, group, own keys, prefix
  CHECK(shaped_prefix_step(24, 4, 8, 30000, 100, 256, true) == PrefixStep::kApart);
  CHECK(shaped_prefix_step(20, 8, 8, 30000, 1000, 256, true) == PrefixStep::kApart);
  CHECK(shaped_prefix_step(64, 4, 8, 3000, 600, 256, true) == PrefixStep::kApart);
  CHECK(shaped_prefix_step(24, 4, 8, 30000, 100, 256, false) == PrefixStep::kWalk);   // even
  CHECK(shaped_prefix_step(8, 4, 8, 8000, 1000, 256, true) == PrefixStep::kWalk);     // too little to share out
  CHECK(shaped_prefix_step(4, 4, 8, 500, 2000, 256, true) == PrefixStep::kWalk);
  CHECK(shaped_prefix_step(64, 8, 8, 2000, 300, 256, true) == PrefixStep::kWalk);     // planes that even it out
  CHECK(shaped_prefix_step(24, 4, 8, 1000, 999, 256, true) == PrefixStep::kWalk);     // (all a window of 1000 leaves)
  printf("done\n");
  return 0;
}
""")


def test_chunks_of_many_planes_are_dealt_along_their_tiles(tmp_path):
    """The calls that the GPU tests make for the sake of that order."""
    run_probe(tmp_path, r"""
static uint32_t along(uint32_t hq, uint32_t hkv, uint32_t batch, uint32_t start, uint32_t interval, uint32_t prefix) {
  const uint32_t group = hq / hkv, own = start + interval, keys = prefix + own;
  const ShapedPlan p = shaped_plan(interval, batch, hkv, group, own, prefix, 256, shaped_part_rows(interval, batch, hq, 256));
  const uint32_t wr = shaped_short_rows({interval * group, batch * hkv, hkv, 256, (double)keys, keys - 0.5 * interval, (double)own,
                                         (double)prefix}, p);
  return shaped_short_along(batch * hkv, keys) ? wr : 0;
}
int main() {
  CHECK(along(32, 4, 9, 300, 16, 0) == 1 && along(8, 8, 9, 2100, 5, 0) == 1 && along(36, 9, 5, 300, 5, 50) == 1);
  CHECK(along(8, 1, 37, 30, 33, 0) == 2 && along(8, 1, 33, 30, 45, 50) == 2);
  printf("done\n");
  return 0;
}
""")
