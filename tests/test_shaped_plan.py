"""How calls with shaped scores or a shared prefix are cut into workgroups (ellm_amd/csrc/shaped_plan.hpp, host code): the
division by multiplication, shares of a walk, plans and the room they need, the ways of a single-token step; what the
generated code of the tile kernel has to keep; refusals that need no device."""
import os
import re
import shutil
import subprocess

import pytest

from ellm_amd import _lib
from test_build_invariants import _ahead, _listing, _scalars

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ellm_amd", "csrc")

PROBE = r"""
#include "shaped_plan.hpp"
#include <cstdio>
#include <cstdlib>
using namespace ellm;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)

static void divisors() {
  uint64_t seen = 0, r = 88172645463325252ull;
  for (uint32_t i = 0; i < 4000; ++i) {
    r ^= r << 13; r ^= r >> 7; r ^= r << 17;
    const uint32_t d = i < 1500 ? i + 1 : i < 1560 ? (1u << (i - 1500) / 2) + i % 2 : (uint32_t)(r >> 33) >> (r & 31);
    if (d == 0) continue;
    const Divisor x = divisor(d);
    for (uint32_t j = 0; j < 400; ++j) {
      r ^= r << 13; r ^= r >> 7; r ^= r << 17;
      uint64_t n = j < 100 ? j : j < 200 ? (uint64_t)d * (j - 100) - (j & 1) : j < 300 ? 0x7fffffffu - (j - 200) : (uint32_t)(r >> 33);
      if (n > 0x7fffffffu) continue;
      const uint32_t q = x.quotient((uint32_t)n);
      CHECK(q == n / d && x.rest((uint32_t)n, q) == n % d);
      ++seen;
    }
  }
  CHECK(seen > 1000000);
}

static void shares() {
  const uint32_t steps[] = {0, 1, 2, 3, 63, 64, 1000, 4099, (1u << 25) - 1, (1u << 26) - 1};
  for (uint32_t n : steps)
    for (uint32_t split = 1; split <= 4096; split += split < 70 ? 1 : 37) {
      const Divisor by = divisor(split);
      CHECK(shaped_share(n, 0, by) == 0 && shaped_share(n, split, by) == n);
      for (uint32_t i = 0; i < split; ++i) {
        const uint32_t here = shaped_share(n, i + 1, by) - shaped_share(n, i, by);
        CHECK(here == n / split || here == n / split + 1);
      }
    }
}

static void plans() {
  const uint32_t heads[][2] = {{1, 1}, {8, 1}, {32, 1}, {80, 1}, {4, 4}, {32, 4}, {64, 8}, {32, 32}};
  const uint32_t intervals[] = {1, 2, 7, 16, 64, 200, 1000, 8192}, keys[] = {1, 63, 64, 65, 1000, 8192, 131072};
  const uint32_t prefixes[] = {0, 1, 64, 300, 5000, 131072}, cus[] = {64, 256, 304};
  for (uint32_t n_cu : cus)
    for (auto& h : heads)
      for (uint32_t interval : intervals)
        for (uint32_t batch = 1; batch <= 3000; batch = batch * 2 + 1) {
          const uint32_t group = h[0] / h[1];
          const uint64_t rows = (uint64_t)interval * batch * h[0];
          if (rows > 0x7fffffffu) continue;
          const size_t room = shaped_part_rows(interval, batch, h[0], n_cu);
          CHECK(room <= (size_t)4 * n_cu * kShapedRows);
          for (uint32_t own : keys)
            for (uint32_t prefix : prefixes) {
              const ShapedPlan p = shaped_plan(interval, batch, h[1], group, own, prefix, n_cu, room);
              CHECK(p.rows_plane == interval * group && p.tiles_plane * kShapedRows >= p.rows_plane && p.n_split >= 1);
              CHECK(p.n_part == p.n_split + p.prefix_split);
              CHECK(p.n_part == 1 || rows * p.n_part <= room);
              CHECK(p.n_split <= 4096 && p.prefix_split <= 4096);
              if (p.prefix_tiles) {
                CHECK(prefix && p.prefix_split >= 1 && p.prefix_rows == interval * group * batch);
                CHECK((uint64_t)p.prefix_tiles * kShapedRows >= p.prefix_rows);
              } else {
                CHECK(p.prefix_split == 0 && p.prefix_rows == 0);
              }
              // no more workgroups than places, except where walks that are not split are more already
              const uint64_t walks = (uint64_t)p.tiles_plane * batch * h[1], ahead = (uint64_t)p.prefix_tiles * h[1];
              if (walks + ahead <= 2 * n_cu) CHECK(walks * p.n_split + ahead * p.prefix_split <= 2 * n_cu);
              if (interval == 1 && prefix && (uint64_t)batch * h[0] <= room) {
                const ShapedPlan q = shaped_prefix_plan(batch, h[1], group, prefix, n_cu, room);
                CHECK(q.prefix_split >= 1 && q.n_part == q.prefix_split && rows * q.n_part <= room);
                CHECK(q.prefix_rows == batch * group && (uint64_t)q.prefix_tiles * kShapedRows >= q.prefix_rows);
              }
            }
        }
}

static void ways() {
  // sequences, K/V heads, group, own keys, prefix
  CHECK(shaped_prefix_step(2, 4, 8, 40, 2000, 256) == PrefixStep::kWalk);
  CHECK(shaped_prefix_step(1, 1, 1, 1, 1, 256) == PrefixStep::kWalk);
  CHECK(shaped_prefix_step(24, 4, 8, 40, 8000, 256) == PrefixStep::kMixed);
  CHECK(shaped_prefix_step(24, 4, 8, 24000, 8000, 256) == PrefixStep::kApart);
  CHECK(shaped_prefix_step(128, 8, 8, 40, 2000, 256) == PrefixStep::kApart);
  CHECK(shaped_prefix_step(8, 1, 80, 40, 40000, 256) == PrefixStep::kApart);     // a group of more than half a tile
  CHECK(shaped_prefix_step(70000, 1, 1, 0x7fffffffu, 0x7fffffffu, 256) == PrefixStep::kApart);
  // a prefix that is not the longer part of a call that splits nothing: neither part is cut past the places there are
  const ShapedPlan p = shaped_plan(1, 8, 32, 1, 40, 2000, 256, 1 << 17);
  CHECK(p.n_split == 1 && p.prefix_split == 8);
  // 241 tokens alone: two walks a tile would find a place, but joining them costs more than it saves
  CHECK(shaped_plan(241, 1, 4, 8, 241, 0, 256, 1 << 17).n_part == 1);
}

static uint32_t chunk_way(uint32_t hq, uint32_t hkv, uint32_t batch, uint32_t prefix, uint32_t start, uint32_t interval,
                          uint32_t* splits) {
  const uint32_t group = hq / hkv, own = start + interval, keys = prefix + own;
  const ShapedPlan p = shaped_plan(interval, batch, hkv, group, own, prefix, 256, shaped_part_rows(interval, batch, hq, 256));
  *splits = p.n_part;
  return shaped_short_rows({interval * group, batch * hkv, hkv, 256, (double)keys, keys - 0.5 * interval, (double)own, (double)prefix}, p);
}

static void chunks() {   // the calls that the GPU tests make for the sake of a kernel
  uint32_t splits;
  CHECK(chunk_way(16, 2, 2, 0, 300, 70, &splits) == 1);
  CHECK(chunk_way(8, 2, 3, 0, 30, 150, &splits) == 1);
  CHECK(chunk_way(64, 1, 6, 0, 200, 45, &splits) == 2);
  CHECK(chunk_way(64, 1, 9, 0, 200, 33, &splits) == 2);
  CHECK(chunk_way(64, 1, 12, 0, 0, 70, &splits) == 0 && splits == 1);
  CHECK(chunk_way(8, 1, 2, 0, 2600, 9, &splits) == 0 && splits > 1);
  CHECK(chunk_way(32, 4, 1, 0, 0, 8192, &splits) == 0 && splits == 1);
  CHECK(chunk_way(32, 4, 1, 0, 0, 2, &splits) == 1);
  CHECK(chunk_way(8, 2, 2, 150, 10, 40, &splits) == 1);
  CHECK(chunk_way(64, 1, 13, 150, 0, 20, &splits) == 2);
  CHECK(chunk_way(32, 4, 2, 5000, 0, 9, &splits) == 0 && splits > 1);
}

int main() { divisors(); shares(); plans(); ways(); chunks(); printf("done\n"); return 0; }
"""


def test_plans_shares_and_divisions(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout


def test_short_walk_kernel_keeps_no_scratch(tmp_path):
    text = _listing("shaped_short.hip", tmp_path)
    assert set(re.findall(r"\.private_segment_fixed_size:\s*(\d+)", text)) == {"0"}
    assert set(re.findall(r"\.[sv]gpr_spill_count:\s*(\d+)", text)) == {"0"}


def test_tile_kernel_keeps_no_scratch_and_leaves_m0_to_the_inline_asm(tmp_path):
    """Its tiles come into LDS by loads in inline asm, which sets M0 without being able to say so; their descriptors must
    not have been written by a vector instruction within the five wait states that the compiler keeps for its own loads."""
    text = _listing("shaped_chunk.hip", tmp_path)
    assert set(re.findall(r"\.private_segment_fixed_size:\s*(\d+)", text)) == {"0"}
    assert set(re.findall(r"\.[sv]gpr_spill_count:\s*(\d+)", text)) == {"0"}
    lines = [re.split(r";|//", l)[0].rstrip() for l in text.splitlines()]
    uses = [l for l in lines if re.search(r"\bm0\b", l)]
    assert uses and all(re.fullmatch(r"\s*s_mov_b32 m0, s\d+\s*", l) for l in uses)
    assert not any("movrel" in l or "s_set_gpr_idx" in l for l in lines)
    jumps = {}
    for n, l in enumerate(lines):
        if (m := re.match(r"\s+s_c?branch\w*\s+(\.LBB\d+_\d+)", l)):
            jumps.setdefault(m.group(1), []).append(n)
    loads = [n for n, l in enumerate(lines) if re.search(r"buffer_load_dwordx4 .* lds$", l)]
    assert loads
    for at in loads:
        reads = _scalars(lines[at])
        for n in _ahead(lines, jumps, at, 5):
            if lines[n].strip().startswith("v_"):
                m = re.match(r"\s*(v_\w+)\s+([^,]+)(?:,\s*([^,]+))?", lines[n])
                written = _scalars(m.group(2)) | (_scalars(m.group(3) or "") if "_co_" in m.group(1) else set())
                assert not written & reads, (lines[n], lines[at])


def test_null_handles_are_refused():
    lib = _lib.load_library()
    assert lib.ellm_attn_set_scores(None, 0.0, None, 0, None, None, 0) == 1
    assert lib.ellm_attn_set_shared_prefix(None, None, None, 0, 0, 0) == 1
    assert b"null handle" in lib.ellm_last_error_string()
