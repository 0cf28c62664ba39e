"""How single-token calls over planes in 8 bits are cut (ellm_amd/csrc/decode_plan.hpp and decode_shares.hpp, host code):
invariants over a sweep of shapes, and the plans of some shapes."""
import os
import re
import shutil
import subprocess

import pytest

from test_build_invariants import _listing

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ellm_amd", "csrc")

PROBE = r"""
#include "decode_plan.hpp"
#include "decode_shares.hpp"
#include <cstdio>
#include <initializer_list>
using namespace ellm;
int main() {
  const uint32_t lens[] = {1, 31, 128, 129, 255, 512, 513, 1000, 2048, 4097, 8192, 40000, 131072, 1u << 20, 0x7fffffffu};
  const uint32_t heads[][2] = {{1, 1}, {8, 1}, {64, 1}, {4, 4}, {32, 4}, {64, 8}, {16, 16}};
  for (uint32_t n_cu : {64u, 256u, 304u})
    for (auto& h : heads)
      for (uint32_t cap = 1; cap <= 130; cap += (cap < 18 ? 1 : 14)) {
        const DecodeWorkspace w = decode_workspace(cap, h[0], h[1], n_cu);
        for (uint32_t batch = 1; batch <= cap; batch += (batch < 18 ? 1 : 14))
          for (uint32_t len : lens) {
            const DecodePlan p = decode_plan(len, batch, h[1], n_cu, kDecodeStepKeysE4m3);
            printf("%u %u %u %u %u %u %u %d\n", n_cu, h[1], cap, batch, len, p.split_len, p.n_split,
                   (int)decode_plan_fits(w, batch, h[0], h[1], h[0] / h[1], p.n_split));
          }
      }
  // workgroups out of 512 and 256: equal planes; a longest plane of 22 pieces on 512 and 11 on 256, of 12 and 6, of 44 and 22; more planes
  // than units; long shares, without and with new rows to write, and of a plane of 17 pieces on 256; the largest call, whose longest plane
  // is all of it: 254 pieces are the most that two folds take, 248 the multiple of 8
  const uint32_t U = 512 * 9;
  auto W = [](uint32_t U, uint32_t longest, uint32_t umin, uint32_t planes, bool rows) {
    return balanced_workgroups_e4m3(512, 256, U, longest + 3, umin + 3, planes, longest, rows);
  };
  printf("shares %u %u %u %u %u %u %u %u %u\n", W(64 * 36, 36, 36, 64, false), W(U, 198, 6, 40, true), W(U, 108, 6, 60, false),
         W(U, 396, 6, 20, false), W(512 * 40, 198, 6, 257, false), W(512 * 25, 50, 6, 256, false), W(512 * 25, 50, 6, 256, true),
         W(512 * 25, 50 * 17, 6, 256, false), W(0x7fffffffu, 0x7ffffffbu, 1, 2, false));
  // what a plane's start is charged with: nothing for equal or long planes
  printf("charge %u %u %u %u\n", balanced_charge(10, 10, 100, 10, kBalancedChargeE4m3), balanced_charge(10, 9, 100, 10, kBalancedChargeE4m3),
         balanced_charge(900, 9, 5130, 10, kBalancedChargeE4m3), balanced_charge(10, 9, 100, 10));
  return 0;
}
"""


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("e4m3_plan")
    src, exe = d / "probe.cpp", d / "probe"
    src.write_text(PROBE)
    subprocess.run([gxx, "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True, timeout=300)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=300).stdout.splitlines()


def test_plans_are_well_formed_and_fit_the_workspace(lines):
    rows = [[int(x) for x in line.split()] for line in lines if line[0].isdigit()]
    assert len(rows) > 10000
    for n_cu, hkv, cap, batch, length, split_len, n_split, fits in rows:
        case = (n_cu, hkv, cap, batch, length, split_len, n_split)
        assert split_len % 128 == 0, case                       # whole steps of the four waves
        assert n_split == -(-length // split_len) and 1 <= n_split <= 256 and fits == 1, case
        assert (n_split - 1) * split_len < length, case         # no split without keys
        assert n_split == 1 or length > 512, case               # planes of up to four steps are not cut
        if split_len == 128:
            assert n_split <= 16, case                          # one fold
    by = {(r[0], r[1], r[3], r[4]): (r[5], r[6]) for r in rows if r[2] == r[3]}
    assert by[(256, 4, 1, 1000)] == (128, 8)
    assert by[(256, 4, 16, 8192)] == (2048, 4)                  # 64 planes x 4 = 256 workgroups
    assert by[(256, 4, 1, 131072)] == (2048, 64)
    assert by[(256, 8, 16, 2048)] == (1024, 2)


def test_shares_of_planes_of_different_lengths(lines):
    found = {line.split()[0]: [int(x) for x in line.split()[1:]] for line in lines if not line[0].isdigit()}
    assert found["shares"] == [256, 256, 512, 512, 512, 256, 512, 512, 248]
    assert found["charge"] == [0, 3, 0, 2]


def test_write_and_read_kernels_stay_in_registers(tmp_path):
    text = _listing("kv_e4m3.hip", tmp_path)
    assert set(re.findall(r"\.private_segment_fixed_size:\s*(\d+)", text)) == {"0"}
    assert set(re.findall(r"\.[sv]gpr_spill_count:\s*(\d+)", text)) == {"0"}
