"""The decode-step operators' host side and what their kernels share with it, without a GPU."""

import subprocess


ROW_PARTS = r"""
#include <cstdio>
#include <cstdint>
#include "ops.h"
using ssb::MlaRowParts;
using ssb::kMlaRanges;
int main() {
  // every record that a plan can write is valid, and its slots are the CTAs' own
  for (int f = 0; f < kMlaRanges; ++f)
    for (int l = f; l < kMlaRanges; ++l)
      for (int s = 0; s < 2; ++s) {
        const MlaRowParts p = {f, l, 2 * f + s, 0};
        if (!p.valid() || p.slot(0) != 2 * f + s) return std::printf("refused %d %d %d\n", f, l, s), 1;
        for (int i = 1; i <= l - f; ++i)
          if (p.slot(i) != 2 * (f + i) || p.slot(i) >= 2 * kMlaRanges)
            return std::printf("slot %d %d %d\n", f, l, i), 1;
      }
  // whatever else memory holds: refused, or within the parts
  const int32_t edge[] = {0, 1, -1, 2, kMlaRanges - 1, kMlaRanges, 2 * kMlaRanges - 1, 2 * kMlaRanges, -2, 294,
                          296, 0x7f800000, 0x7fffffff, static_cast<int32_t>(0x80000000u),
                          static_cast<int32_t>(0xffff8000u), 0x3f800000};
  uint64_t x = 88172645463325252ull;
  auto rnd = [&] { x ^= x << 13, x ^= x >> 7, x ^= x << 17; return static_cast<int32_t>(x >> 20); };
  auto check = [&](const MlaRowParts& p) {
    if (!p.valid()) return true;
    if (p.last < p.first || p.last - p.first >= kMlaRanges) return false;
    for (int i = 0; i <= p.last - p.first; ++i)
      if (p.slot(i) < 0 || p.slot(i) >= 2 * kMlaRanges) return false;
    return true;
  };
  for (int a : edge)
    for (int b : edge)
      for (int c : edge)
        if (!check({a, b, c, 0})) return std::printf("accepted %d %d %d\n", a, b, c), 1;
  for (int n = 0; n < 4000000; ++n) {
    const bool small = n & 1;
    const int32_t a = rnd(), b = rnd(), c = rnd();
    if (!check(small ? MlaRowParts{a % 400, b % 400, c % 400, 0} : MlaRowParts{a, b, c, 0}))
      return std::printf("accepted %d %d %d\n", a, b, c), 1;
  }
  if (MlaRowParts{0, 0x7fffffff, 0, 0}.valid() || MlaRowParts{-1, -1, -2, 0}.valid() || MlaRowParts{3, 2, 6, 0}.valid())
    return std::printf("accepted a range outside\n"), 1;
  std::puts("ok");
}
"""


def test_a_rows_record_stays_within_the_parts_whatever_memory_holds(tmp_path):
    """The join reads parts by a row's record; a CTA that gave up leaves there what the workspace held before."""
    from ssengine_b200 import _build

    src, exe = tmp_path / "row_parts.cu", tmp_path / "row_parts"
    src.write_text(ROW_PARTS)
    subprocess.run([_build.nvcc(), *_build.ARCH, "-std=c++17", "-O1", f"-I{_build.CSRC}", "-o", str(exe), str(src)],
                   check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout
