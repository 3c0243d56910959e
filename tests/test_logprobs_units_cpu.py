"""CPU test of the units in which k_token_logprobs reads its rows (csrc/units.cuh, the kernel's own arithmetic): nothing
outside a row is read, and each of its elements is taken once."""
import subprocess

from conftest import PKG_DIR

SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#define __host__
#define __device__
#define __forceinline__ inline
#include "units.cuh"

// All that a part's copies and loads take of one row: `stage` units at a time, whole ones by address, others by element.
static void check(int off, int n, int parts, int stage) {
  alignas(16) static float room[1 << 16];
  const float *row = room + 4 + off;
  const UnitRow r = unit_row(row, n);
  std::vector<int> taken(n, 0);
  int units = 0;
  for (int p = 0; p < parts; p++) {
    int first, end;
    part_of(r, p, parts, &first, &end);
    if (first != units) { printf("parts do not follow each other\n"); exit(1); }
    units = end;
    int whole0, whole1;
    whole_of(r, first, end, &whole0, &whole1);
    if (whole0 > first + 1 || whole1 < end - 1) { printf("more than two edges\n"); exit(1); }
    for (int u = first; u < end; u += stage) {
      const int upto = u + stage < end ? u + stage : end, from = u > whole0 ? u : whole0, to = upto < whole1 ? upto : whole1;
      for (int x = u; x < upto; x++) {
        const bool copied = x >= from && x < to;
        if (copied != whole(r, x) || copied != (element_of(r, x, 0) >= 0 && element_of(r, x, 3) >= 0)) { printf("off %d n %d parts %d: unit %d\n", off, n, parts, x); exit(1); }
        if (copied) {
          const float *at = unit_at(r, x);
          if (((uintptr_t)at & 15) || at < row || at + 4 > row + n) { printf("off %d n %d: unit %d outside\n", off, n, x); exit(1); }
          for (int i = 0; i < 4; i++) {
            if (at + i != row + element_of(r, x, i)) { printf("off %d n %d: unit %d misplaced\n", off, n, x); exit(1); }
            taken[at + i - row]++;
          }
        } else {
          for (int i = 0; i < 4; i++)
            if (element_of(r, x, i) >= 0)
              taken[element_of(r, x, i)]++;
        }
      }
    }
  }
  if (units != r.count) { printf("units left over\n"); exit(1); }
  for (int i = 0; i < n; i++)
    if (taken[i] != 1) { printf("off %d n %d parts %d: element %d taken %d times\n", off, n, parts, i, taken[i]); exit(1); }
}

int main() {
  for (int off = 0; off < 4; off++)
    for (int parts = 1; parts <= 8; parts *= 2)
      for (int stage : {1, 2, 3, 8, 1024})
        for (int n = 1; n < 700; n += n < 80 ? 1 : 37)
          check(off, n, parts, stage);
  for (int off = 0; off < 4; off++)
    for (int n : {4096, 4097, 4098, 4099, 50001})
      check(off, n, 2, 1024);
  // The largest vocabulary: nothing wraps.
  const UnitRow r = unit_row(reinterpret_cast<const float *>((uintptr_t)28), 0x7fffffff);
  if (whole(r, 0) || !whole(r, 1) || !whole(r, r.count - 2) || whole(r, r.count - 1)) { printf("large\n"); return 1; }
  if (r.off != 3 || r.count != 0x20000001 || element_of(r, r.count - 1, 1) != 0x7ffffffe || element_of(r, r.count - 1, 2) != -1 ||
      (uintptr_t)unit_at(r, 0x1fffffff) != 16 + 16ull * 0x1fffffff) { printf("large\n"); return 1; }
  puts("ok");
}
"""


def test_only_the_rows_own_elements_are_read(tmp_path):
    (tmp_path / "units.cpp").write_text(SOURCE)
    exe = tmp_path / "units"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{PKG_DIR / 'csrc'}", str(tmp_path / "units.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout
