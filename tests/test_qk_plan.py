"""How a call of the head norm with rotation is cut into tiles: the host's rules (egnn_qk_plan.h), compiled for the CPU."""
import subprocess

from pymolecular_amd import _build

DIVISIONS = r"""
#include <cstdio>
#include <initializer_list>
#include "egnn_qk_plan.h"
using namespace egnn::qk;
// The kernel's numbers of rows and heads of a tile, against integer division: they are monotone between a row's first head and
// its last, so these two show all.
int main() {
  long checked = 0;
  for (int D : {2, 4, 6, 8, 10, 16, 24, 32, 34, 48, 64, 96, 126, 128})
    for (int how = 0; how < 8; ++how)
      for (long N : {1l, 5000l, 263168l, 524288l, 2147483647l})
        for (int H = 1; H <= 4096; ++H)
          for (int few : {1, 2, 3, 64}) {
            if (few > H) continue;
            EgnnQkDims d{};
            const bool bwd = how & 1;
            d.N = N; d.Hq = how & 2 ? few : H; d.Hk = how & 2 ? H : few; d.D = D; d.rotary = D; d.interleaved = how >> 2;
            d.dtype = EGNN_BF16; d.base = 1e4;
            const int rows = tile_rows(&d, bwd);
            if (rows < 1 || rows * (D / 2 + 2) > kTable) { printf("D %d H %d %d N %ld: %d rows\n", D, H, few, N, rows); return 1; }
            if (H == 1) continue;
            for (long r = 0; r < rows; ++r)
              for (long k : {r * H, r * H + H - 1}) {
                ++checked;
                if ((long)((unsigned long)k * reciprocal(H) >> 32) != r) {
                  printf("D %d H %d %d N %ld bwd %d: head %ld of row %ld\n", D, H, few, N, (int)bwd, k - r * H, r);
                  return 1;
                }
              }
          }
  printf("%ld\n", checked);
}
"""


def _run(tmp_path, program, *flags):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(program)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(_build.CSRC), *flags, str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)


def test_rows_of_a_tile_are_divided_exactly(tmp_path):
    r = _run(tmp_path, DIVISIONS)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout) > 10 ** 7
