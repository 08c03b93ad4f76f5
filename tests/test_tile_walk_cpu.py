"""The order of a product's tiles and the walk over their stages (csrc/tile_walk.h), compiled for the host."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38_flash_ops_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include <utility>
#include "tile_walk.h"
#define CHECK(x) do { if (!(x)) { printf("%s: m_tiles %d n_tiles %d group %d walkers %d kcount %d stages %d\n", #x, mt, nt, group, walkers, kcount, stages); exit(1); } } while (0)
int main() {
  for (int mt : {1, 2, 3, 7, 8, 9, 16, 17, 33}) for (int nt : {1, 2, 3, 40, 41}) for (int group : {1, mt < 8 ? mt : 8}) for (int walkers : {1, 2, 5, 74, 148})
    for (int kcount : {1, 2, 5}) for (int stages : {2, 3, 12}) {
      const int tiles = mt * nt;
      if (walkers > tiles) continue;
      const qfg::TileGrid grid = {mt, nt, group, 48, 256};
      std::set<std::pair<int, int>> seen;
      for (int first = 0; first < walkers; ++first) {
        int count = 0;
        qfg::StageWalk walk(grid, first);
        for (; walk.tile < tiles; walk.Next(grid, tiles, walkers, kcount, stages), ++count) {
          CHECK(walk.k == count % kcount && walk.stage == count % stages && walk.round == count / stages);
          CHECK(walk.at.n0 % 256 == 0 && walk.at.n0 < nt * 256 && walk.at.m0 % 48 == 0 && walk.at.m0 < mt * 48);
          if (walk.k == 0) CHECK(seen.insert({walk.at.n0, walk.at.m0}).second);
        }
        CHECK(count == (tiles - first + walkers - 1) / walkers * kcount);
      }
      CHECK(static_cast<int>(seen.size()) == tiles);
    }
  puts("walked");
}
"""


def test_every_tile_once_and_nothing_past_the_last(tmp_path):
    """Built to stop at undefined arithmetic (a division by zero rows of a group that does not exist)."""
    source, program = tmp_path / "walk.cc", tmp_path / "walk"
    source.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O0", "-fsanitize=integer-divide-by-zero,signed-integer-overflow", "-fsanitize-undefined-trap-on-error", "-I" + CSRC,
                           str(source), "-o", str(program)])
    r = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "walked\n", (r.returncode, r.stdout)
