// Which tile comes when, of a product cut into row blocks and column blocks, and the walk of a CTA (or cluster) over its tiles and their stages.
// Plain C++, so that it can be compiled and tested without a GPU.
#pragma once

#ifdef __CUDACC__
#define QFG_WALK __host__ __device__ __forceinline__
#else
#define QFG_WALK inline
#endif

namespace qfg {

struct At {
  int n0, m0;  // the first column and row
};

// Tiles go down `group` row blocks, then on to the next column block, and through all of these before the next group: the tiles of a wave then share
// about as many rows of x as columns of w in L2.
struct TileGrid {
  int m_tiles, n_tiles, group;  // row blocks, column blocks
  int bm, bn;                   // rows and columns of a tile

  QFG_WALK At Locate(int tile) const {  // tile < m_tiles * n_tiles
    const int g = tile / (group * n_tiles), rest = tile - g * group * n_tiles, left = m_tiles - g * group, rows = group < left ? group : left, nt = rest / rows;
    return {nt * bn, (g * group + rest - nt * rows) * bm};
  }
};

// Every stage of every tile from `first` on, `step` apart, through a ring of `stages`.
struct StageWalk {
  int tile, k = 0, stage = 0, round = 0;  // round: how often the ring has been gone through
  At at;

  QFG_WALK StageWalk(const TileGrid& grid, int first) : tile(first), at(grid.Locate(first)) {}
  QFG_WALK void Next(const TileGrid& grid, int tiles, int step, int kcount, int stages) {
    if (++stage == stages) {
      stage = 0;
      ++round;
    }
    if (++k == kcount) {
      k = 0;
      tile += step;
      if (tile < tiles) at = grid.Locate(tile);  // behind the last group there are no rows to divide by
    }
  }
};

}  // namespace qfg
