// Interface of the tcgen05 dense-product kernel (linear_tile.cu).
#pragma once

#include <cuda.h>

#include "train_kernels.h"

namespace moe {

struct LinearTileArgs {
  int64_t m;              // rows of D
  int64_t out_cols;       // columns of y: n, or n / 2 for a gated tile
  int gate_rows;          // gated: rows of B between a column's first- and second-half row
  int m_tiles, n_tiles, n_tile;
  int flip;               // the tile's rows are y's columns (few tokens): n_tile is then its token count
  int tile_rows;          // tokens per tile: 256, or n_tile if flipped
  int k_blocks;           // 64-wide K-blocks over all terms of A
  int term_blocks;        // of one term
  int terms;
  int splits;
  int chain;              // K-blocks per accumulator, where a unit is longer
  int64_t full_tiles;     // tiles done whole; the others leave `splits` K slices to the join
  int64_t units;          // full_tiles + splits * (number of the others)
  int early, join_early;  // see train_kernels.h
  int vec;                // rows of y, the residual and the kept z can be accessed in 16 bytes (else a kept z has full_tiles 0)
  float* partial;         // fp32 [tiles not whole][splits][tile_rows][columns], 16-byte aligned; 256 columns if flipped, else n_tile
  LinearEpilogue ep;
};
struct LinearTileMaps {
  CUtensorMap a, b;       // operands
  CUtensorMap out, res;   // bf16 y and its residual in 32 x 32 boxes (vec)
};
// K-blocks per accumulator where long sums are cut: see the kernel's comment on sums. Kept pre-activations have a length that
// y's type does not change, so that their bytes do not depend on it: the root of the K-blocks, 8 at most.
constexpr int linear_chain(bool gated, bool f32, bool keep, int64_t k_blocks) {
  if (!keep) return !f32 ? 256 : gated ? 6 : 12;
  int c = 1;
  while (c < 8 && (c + 1) * c < k_blocks) ++c;
  return c;
}
struct LinearTilePlan {
  int n_tile, splits, flip;
  int64_t full, tail;     // whole tiles, tiles left to the join
};
LinearTilePlan plan_linear_tile(int64_t m, int64_t out_cols, int64_t k_blocks, bool gated, bool grad, bool vec,
                                const LinearEpilogue& ep, int pairs);
cudaError_t launch_linear_tile(bool a_mn, bool b_mn, bool gated, bool keep, const LinearTileMaps& maps,
                               const LinearTileArgs& a, int num_sms, cudaStream_t st);
// The second kernel of a product with tiles that were not done whole.
cudaError_t launch_linear_join(bool gated, bool keep, const LinearTileArgs& a, cudaStream_t st);
// One launch that copies up to two matrices into rows TMA can read (base and row
// stride multiples of 16 bytes).
struct PadArgs {
  const void* src[2];
  void* dst[2];
  int64_t lds[2], ldd[2], rows[2];
  int cols[2];
  int count, early;
  void add(const void* s, int64_t ls, int64_t r, int64_t c, void* d, int64_t ld) {
    src[count] = s;
    dst[count] = d;
    lds[count] = ls;
    ldd[count] = ld;
    rows[count] = r;
    cols[count++] = (int)c;
  }
};
cudaError_t launch_pad(const PadArgs& a, cudaStream_t st);

}  // namespace moe
