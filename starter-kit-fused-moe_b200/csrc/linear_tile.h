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
  int k_blocks;           // 64-wide K-blocks over all terms of A
  int term_blocks;        // of one term
  int terms;
  int splits;
  int chain;              // K-blocks per accumulator where long sums are cut (fp32 y, kept pre-activations)
  int64_t full_tiles;     // tiles done whole; the others leave `splits` K slices to the join
  int64_t units;          // full_tiles + splits * (number of the others)
  int vec;                // rows of y, the residual and the kept z can be accessed in 16 bytes (else full_tiles is 0)
  float* partial;         // fp32 [tiles not whole][splits][256][n_tile], 16-byte aligned
  LinearEpilogue ep;
};
struct LinearTileMaps {
  CUtensorMap a, b;       // operands
  CUtensorMap out, res;   // bf16 y and its residual in 32 x 32 boxes (vec)
};
struct LinearTilePlan {
  int n_tile, splits;
  int64_t full, tail;     // whole tiles, tiles left to the join
};
LinearTilePlan plan_linear_tile(int64_t m, int64_t out_cols, int64_t k_blocks, bool gated, bool keep, bool b_mn, bool direct,
                                int pairs);
cudaError_t launch_linear_tile(bool a_mn, bool b_mn, bool gated, bool keep, const LinearTileMaps& maps,
                               const LinearTileArgs& a, int num_sms, cudaStream_t st);
// One launch that copies up to two matrices into rows TMA can read (base and row
// stride multiples of 16 bytes).
struct PadArgs {
  const void* src[2];
  void* dst[2];
  int64_t lds[2], ldd[2], rows[2];
  int cols[2];
  int count;
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
