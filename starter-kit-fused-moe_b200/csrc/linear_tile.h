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
  int splits;
  int64_t units;          // tiles * splits
  int vec;                // y (and the residual) can be accessed in 16 bytes
  float* partial;         // splits > 1: [units][2][n_tile][128] fp32
  int* arrivals;          // splits > 1: [tiles][2], zero at launch
  LinearEpilogue ep;
};
struct LinearTilePlan {
  int n_tile, splits;
  int64_t tiles;
};
LinearTilePlan plan_linear_tile(int64_t m, int64_t out_cols, int64_t k_blocks, bool gated, bool keep, bool b_mn, int pairs);
cudaError_t launch_linear_tile(bool a_mn, bool b_mn, bool gated, bool keep, const CUtensorMap& tmA,
                               const CUtensorMap& tmB, const LinearTileArgs& a, int num_sms, cudaStream_t st);
cudaError_t launch_pad_rows(const void* src, int64_t lds, int64_t rows, int64_t cols, void* dst, int64_t ldd,
                            cudaStream_t st);

}  // namespace moe
