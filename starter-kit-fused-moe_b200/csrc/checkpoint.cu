// 8-bit activation checkpoints: x [rows, cols] (bf16 or f32) -> e4m3
// [rows, cols] + e8m0 [ceil(cols / 128), rows], and back (see train_common.cuh
// for the format). The operator's own quantiser (quantize.cu) divides by
// amax / 448 in fp32; checkpoints use powers of two so that restored values are
// exact in bf16.
//
// Both kernels are bound by HBM: 3 bytes per bf16 value to keep, 3 to bring
// back. A warp walks R rows of one block column and a CTA holds 8 neighbouring
// block columns, so each row is read in 2 KB runs, and the R scales of a warp
// leave as one run of bytes ([blocks, rows] keeps the scales of consecutive rows
// together, the framework's layout). Keeping: 8 lanes take a block of a row (16
// values each, the maximum found on packed 16-bit magnitudes), so that four
// rows share each reduction step; 16 lanes per block spent twice the
// instructions and left the issue slots half busy at 3.7 TB/s.
#include "train_common.cuh"

namespace moe {

constexpr int kCkWarps = 8;

// 16 values of a lane as raw words: bf16 columns 8 sub + 64 h (h < 2) or f32
// columns 4 sub + 32 h (h < 4); element-wise (VEC false) columns sub + 8 j.
template <typename T_IN>
constexpr int kCkRaw = sizeof(T_IN) * 4;

template <typename T_IN, int R, bool VEC>
__global__ void __launch_bounds__(kCkWarps * 32) checkpoint_kernel(const T_IN* __restrict__ x, int64_t rows,
                                                                   int64_t cols, int64_t ldx, uint8_t* __restrict__ q,
                                                                   uint8_t* __restrict__ scale) {
  constexpr bool BF = sizeof(T_IN) == 2;
  constexpr int W = kCkRaw<T_IN>, PER = BF ? 8 : 4, STEP = BF ? 64 : 32, N16 = W / 4;
  constexpr int ITER = R / 4, U = ITER < (BF ? 4 : 2) ? ITER : (BF ? 4 : 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7, rs = lane >> 3;
  const int64_t kb = (int64_t)blockIdx.y * kCkWarps + warp;
  const int64_t c0 = kb * kBlock;
  pdl_wait();
  pdl_trigger();
  if (c0 >= cols) return;
  const int64_t r0 = (int64_t)blockIdx.x * R;
  uint32_t code_mine = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < ITER; i0 += U) {
    uint32_t raw[U][W];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + 4 * (i0 + u) + rs;
      const T_IN* src = x + row * ldx + c0;
#pragma unroll
      for (int j = 0; j < W; ++j) raw[u][j] = 0;
      if (row < rows) {
        if constexpr (VEC) {
#pragma unroll
          for (int h = 0; h < N16; ++h)
            if (c0 + PER * sub + STEP * h < cols)
              *reinterpret_cast<uint4*>(&raw[u][4 * h]) = __ldg(reinterpret_cast<const uint4*>(src + PER * sub + STEP * h));
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + sub + 8 * j < cols) {
              if constexpr (BF)
                raw[u][j >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(src) + sub + 8 * j) << (16 * (j & 1));
              else
                raw[u][j] = __ldg(reinterpret_cast<const uint32_t*>(src) + sub + 8 * j);
            }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // largest magnitude as the bits of a float (NaN above infinity above all)
      uint32_t amax = 0;
      if constexpr (BF) {
#pragma unroll
        for (int j = 0; j < W; ++j) amax = __vmaxu2(amax, raw[u][j] & 0x7fff7fffu);
        amax = max(amax & 0xffff0000u, amax << 16);
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) amax = max(amax, raw[u][j] & 0x7fffffffu);
      }
#pragma unroll
      for (int d = 4; d >= 1; d >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, d));
      const uint32_t code = e8m0_of_amax(amax);
      if (sub == i0 + u) code_mine = code;           // lane (rs, sub) keeps the code of row 4 sub + rs
      const float inv = e8m0_inverse(code);
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        v[j] = inv * __uint_as_float(!BF ? raw[u][BF ? 0 : j] : j & 1 ? raw[u][j >> 1] & 0xffff0000u : raw[u][j >> 1] << 16);
      if (code == kTopScaleCode) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = hold_finite(v[j]);
      }
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = e4m3x4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      const int64_t row = r0 + 4 * (i0 + u) + rs;
      if (row >= rows) continue;
      uint8_t* dst = q + row * cols + c0;
      if constexpr (VEC) {
#pragma unroll
        for (int h = 0; h < N16; ++h)
          if (c0 + PER * sub + STEP * h < cols) {
            if constexpr (BF) *reinterpret_cast<uint2*>(dst + PER * sub + STEP * h) = make_uint2(o[2 * h], o[2 * h + 1]);
            else *reinterpret_cast<uint32_t*>(dst + PER * sub + STEP * h) = o[h];
          }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + sub + 8 * j < cols) dst[sub + 8 * j] = (uint8_t)(o[j >> 2] >> (8 * (j & 3)));
      }
    }
  }
  const int64_t row = r0 + 4 * sub + rs;
  if (sub < ITER && row < rows) scale[kb * rows + row] = (uint8_t)code_mine;
}

// q, scale -> bf16 / f32 out with row stride ldo; `batch` matrices one after the
// other (blockIdx.z). A half-warp takes one block of a row, 8 values per lane.
template <typename T_OUT, int R, bool VEC>
__global__ void __launch_bounds__(kCkWarps * 32) restore_kernel(const uint8_t* __restrict__ q,
                                                                const uint8_t* __restrict__ scale, int64_t rows,
                                                                int64_t cols, int64_t blocks, T_OUT* __restrict__ out,
                                                                int64_t ldo) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 15, half = lane >> 4;
  const int64_t kb = (int64_t)blockIdx.y * kCkWarps + warp;
  const int64_t c0 = kb * kBlock;
  pdl_wait();
  pdl_trigger();
  if (c0 >= cols) return;
  q += (int64_t)blockIdx.z * rows * cols;
  scale += (int64_t)blockIdx.z * blocks * rows;
  out += (int64_t)blockIdx.z * rows * ldo;
  const int64_t r0 = (int64_t)blockIdx.x * R;
  const uint32_t code = lane < R && r0 + lane < rows ? scale[kb * rows + r0 + lane] : 127u;
  constexpr int U = R >= 8 ? 4 : R / 2;
#pragma unroll 1
  for (int i0 = 0; i0 < R / 2; i0 += U) {
    uint2 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + 2 * (i0 + u) + half;
      raw[u] = make_uint2(0, 0);
      if (row >= rows) continue;
      const uint8_t* src = q + row * cols + c0;
      if constexpr (VEC) {
        if (c0 + 8 * sub < cols) raw[u] = __ldg(reinterpret_cast<const uint2*>(src) + sub);
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + sub + 16 * j < cols) w[j >> 2] |= (uint32_t)src[sub + 16 * j] << (8 * (j & 3));
        raw[u] = make_uint2(w[0], w[1]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int l = 2 * (i0 + u) + half;
      const int64_t row = r0 + l;
      const float s = e8m0_value(__shfl_sync(0xffffffffu, code, l));
      if (row >= rows) continue;
      const float2 a = e4m3x2_value(raw[u].x & 0xffffu), b = e4m3x2_value(raw[u].x >> 16);
      const float2 c = e4m3x2_value(raw[u].y & 0xffffu), d = e4m3x2_value(raw[u].y >> 16);
      const float v[8] = {a.x * s, a.y * s, b.x * s, b.y * s, c.x * s, c.y * s, d.x * s, d.y * s};
      T_OUT* dst = out + row * ldo + c0;
      if constexpr (VEC) {
        if (c0 + 8 * sub < cols) {
          if constexpr (sizeof(T_OUT) == 2) {
            reinterpret_cast<uint4*>(dst)[sub] = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                                            pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
          } else {
            reinterpret_cast<float4*>(dst)[2 * sub] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(dst)[2 * sub + 1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + sub + 16 * j < cols) dst[sub + 16 * j] = (T_OUT)v[j];
      }
    }
  }
}

// Rows per warp: as many as keep about 16 warps on every SM.
static int rows_per_warp(int64_t rows, int64_t blocks, int least) {
  for (int r : {32, 8})
    if ((rows + r - 1) / r * blocks >= 148 * 16) return r;
  return least;
}

template <typename T_IN, bool VEC>
static cudaError_t checkpoint_r(const T_IN* x, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q, uint8_t* scale,
                                cudaStream_t st) {
  const int64_t nb = (cols + kBlock - 1) / kBlock;
  const int r = rows_per_warp(rows, nb, 4);
  const dim3 grid((unsigned)((rows + r - 1) / r), (unsigned)((nb + kCkWarps - 1) / kCkWarps));
  const dim3 block(kCkWarps * 32);
  if (r == 32) return launch_kernel(checkpoint_kernel<T_IN, 32, VEC>, grid, block, 0, st, true, x, rows, cols, ldx, q, scale);
  if (r == 8) return launch_kernel(checkpoint_kernel<T_IN, 8, VEC>, grid, block, 0, st, true, x, rows, cols, ldx, q, scale);
  return launch_kernel(checkpoint_kernel<T_IN, 4, VEC>, grid, block, 0, st, true, x, rows, cols, ldx, q, scale);
}

template <typename T_OUT, bool VEC>
static cudaError_t restore_r(const uint8_t* q, const uint8_t* scale, int64_t batch, int64_t rows, int64_t cols,
                             T_OUT* out, int64_t ldo, cudaStream_t st) {
  const int64_t nb = (cols + kBlock - 1) / kBlock;
  const int r = rows_per_warp(rows, nb * batch, 2);
  const dim3 grid((unsigned)((rows + r - 1) / r), (unsigned)((nb + kCkWarps - 1) / kCkWarps), (unsigned)batch);
  const dim3 block(kCkWarps * 32);
  if (r == 32) return launch_kernel(restore_kernel<T_OUT, 32, VEC>, grid, block, 0, st, true, q, scale, rows, cols, nb, out, ldo);
  if (r == 8) return launch_kernel(restore_kernel<T_OUT, 8, VEC>, grid, block, 0, st, true, q, scale, rows, cols, nb, out, ldo);
  return launch_kernel(restore_kernel<T_OUT, 2, VEC>, grid, block, 0, st, true, q, scale, rows, cols, nb, out, ldo);
}

static bool al(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

cudaError_t launch_checkpoint(const void* x, bool bf16, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q,
                              uint8_t* scale, cudaStream_t st) {
  if (rows == 0 || cols == 0) return cudaSuccess;
  const bool vec = al(x, 16) && al(q, 8) && cols % 8 == 0 && ldx % (bf16 ? 8 : 4) == 0;
  if (bf16) {
    const auto* p = static_cast<const __nv_bfloat16*>(x);
    return vec ? checkpoint_r<__nv_bfloat16, true>(p, rows, cols, ldx, q, scale, st)
               : checkpoint_r<__nv_bfloat16, false>(p, rows, cols, ldx, q, scale, st);
  }
  const auto* p = static_cast<const float*>(x);
  return vec ? checkpoint_r<float, true>(p, rows, cols, ldx, q, scale, st)
             : checkpoint_r<float, false>(p, rows, cols, ldx, q, scale, st);
}

cudaError_t launch_restore(const uint8_t* q, const uint8_t* scale, int64_t batch, int64_t rows, int64_t cols, void* out,
                           bool f32, int64_t ldo, cudaStream_t st) {
  if (batch == 0 || rows == 0 || cols == 0) return cudaSuccess;
  const bool vec = al(q, 8) && al(out, 16) && cols % 8 == 0 && ldo % (f32 ? 4 : 8) == 0;
  if (f32) {
    auto* p = static_cast<float*>(out);
    return vec ? restore_r<float, true>(q, scale, batch, rows, cols, p, ldo, st)
               : restore_r<float, false>(q, scale, batch, rows, cols, p, ldo, st);
  }
  auto* p = static_cast<__nv_bfloat16*>(out);
  return vec ? restore_r<__nv_bfloat16, true>(q, scale, batch, rows, cols, p, ldo, st)
             : restore_r<__nv_bfloat16, false>(q, scale, batch, rows, cols, p, ldo, st);
}

}  // namespace moe
