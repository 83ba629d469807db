// Dense products in their simplest form: an fp32 register-tiled product with
// arbitrary strides, then a separate epilogue pass.
#include "train_common.cuh"

namespace moe {

__global__ void __launch_bounds__(256) simple_gemm_kernel(const __nv_bfloat16* __restrict__ A, int64_t am, int64_t ak,
                                                          const __nv_bfloat16* __restrict__ B, int64_t bn, int64_t bk,
                                                          int m, int n, int k, int accumulate, float* __restrict__ out) {
  __shared__ float sa[16][65], sb[16][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i >> 4, c = i & 15;
      sa[c][r] = m0 + r < m && k0 + c < k ? (float)A[(m0 + r) * am + (k0 + c) * ak] : 0.f;
      sb[c][r] = n0 + r < n && k0 + c < k ? (float)B[(n0 + r) * bn + (k0 + c) * bk] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 16; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[c][ty + 16 * i], sb[c][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
      if (r < m && c < n) out[r * n + c] = acc[i][j] + (accumulate ? out[r * n + c] : 0.f);
    }
}

// One warp per (row, 128 output columns): bias, activation, residual, and the
// pre-activation's 8-bit blocks.
__global__ void __launch_bounds__(32) simple_epilogue_kernel(const float* __restrict__ z, int m, int n, int O,
                                                             LinearEpilogue ep) {
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x, c0 = (int64_t)blockIdx.y * 128;
  const int halves = ep.act == kActSwiglu ? 2 : 1;
  const int64_t nb = (O + 127) / 128;
  const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(ep.bias);
  float v[2][4];
  for (int h = 0; h < halves; ++h) {
    uint32_t amax = 0;
    for (int j = 0; j < 4; ++j) {
      const int64_t c = c0 + lane + 32 * j;
      float t = 0.f;
      if (c < O) t = z[row * n + h * O + c] + (bias ? (float)bias[h * O + c] : 0.f);
      v[h][j] = t;
      amax = max(amax, __float_as_uint(t) & 0x7fffffffu);
    }
    if (ep.z8) {
      amax = __reduce_max_sync(0xffffffffu, amax);
      const uint32_t code = e8m0_of_amax(amax);
      const float inv = e8m0_inverse(code);
      if (lane == 0) ep.z_scale[((int64_t)h * nb + blockIdx.y) * m + row] = (uint8_t)code;
      for (int j = 0; j < 4; ++j) {
        const int64_t c = c0 + lane + 32 * j;
        if (c < O)
          ep.z8[((int64_t)h * m + row) * O + c] = (uint8_t)__nv_cvt_float_to_fp8(
              code == kTopScaleCode ? hold_finite(v[h][j] * inv) : v[h][j] * inv, __NV_SATFINITE, __NV_E4M3);
      }
    }
  }
  for (int j = 0; j < 4; ++j) {
    const int64_t c = c0 + lane + 32 * j;
    if (c >= O) continue;
    float y = halves == 2 ? v[0][j] * act_value(v[1][j], kActSilu) : act_value(v[0][j], ep.act);
    if (ep.residual) y += (float)static_cast<const __nv_bfloat16*>(ep.residual)[row * ep.ldr + c];
    if (ep.y_f32) static_cast<float*>(ep.y)[row * ep.ldy + c] = y;
    else static_cast<__nv_bfloat16*>(ep.y)[row * ep.ldy + c] = __float2bfloat16_rn(y);
  }
}

__global__ void simple_store_kernel(const float* __restrict__ z, int64_t count, void* out, int f32) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= count) return;
  if (f32) static_cast<float*>(out)[i] = z[i];
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(z[i]);
}

cudaError_t launch_simple_gemm(const void* A, int64_t am, int64_t ak, const void* B, int64_t bn, int64_t bk, int m,
                               int n, int k, bool accumulate, float* out, cudaStream_t st) {
  if (m == 0 || n == 0) return cudaSuccess;
  simple_gemm_kernel<<<dim3(ceil_div(n, 64), ceil_div(m, 64)), 256, 0, st>>>(
      static_cast<const __nv_bfloat16*>(A), am, ak, static_cast<const __nv_bfloat16*>(B), bn, bk, m, n, k, accumulate, out);
  return cudaGetLastError();
}
cudaError_t launch_simple_epilogue(const float* z, int m, int n, const LinearEpilogue& ep, cudaStream_t st) {
  if (m == 0 || n == 0) return cudaSuccess;
  const int O = ep.act == kActSwiglu ? n / 2 : n;
  simple_epilogue_kernel<<<dim3(m, ceil_div(O, 128)), 32, 0, st>>>(z, m, n, O, ep);
  return cudaGetLastError();
}
cudaError_t launch_simple_store(const float* z, int64_t count, void* out, bool f32, cudaStream_t st) {
  if (count == 0) return cudaSuccess;
  simple_store_kernel<<<(unsigned)((count + 255) / 256), 256, 0, st>>>(z, count, out, f32);
  return cudaGetLastError();
}

}  // namespace moe
