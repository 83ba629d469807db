// Gradient of a dense product's pre-activation, dz = dy * act'(z^) with z^ the
// 8-bit checkpoint of z, and its column sums (the bias gradient).
//
//   relu'(z) = [z > 0] (NaN for NaN: a block that overflowed does not leave the
//   gradients in silence), silu'(z) = s (1 + z (1 - s)), gelu'(z) = Phi(z) + z phi(z),
//   SwiGLU y = a silu(b): da = dy silu(b), db = dy a silu'(b), stored as [da | db].
//
// dz is computed in fp32 and written in bf16, the operand type of the two
// gradient products (half a step, at most 2^-8 relative, per value; the products sum
// many of them in fp32). With `terms` = 3 the remainder follows as two more bf16
// matrices, which together hold dz's 24 bits, so that fp32 gradients are as
// exact as an fp32 product (two terms left 2.5e-6 of the result's norm).
//
// Bound by HBM: dy, one byte per z value, two (or six) written per dz value.
// 32 threads take 256 columns (8 neighbouring ones each, 16-byte accesses) and
// 8 thread rows walk a chunk of 64 rows, so a column's sum is in registers until
// the chunk ends; the chunks' sums are added in order by a second kernel, hence
// the bias gradient does not depend on the order in which blocks ran.
#include "train_common.cuh"

namespace moe {

constexpr int kAgRows = 64, kAgCols = 256;

// FAST (dz rounded to bf16 once): hardware exponential and reciprocal, good to
// 2^-20 of 1 + |z|; the exact ones bound the kernel by arithmetic (121 us instead
// of 60 at 16384 x 4096) and serve the three-term form.
template <int HALVES, bool F32, bool VEC, bool FAST>
__global__ void __launch_bounds__(256, 2) act_grad_kernel(ActGradArgs a, int O) {
  __shared__ float red[8][kAgCols];
  __shared__ float scales[HALVES][2][kAgRows];
  pdl_wait();
  pdl_trigger();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * kAgRows;
  const int64_t rend = min(r0 + kAgRows, (int64_t)a.m);
  const int64_t c0 = (int64_t)blockIdx.y * kAgCols;
  auto col = [&](int j) -> int64_t { return VEC ? c0 + 8 * tx + j : c0 + tx + 32 * j; };
  const int64_t nb = (O + 127) / 128;
  __nv_bfloat16* dz = static_cast<__nv_bfloat16*>(a.dz);
  const int64_t term = (int64_t)a.m * a.ldz;
  float sum[HALVES][8];
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[h][j] = 0.f;

  // the chunk's block scales: 2 blocks of 128 columns by 64 rows per half
  if (a.z8 != nullptr)
    for (int i = threadIdx.x; i < HALVES * 2 * kAgRows; i += 256) {
      const int64_t row = r0 + i % kAgRows, kb = 2 * blockIdx.y + (i / kAgRows) % 2;
      scales[i / (2 * kAgRows)][(i / kAgRows) % 2][i % kAgRows] =
          row < rend && kb < nb ? e8m0_value(a.z_scale[((int64_t)(i / (2 * kAgRows)) * nb + kb) * a.m + row]) : 0.f;
    }
  __syncthreads();

  // VEC: four rows' loads are in flight together
  constexpr int U = VEC ? 4 : 1;
  struct Raw {
    uint32_t dy[F32 ? 8 : 4];
    uint2 z[HALVES];
  };
#pragma unroll 1
  for (int64_t row0 = r0 + ty; row0 < rend; row0 += 8 * U) {
    Raw raw[U];
    if constexpr (VEC) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + 8 * u;
#pragma unroll
        for (int j = 0; j < (F32 ? 8 : 4); ++j) raw[u].dy[j] = 0;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) raw[u].z[h] = make_uint2(0, 0);
        if (row < rend && col(0) < O) {
          const uint4* p = F32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(a.dy) + row * a.ldg + col(0))
                               : reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.dy) + row * a.ldg + col(0));
#pragma unroll
          for (int i = 0; i < (F32 ? 2 : 1); ++i) {
            const uint4 w = __ldg(p + i);
            raw[u].dy[4 * i] = w.x;
            raw[u].dy[4 * i + 1] = w.y;
            raw[u].dy[4 * i + 2] = w.z;
            raw[u].dy[4 * i + 3] = w.w;
          }
          if (a.z8 != nullptr)
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
              raw[u].z[h] = __ldg(reinterpret_cast<const uint2*>(a.z8 + ((int64_t)h * a.m + row) * O + col(0)));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + 8 * u;
      if (row >= rend) break;
      float dy[8], z[HALVES][8];
      if constexpr (VEC) {
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < 8; ++j) dy[j] = __uint_as_float(raw[u].dy[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf16(raw[u].dy[j]);
            dy[2 * j] = f.x;
            dy[2 * j + 1] = f.y;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dy[j] = 0.f;
          if (col(j) < O)
            dy[j] = F32 ? static_cast<const float*>(a.dy)[row * a.ldg + col(j)]
                        : (float)static_cast<const __nv_bfloat16*>(a.dy)[row * a.ldg + col(j)];
        }
      }
      if (a.z8 != nullptr) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          if constexpr (VEC) {
            const float s = scales[h][tx >> 4][row - r0];        // 8 aligned columns share a block
            const uint2 w = raw[u].z[h];
            const float2 p0 = e4m3x2_value(w.x & 0xffffu), p1 = e4m3x2_value(w.x >> 16);
            const float2 p2 = e4m3x2_value(w.y & 0xffffu), p3 = e4m3x2_value(w.y >> 16);
            z[h][0] = p0.x * s; z[h][1] = p0.y * s; z[h][2] = p1.x * s; z[h][3] = p1.y * s;
            z[h][4] = p2.x * s; z[h][5] = p2.y * s; z[h][6] = p3.x * s; z[h][7] = p3.y * s;
          } else {
            const uint8_t* zr = a.z8 + ((int64_t)h * a.m + row) * O;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              z[h][j] = col(j) < O ? e4m3_value(zr[col(j)]) * scales[h][j >> 2][row - r0] : 0.f;
          }
        }
        if constexpr (HALVES == 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float b = z[1][j], s = FAST ? sigmoid_fast(b) : sigmoid_f(b), av = z[0][j];
            // __fmul_rn: dz is a rounded value, never the inside of an FMA, so the sums do not
            // depend on which outputs are asked for
            z[0][j] = __fmul_rn(dy[j], b * s);
            z[1][j] = __fmul_rn(dy[j] * av, s * (1.0f + b * (1.0f - s)));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) z[0][j] = __fmul_rn(dy[j], act_slope<FAST>(z[0][j], a.act));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[0][j] = dy[j];
      }
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[h][j] += z[h][j];
        if (dz == nullptr) continue;
        __nv_bfloat16* out = dz + row * a.ldz + (int64_t)h * O;
        // FAST: one term; else three, each the rounded remainder of those before it (the
        // differences are exact); a non-finite value is whole in the first
#pragma unroll
        for (int t = 0; t < (FAST ? 1 : 3); ++t) {
          if constexpr (VEC) {
            if (col(0) < O)
              *reinterpret_cast<uint4*>(out + t * term + col(0)) =
                  make_uint4(pack_bf16(z[h][0], z[h][1]), pack_bf16(z[h][2], z[h][3]), pack_bf16(z[h][4], z[h][5]),
                             pack_bf16(z[h][6], z[h][7]));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (col(j) < O) out[t * term + col(j)] = __float2bfloat16_rn(z[h][j]);
          }
          if constexpr (!FAST)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float part = __bfloat162float(__float2bfloat16_rn(z[h][j]));
              z[h][j] = isfinite(part) ? z[h][j] - part : 0.f;
            }
        }
      }
    }
  }
  if (a.colsum == nullptr) return;
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) red[ty][VEC ? 8 * tx + j : tx + 32 * j] = sum[h][j];
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += red[i][threadIdx.x];
    if (c0 + threadIdx.x < O) a.colsum[(int64_t)blockIdx.x * a.n + (int64_t)h * O + c0 + threadIdx.x] = t;
  }
}

// Sums of the chunks' column sums, 32 columns per block, 8 interleaved chunk
// groups; fp64 because a long batch adds hundreds of chunks.
__global__ void __launch_bounds__(256) colsum_finish_kernel(const float* __restrict__ colsum, int chunks, int n,
                                                            void* __restrict__ out, int f32, int early) {
  __shared__ double red[8][32];
  if (!early) pdl_wait();
  pdl_trigger();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  double t = 0.0;
  if (c < n)
    for (int i = ty; i < chunks; i += 8) t += (double)__ldcg(colsum + (int64_t)i * n + c);
  red[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && c < n) {
    for (int i = 1; i < 8; ++i) t += red[i][tx];
    if (f32) static_cast<float*>(out)[c] = (float)t;
    else static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn((float)t);
  }
  if (early) pdl_wait();
}

int act_grad_chunks(int m, int) { return ceil_div(m, kAgRows); }

static bool al(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

cudaError_t launch_act_grad(const ActGradArgs& a, cudaStream_t st) {
  if (a.m == 0 || a.n == 0) return cudaSuccess;
  const bool two = a.act == kActSwiglu;
  const int O = two ? a.n / 2 : a.n;
  const bool vec = al(a.dy, 16) && a.ldg % (a.dy_f32 ? 4 : 8) == 0 && O % 8 == 0 && (!a.z8 || al(a.z8, 8)) &&
                   (!a.dz || (al(a.dz, 16) && a.ldz % 8 == 0));
  const dim3 grid((unsigned)act_grad_chunks(a.m, a.n), (unsigned)ceil_div(O, kAgCols));
#define MOE_AG(H, F, V)                                                                                      \
  return a.terms == 1 ? launch_kernel(act_grad_kernel<H, F, V, true>, grid, dim3(256), 0, st, true, a, O) \
                      : launch_kernel(act_grad_kernel<H, F, V, false>, grid, dim3(256), 0, st, true, a, O)
  if (two) {
    if (a.dy_f32) { if (vec) MOE_AG(2, true, true); else MOE_AG(2, true, false); }
    else { if (vec) MOE_AG(2, false, true); else MOE_AG(2, false, false); }
  } else {
    if (a.dy_f32) { if (vec) MOE_AG(1, true, true); else MOE_AG(1, true, false); }
    else { if (vec) MOE_AG(1, false, true); else MOE_AG(1, false, false); }
  }
#undef MOE_AG
}

cudaError_t launch_colsum_finish(const float* colsum, int chunks, int n, void* out, bool f32, bool early, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  return launch_kernel(colsum_finish_kernel, dim3(ceil_div(n, 32)), dim3(256), 0, st, true, colsum, chunks, n, out, (int)f32,
                       (int)early);
}

}  // namespace moe
