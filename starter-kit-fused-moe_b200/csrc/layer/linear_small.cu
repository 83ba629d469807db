// Dense products of a few tokens (m <= 32): y = act(x W^T + b) + r, bound by
// the stream of W (2 n k bytes once through HBM), or for small W by latency.
//
// A CTA takes 16 rows of W (for SwiGLU 8 rows of each half, so both factors of
// an output end in the same thread) and all tokens; its 8 warps, and the 1-8
// CTAs of a cluster, split K in chunks of 64 (128 bytes of every row). A warp
// loads W straight into mma.sync fragments with 16-byte loads: lane (g, t) of
// the m16n8k16 layout takes 8 neighbouring values of row g at 8 t, and the
// token operand is taken at the same positions, so the permutation of K inside
// a chunk cancels and nothing passes through shared memory. (A tcgen05 tile would
// spend its rows on padding; the tensor work is not what bounds this.) The partial
// sums meet in shared memory, then across the cluster in distributed shared memory,
// both in a fixed order. The tensor core's additions truncate, so a chain of more
// than 64 of them per warp (K > 8192, or more with a cluster) is cut (CUT): rounded to
// nearest after every 16 or 8. Uncut, K = 262144 lost 1.7e-4 of a sum of one sign. Everywhere, it
// would cost registers and with them an SM's fourth CTA (16 x 2048 x 7168: 14.3 us, not 10.9).
#include "cta_pair.cuh"
#include "train_common.cuh"

namespace moe {

constexpr int kLsWarps = 8;

struct LinearSmallArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* w;
  int64_t ldx, ldw, out_cols;
  int m, k, n;
  LinearEpilogue ep;
};

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
// 8 values of a row at column c (zeros past k).
template <bool VEC>
__device__ __forceinline__ uint4 ls_load(const __nv_bfloat16* row, int c, int k) {
  if constexpr (VEC) {
    return c < k ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = c + 2 * i < k ? __ldg(p + c + 2 * i) : 0, hi = c + 2 * i + 1 < k ? __ldg(p + c + 2 * i + 1) : 0;
      w[i] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

constexpr int ls_unroll(int nt8, bool vec) { return nt8 == 1 && vec ? 4 : 2; }     // chunks in flight

template <int NT8, bool GATED, bool VEC, bool CUT>
__global__ void __launch_bounds__(kLsWarps * 32) linear_small_kernel(LinearSmallArgs a) {
  constexpr int TOK = 8 * NT8, OUT = GATED ? 8 : 16;
  constexpr int U = ls_unroll(NT8, VEC);
  __shared__ float red[kLsWarps][16][TOK + 1];
  __shared__ float part[16][TOK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int cl = gridDim.y, crank = blockIdx.y;
  const int64_t j0 = (int64_t)blockIdx.x * OUT;
  pdl_wait();
  pdl_trigger();
  // rows past the matrix repeat its last one; their results are not stored
  const int64_t r0 = min(j0 + g, a.out_cols - 1);
  const int64_t r1 = GATED ? a.out_cols + r0 : min(j0 + 8 + g, a.out_cols - 1);
  const __nv_bfloat16* w0 = a.w + r0 * a.ldw;
  const __nv_bfloat16* w1 = a.w + r1 * a.ldw;
  float acc[NT8][4], sum[CUT ? NT8 : 1][4];
#pragma unroll
  for (int i = 0; i < NT8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[i][j] = 0.f;
      if constexpr (CUT) sum[i][j] = 0.f;
    }
  const int chunks = (a.k + 63) / 64, step = kLsWarps * cl;
  for (int c0 = crank * kLsWarps + warp; c0 < chunks; c0 += U * step) {
    uint4 wa[U][2], wb[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = (c0 + u * step) * 64 + 32 * h + 8 * t;     // past k: zeros
        wa[u][h] = ls_load<VEC>(w0, c, a.k);
        wb[u][h] = ls_load<VEC>(w1, c, a.k);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT8; ++i) {
        const int tok = 8 * i + g;
        const __nv_bfloat16* xr = a.x + (int64_t)min(tok, a.m - 1) * a.ldx;
        const int lim = tok < a.m ? a.k : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 xv = ls_load<VEC>(xr, (c0 + u * step) * 64 + 32 * h + 8 * t, lim);
          mma_16816(acc[i], wa[u][h].x, wb[u][h].x, wa[u][h].y, wb[u][h].y, xv.x, xv.y);
          mma_16816(acc[i], wa[u][h].z, wb[u][h].z, wa[u][h].w, wb[u][h].w, xv.z, xv.w);
        }
      }
    if constexpr (CUT)
#pragma unroll
      for (int i = 0; i < NT8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[i][j] += acc[i][j];
          acc[i][j] = 0.f;
        }
  }
#pragma unroll
  for (int i = 0; i < NT8; ++i) {
    if constexpr (CUT)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = sum[i][j];
    red[warp][g][8 * i + 2 * t] = acc[i][0];
    red[warp][g][8 * i + 2 * t + 1] = acc[i][1];
    red[warp][g + 8][8 * i + 2 * t] = acc[i][2];
    red[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * TOK; i += kLsWarps * 32) {
    const int r = i & 15, tok = i >> 4;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kLsWarps; ++w) s += red[w][r][tok];
    part[r][tok] = s;
  }
  if (cl > 1) cluster_sync_all();
  else __syncthreads();
  if (crank == 0) {
    const LinearEpilogue& ep = a.ep;
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(ep.bias);
    auto total = [&](int r, int tok) {
      float s = part[r][tok];
      for (int c = 1; c < cl; ++c) s += ld_cluster_f32(mapa_shared(smem_u32(&part[r][tok]), c));
      return s;
    };
    for (int i = threadIdx.x; i < OUT * a.m; i += kLsWarps * 32) {
      const int r = i % OUT, tok = i / OUT;
      const int64_t col = j0 + r;
      if (col >= a.out_cols) continue;
      float v = total(r, tok) + (bias ? __bfloat162float(bias[col]) : 0.f);
      if constexpr (GATED) {
        const float b = total(r + 8, tok) + (bias ? __bfloat162float(bias[a.out_cols + col]) : 0.f);
        v *= act_value(b, kActSilu);
      } else {
        v = act_value(v, ep.act);
      }
      if (ep.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(ep.residual)[tok * ep.ldr + col]);
      if (ep.y_f32) static_cast<float*>(ep.y)[tok * ep.ldy + col] = v;
      else static_cast<__nv_bfloat16*>(ep.y)[tok * ep.ldy + col] = __float2bfloat16_rn(v);
    }
  }
  if (cl > 1) cluster_sync_all();      // the partial sums stay until rank 0 has read them
}

template <int NT8, bool GATED>
static cudaError_t launch_ls(const LinearSmallArgs& a, bool vec, cudaStream_t st) {
  const int64_t groups = (a.out_cols + (GATED ? 7 : 15)) / (GATED ? 8 : 16);
  const int chunks = (a.k + 63) / 64;
  // enough CTAs to fill the SMs a few times over, as long as every warp has a chunk
  int cl = 1;
  while (cl < 8 && groups * cl < 3 * 148 && chunks > kLsWarps * cl) cl *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = cl;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)groups, cl);
  cfg.blockDim = dim3(kLsWarps * 32);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  // additions of a warp's chain: 4 per chunk, whole rounds
  const int u = ls_unroll(NT8, vec), round = kLsWarps * cl * u;
  const bool cut = 4 * u * ((chunks + round - 1) / round) > 64;
  if (vec)
    return cut ? cudaLaunchKernelEx(&cfg, linear_small_kernel<NT8, GATED, true, true>, a)
               : cudaLaunchKernelEx(&cfg, linear_small_kernel<NT8, GATED, true, false>, a);
  return cut ? cudaLaunchKernelEx(&cfg, linear_small_kernel<NT8, GATED, false, true>, a)
             : cudaLaunchKernelEx(&cfg, linear_small_kernel<NT8, GATED, false, false>, a);
}

cudaError_t launch_linear_small(const void* x, int64_t ldx, const void* w, int64_t ldw, int m, int k, int n,
                                const LinearEpilogue& ep, cudaStream_t st) {
  const bool gated = ep.act == kActSwiglu;
  LinearSmallArgs a{static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(w), ldx, ldw,
                    gated ? n / 2 : n, m, k, n, ep};
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && ldx % 8 == 0 &&
                   ldw % 8 == 0 && k % 8 == 0;
  if (m <= 8) return gated ? launch_ls<1, true>(a, vec, st) : launch_ls<1, false>(a, vec, st);
  if (m <= 16) return gated ? launch_ls<2, true>(a, vec, st) : launch_ls<2, false>(a, vec, st);
  return gated ? launch_ls<4, true>(a, vec, st) : launch_ls<4, false>(a, vec, st);
}

}  // namespace moe
