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

// 16 values of a lane as raw words: VEC bf16 columns 8 sub + 64 h (h < 2), else
// columns 4 sub + 32 h (h < 4). Without VEC (rows at any element) bf16 pairs come
// from aligned words, and the bytes leave as aligned words put together with the
// lane before: 143 instead of 242 us for 16384 x 7167 in bf16 (100 for 7166), 137
// instead of 199 in fp32, where the words are whole values.
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
  const int first = (int)-c0, end = (int)(cols - c0);          // the row, from the block's first column
  const int left = min(kBlock, end);
  const bool inside = c0 > 0 && end > kBlock;                  // elements before and behind the block belong to the row
  uint32_t code_mine = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < ITER; i0 += U) {
    uint32_t raw[U][W];
    if (BF && !VEC && inside) {                        // loads without conditions (a row past the last one: the last one's)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T_IN* src = x + min(r0 + 4 * (i0 + u) + rs, rows - 1) * ldx + c0 + 4 * sub;
        const int odd = (int)(reinterpret_cast<uintptr_t>(src) >> 1 & 1);
        const uint32_t* word = reinterpret_cast<const uint32_t*>(src - odd);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t a = __ldg(word + 16 * h), b = __ldg(word + 16 * h + 1), d = __ldg(word + 16 * h + 1 + odd);
          raw[u][2 * h] = __funnelshift_r(a, b, 16 * odd);
          raw[u][2 * h + 1] = __funnelshift_r(b, d, 16 * odd);
        }
      }
    } else
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
          for (int h = 0; h < 4; ++h) {
            const int c = 4 * sub + 32 * h;
            if constexpr (BF) {
              const uint16_t* row16 = reinterpret_cast<const uint16_t*>(src);
              if (reinterpret_cast<uintptr_t>(src) & 2) {
                const uint32_t a = load_pair<false>(row16, c - 1, first, end), b = load_pair<false>(row16, c + 1, first, end);
                const uint32_t d = load_pair<false>(row16, c + 3, first, end);
                raw[u][2 * h] = a >> 16 | b << 16;
                raw[u][2 * h + 1] = b >> 16 | d << 16;
              } else {
                raw[u][2 * h] = load_pair<false>(row16, c, first, end);
                raw[u][2 * h + 1] = load_pair<false>(row16, c + 2, first, end);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c + e < left) raw[u][4 * h + e] = __ldg(reinterpret_cast<const uint32_t*>(src) + c + e);
            }
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
      uint8_t* dst = q + row * cols + c0;
      if constexpr (!VEC) {
        // aligned word sub + 8 h of the block holds positions p .. p + 3, the first ones from the lane before
        const int shift = (int)(reinterpret_cast<uintptr_t>(dst) & 3);
        uint32_t carry = 0;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t up = __shfl_sync(0xffffffffu, o[h], (lane & 24) | ((sub + 7) & 7));
          const uint32_t before = sub ? up : carry;          // lane 0: the last lane's word of the step before
          carry = up;
          const uint32_t w = __funnelshift_l(before, o[h], 8 * shift);
          const int p = 4 * (sub + 8 * h) - shift;
          if (row >= rows) continue;
          if (p >= 0 && p + 3 < left) {
            *reinterpret_cast<uint32_t*>(dst + p) = w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (p + e >= 0 && p + e < left) dst[p + e] = (uint8_t)(w >> (8 * e));
          }
        }
        if (sub == 7 && row < rows)                          // the last word's bytes past the aligned ones
#pragma unroll
          for (int e = 1; e < 4; ++e)
            if (e >= 4 - shift && 124 + e < left) dst[124 + e] = (uint8_t)(o[3] >> (8 * e));
      }
      if (row >= rows) continue;
      if constexpr (VEC) {
#pragma unroll
        for (int h = 0; h < N16; ++h)
          if (c0 + PER * sub + STEP * h < cols) {
            if constexpr (BF) *reinterpret_cast<uint2*>(dst + PER * sub + STEP * h) = make_uint2(o[2 * h], o[2 * h + 1]);
            else *reinterpret_cast<uint32_t*>(dst + PER * sub + STEP * h) = o[h];
          }
      }
    }
  }
  const int64_t row = r0 + 4 * sub + rs;
  if (sub < ITER && row < rows) scale[kb * rows + row] = (uint8_t)code_mine;
}

// q, scale -> bf16 / f32 out with row stride ldo; `batch` matrices one after the
// other (blockIdx.z). A half-warp takes one block of a row, 8 values per lane.
// VEC: out in 16-byte pieces, q too, or (SHIFT) put together from aligned words
// that hold at least one byte of the row.
template <typename T_OUT, int R, bool VEC, bool SHIFT, bool EARLY>
__global__ void __launch_bounds__(kCkWarps * 32) restore_kernel(const uint8_t* __restrict__ q,
                                                                const uint8_t* __restrict__ scale, int64_t rows,
                                                                int64_t cols, int64_t blocks, T_OUT* __restrict__ out,
                                                                int64_t ldo) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 15, half = lane >> 4;
  const int64_t kb = (int64_t)blockIdx.y * kCkWarps + warp;
  const int64_t c0 = kb * kBlock;
  if (!EARLY) pdl_wait();
  pdl_trigger();
  if (c0 >= cols) {
    if (EARLY) pdl_wait();
    return;
  }
  q += (int64_t)blockIdx.z * rows * cols;
  scale += (int64_t)blockIdx.z * blocks * rows;
  out += (int64_t)blockIdx.z * rows * ldo;
  const int64_t r0 = (int64_t)blockIdx.x * R;
  const uint32_t code = lane < R && r0 + lane < rows ? load_input<EARLY>(scale + kb * rows + r0 + lane) : 127u;
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
      if constexpr (SHIFT) {
        const uint8_t* at = src + 8 * sub;
        const int shift = (int)(reinterpret_cast<uintptr_t>(at) & 3);
        const uint32_t* word = reinterpret_cast<const uint32_t*>(at - shift);
        const int64_t left = cols - c0 - 8 * sub + shift;      // bytes of the row from the first word on
        uint32_t w[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) w[j] = 4 * j < left && 4 * j < 8 + shift && left > shift ? load_input<EARLY>(word + j) : 0;
        raw[u] = make_uint2(__funnelshift_r(w[0], w[1], 8 * shift), __funnelshift_r(w[1], w[2], 8 * shift));
      } else if constexpr (VEC) {
        if (c0 + 8 * sub < cols) raw[u] = load_input<EARLY>(reinterpret_cast<const uint2*>(src) + sub);
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c0 + sub + 16 * j < cols) w[j >> 2] |= (uint32_t)load_input<EARLY>(src + sub + 16 * j) << (8 * (j & 3));
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
        if (c0 + 8 * sub < cols) {                             // SHIFT: past cols, into the row's padding
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
  if (EARLY) pdl_wait();
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

// The same where rows lie one after the other at any alignment: q and out have the
// same flat index, so both move in aligned pieces of 16 values, and only the
// scales follow blocks and rows: 74 instead of 123 us for 16384 x 7167 to bf16.
template <typename T_OUT, typename I>
__global__ void __launch_bounds__(256) restore_flat_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                           int64_t total, I rows, I cols, int64_t blocks,
                                                           T_OUT* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  const int64_t f = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (f >= total) return;
  I row = (I)f / cols, col = (I)f - row * cols, b = row / rows;
  row -= b * rows;
  const int count = (int)min((int64_t)16, total - f);
  uint32_t w[4] = {0, 0, 0, 0};
  if (count == 16) {
    const uint4 p = __ldg(reinterpret_cast<const uint4*>(q + f));
    w[0] = p.x;
    w[1] = p.y;
    w[2] = p.z;
    w[3] = p.w;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < count) w[i >> 2] |= (uint32_t)__ldg(q + f + i) << (8 * (i & 3));
  }
  auto scale_at = [&] { return e8m0_value(__ldg(scale + ((int64_t)b * blocks + (int64_t)(col / kBlock)) * (int64_t)rows + (int64_t)row)); };
  float s = scale_at(), v[16];
  int same = (int)min((I)(kBlock - col % kBlock), cols - col);   // values that share it
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 p = e4m3x2_value((w[i >> 2] >> (8 * (i & 3))) & 0xffffu);
    v[i] = p.x;
    v[i + 1] = p.y;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (same == 0 && i < count) {
      if (col == cols) {
        col = 0;
        if (++row == rows) {
          row = 0;
          ++b;
        }
      }
      same = (int)min((I)kBlock, cols - col);
      s = scale_at();
    }
    v[i] *= s;
    ++col;
    --same;
  }
  if (count == 16) {
    uint4* dst = reinterpret_cast<uint4*>(out + f);
    if constexpr (sizeof(T_OUT) == 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        dst[i] = make_uint4(pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                            pack_bf16(v[8 * i + 4], v[8 * i + 5]), pack_bf16(v[8 * i + 6], v[8 * i + 7]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        dst[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                            __float_as_uint(v[4 * i + 3]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < count) out[f + i] = (T_OUT)v[i];
  }
}

template <typename T_OUT>
static cudaError_t restore_flat(const uint8_t* q, const uint8_t* scale, int64_t batch, int64_t rows, int64_t cols,
                                T_OUT* out, cudaStream_t st) {
  const int64_t total = batch * rows * cols, nb = (cols + kBlock - 1) / kBlock;
  const dim3 grid((unsigned)((total + 4095) / 4096)), block(256);
  if (total < 0xffff0000ll)
    return launch_kernel(restore_flat_kernel<T_OUT, uint32_t>, grid, block, 0, st, true, q, scale, total, (uint32_t)rows,
                         (uint32_t)cols, nb, out);
  return launch_kernel(restore_flat_kernel<T_OUT, uint64_t>, grid, block, 0, st, true, q, scale, total, (uint64_t)rows,
                       (uint64_t)cols, nb, out);
}

template <typename T_OUT, bool VEC, bool SHIFT, bool EARLY>
static cudaError_t restore_r(const uint8_t* q, const uint8_t* scale, int64_t batch, int64_t rows, int64_t cols,
                             T_OUT* out, int64_t ldo, cudaStream_t st) {
  const int64_t nb = (cols + kBlock - 1) / kBlock;
  const int r = rows_per_warp(rows, nb * batch, 2);
  const dim3 grid((unsigned)((rows + r - 1) / r), (unsigned)((nb + kCkWarps - 1) / kCkWarps), (unsigned)batch);
  const dim3 block(kCkWarps * 32);
#define MOE_RESTORE(R) \
  return launch_kernel(restore_kernel<T_OUT, R, VEC, SHIFT, EARLY>, grid, block, 0, st, true, q, scale, rows, cols, nb, out, ldo)
  if (r == 32) MOE_RESTORE(32);
  if (r == 8) MOE_RESTORE(8);
  MOE_RESTORE(2);
#undef MOE_RESTORE
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
                           bool f32, cudaStream_t st) {
  if (batch == 0 || rows == 0 || cols == 0) return cudaSuccess;
  const bool vec = al(q, 8) && al(out, 16) && cols % 8 == 0, flat = al(q, 16) && al(out, 16);
  if (f32) {
    auto* p = static_cast<float*>(out);
    return vec    ? restore_r<float, true, false, false>(q, scale, batch, rows, cols, p, cols, st)
           : flat ? restore_flat(q, scale, batch, rows, cols, p, st)
                  : restore_r<float, false, false, false>(q, scale, batch, rows, cols, p, cols, st);
  }
  auto* p = static_cast<__nv_bfloat16*>(out);
  return vec    ? restore_r<__nv_bfloat16, true, false, false>(q, scale, batch, rows, cols, p, cols, st)
         : flat ? restore_flat(q, scale, batch, rows, cols, p, st)
                : restore_r<__nv_bfloat16, false, false, false>(q, scale, batch, rows, cols, p, cols, st);
}

cudaError_t launch_restore_rows(const uint8_t* q, const uint8_t* scale, int64_t rows, int64_t cols, void* out, int64_t ldo,
                                bool early, cudaStream_t st) {
  auto* p = static_cast<__nv_bfloat16*>(out);
  if (al(q, 8) && cols % 8 == 0)
    return early ? restore_r<__nv_bfloat16, true, false, true>(q, scale, 1, rows, cols, p, ldo, st)
                 : restore_r<__nv_bfloat16, true, false, false>(q, scale, 1, rows, cols, p, ldo, st);
  return early ? restore_r<__nv_bfloat16, true, true, true>(q, scale, 1, rows, cols, p, ldo, st)
               : restore_r<__nv_bfloat16, true, true, false>(q, scale, 1, rows, cols, p, ldo, st);
}

}  // namespace moe
