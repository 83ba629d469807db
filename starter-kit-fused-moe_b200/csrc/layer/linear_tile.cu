// Dense bf16 products on tcgen05: D[m, n] = sum_k A(m, k) B(n, k), fp32
// accumulation, with the epilogues of a layer.
//
//   forward      A = x   (K-major)     B = W   (K-major)    y = act(D + b) + r, z kept in 8 bits
//   grad_x       A = dz  (K-major)     B = W   (N-major: contraction over W's rows)
//   grad_weight  A = dz  (M-major)     B = x^  (N-major: contraction over the tokens)
//
// A pair of CTAs (a two-CTA cluster, tcgen05 cta_group::2) computes a 256-row
// tile of NT columns: each CTA loads its own 128 rows of A and NT / 2 of B's
// rows, 64 of K per stage, so a stage is at most 32 KB per SM and the operand
// stream (a single CTA with the same tile needs 48 KB per stage) stays below
// what an SM takes in from L2 (68 bytes per cycle measured) while the MMA runs
// at full rate: 512 cycles per 64 of K at NT = 256. Operands arrive by TMA in
// the 128-byte swizzle, in whichever of the two majors they lie in memory, so
// nothing is transposed. dz may come as several bf16 terms (see act_grad.cu):
// the contraction then runs over the terms one after the other with B's
// coordinates repeating.
//
// Sums. The tensor core adds to its fp32 accumulator by truncation, so a long
// chain drifts: 8e-6 of the result's norm at K = 7168, 2e-6 at 2048, 5e-7 at 512 for
// values of both signs (an fp32 product with rounding: 1.0e-6, 4.5e-7, 1.9e-7), and
// 3.7e-7 per 64 of K for values of one sign, which is 1.5e-3 of a bf16 result at
// K = 262144. So the chain is cut (CHAIN): the epilogue warps add each partial
// accumulator to fp32 registers, rounding to nearest, while the tensor core fills
// the other one. The reads of TMEM cost the tensor core about a K-block each.
//  - bf16 results: every 256 K-blocks of 64, which costs nothing that can be seen and
//    leaves 1e-4 of a result at most.
//  - fp32 results: every 12, gated ones every 6, as both factors drift the same way, which
//    keeps them within 1e-6 of the norm: 7e-7 both (16: 1.0e-6, where an fp32 product has 2.5e-7 at
//    K = 1024 and 9e-7 at 7168; 2 % less time at 4096 x 7168 x 4096). Up to K = 768 (384) that is no
//    cut at all.
//  - kept pre-activations, of which an error moves some to the next e4m3 step: every
//    c K-blocks, c the root of their number (8 at most), because the drift grows with c and
//    the error of an fp32 product with the root of K. At 8192 x 512 x 2048 (silu) 1.3e-4 of the norm in
//    such steps and 52 us, uncut 2.0e-4 and 43 us (fp32 1.2e-4); at K = 1024 1.7e-4 and 62 us,
//    with 8 2.3e-4 and 55 us (1.6e-4); at K = 7168 2.5e-4 (2.5e-4).
//
// Warps: 0 TMA producer, 1 MMA issuer (the leader CTA's), 4-11 epilogue. The two
// accumulators of NT columns in TMEM also let a tile's epilogue overlap the next
// tile's products. Persistent grid, one pair per two SMs; tiles are walked in
// bands of 8 row tiles so that the tiles in flight share both operands in L2.
//
// The tiles that do not fill a last round of the pairs (all of them, when there
// are fewer tiles than pairs) are cut into K slices: the slices leave fp32
// partial tiles in the workspace and a second kernel, launched to start as this
// one ends, adds them in slice order and runs the epilogue on all SMs. (Letting
// the slice that arrives last do it kept the other SMs idle: 36 instead of 20 us
// at 1037 x 1111 x 515.) With a kept pre-activation, outputs whose rows 16-byte
// accesses cannot reach take that way for every tile: the second kernel reaches
// any column with whole warps, while a lane holding a row of the tile stores
// element by element (215 instead of 60 us for a 1911 x 594 x 5181 product).
//
// Every wait is bounded (2 s). One that runs out makes the kernel write NaN to
// the tiles it still owes, so a failed call never returns plausible numbers; the
// block then gives its copies in flight a millisecond before it leaves.
#include "cta_pair.cuh"
#include "linear_tile.h"
#include "moe_kernels.h"
#include "train_common.cuh"

namespace moe {

constexpr int kLtStages = 6, kLtStageBytes = 32768, kLtTileA = 16384;
constexpr int kLtThreads = 384, kLtEpiWarps = 8, kLtTmemCols = 512;
// CHAIN keeps 128 sums per epilogue thread in registers: the warpgroup of the producer
// and the MMA issuer hands registers to the two epilogue warpgroups. The split
// has to add up to what the block is launched with.
constexpr int kLtRegsLaunch = 168, kLtRegsIssue = 40, kLtRegsEpi = 232;
static_assert(kLtRegsIssue * 128 + kLtRegsEpi * 256 <= kLtRegsLaunch * kLtThreads, "register split");
constexpr int kLtBand = 8;
constexpr int kLtStaging = 4096;     // per epilogue warp: a 32 x 32 box of fp32, or two of bf16

struct LinearTileSmem {
  uint64_t full[kLtStages];
  uint64_t empty[kLtStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint32_t tmem_base;
  int abort_flag;
  uint64_t res[kLtEpiWarps][2];   // a warp's residual boxes have arrived
};
constexpr size_t kLtSmem = 1024 + (size_t)kLtStages * kLtStageBytes + (size_t)kLtEpiWarps * kLtStaging + sizeof(LinearTileSmem);
static_assert(kLtSmem <= 232448, "shared memory budget");

// bf16 x bf16 -> f32, M = 256 over the pair; a_mn / b_mn: operand stored with M / N innermost.
__device__ __forceinline__ uint32_t idesc_bf16(int n, int a_mn, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}
// Descriptor of an M- or N-major operand in the 128-byte swizzle: 64 values of
// M (N) by 8 of K make a 1024-byte group; the next 8 of K follow (stride 1024),
// the next 64 of M are 64 K-rows (8192 bytes) away.
__device__ __forceinline__ uint64_t sdesc_sw128_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(8192 >> 4) << 16;    // LBO: next 64 of M / N
  d |= (uint64_t)(1024 >> 4) << 32;    // SBO: next 8 of K
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_bf16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* m, uint32_t bar_cluster, int x, int y,
                                                 int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// 32 lanes x 32-bit, 32 or 64 consecutive columns per thread. A load of TMEM
// queues behind the MMAs issued so far, so partial sums are taken in few
// instructions: 32 columns at a time held the tensor core up for 1.6 us per
// accumulator, 64 for 0.8.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%2"
      "7,%28,%29,%30,%31"
      "}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%2"
      "7,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%5"
      "2,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr));
}

// The producer's and the issuer's loops run with their whole warp converged and
// elect one lane around the instructions themselves: the operands then stay in
// uniform registers. Under a lane == 0 branch every tcgen05.mma cost 62 cycles of
// issue and the loop 545 a stage, as long as the MMAs themselves at NT = 256.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

struct LtUnit {
  int mt, nt, kb0, kb1, slice;
  int64_t tile;
};
// Row and column tile of a tile index: bands of 8 row tiles, rows fastest.
__device__ __forceinline__ void lt_place(const LinearTileArgs& a, int64_t tile, int& mt, int& nt) {
  const int64_t per_band = (int64_t)kLtBand * a.n_tiles;
  const int band = (int)(tile / per_band);
  const int in = (int)(tile - band * per_band);
  const int rows = min(kLtBand, a.m_tiles - band * kLtBand);
  nt = in / rows;
  mt = band * kLtBand + in - nt * rows;
}
template <bool FLIP>
__device__ __forceinline__ LtUnit lt_unit(const LinearTileArgs& a, int64_t u) {
  LtUnit r;
  if (u < a.full_tiles) {
    r.tile = u;
    r.slice = -1;
    r.kb0 = 0;
    r.kb1 = a.k_blocks;
  } else {
    const int64_t v = u - a.full_tiles, i = v / a.splits;
    r.tile = a.full_tiles + i;
    r.slice = (int)(v - i * a.splits);
    r.kb0 = (int)((int64_t)r.slice * a.k_blocks / a.splits);
    r.kb1 = (int)((int64_t)(r.slice + 1) * a.k_blocks / a.splits);
  }
  if constexpr (FLIP) {
    r.mt = (int)r.tile;
    r.nt = 0;
  } else {
    lt_place(a, r.tile, r.mt, r.nt);
  }
  return r;
}

// ---- epilogue pieces, 16 or 32 columns of one row per thread
__device__ __forceinline__ void lt_bias16(const __nv_bfloat16* bias, int64_t c, int64_t end, float* v) {
  if (c + 16 <= end && (reinterpret_cast<uintptr_t>(bias + c) & 15) == 0) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(bias + c)), b = __ldg(reinterpret_cast<const uint4*>(bias + c) + 1);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = unpack_bf16(w[i]);
      v[2 * i] += f.x;
      v[2 * i + 1] += f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c + i < end) v[i] += __bfloat162float(bias[c + i]);
  }
}
__device__ __forceinline__ void lt_bias32(const __nv_bfloat16* bias, int64_t c, int64_t end, float* v) {
  lt_bias16(bias, c, end, v);
  lt_bias16(bias, c + 16, end, v + 16);
}
// bf16 results take silu and gelu from the hardware exponential and reciprocal (2^-20 of
// 1 + |z|), fp32 ones from the exact ones: the epilogue is bound by its
// instructions, and silu's exact quotient is half of them.
__device__ __forceinline__ float lt_silu(float z, bool exact) {
  return exact ? act_value(z, kActSilu) : z * sigmoid_fast(z);
}
__device__ __forceinline__ void lt_act32(float* v, int act, bool exact) {
  if (act == kActNone) return;
  if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = act_value(v[i], kActRelu);
  } else if (act == kActGelu) {
    if (exact) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_value(v[i], kActGelu);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= normal_cdf<true>(v[i]);
    }
  } else if (exact) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = lt_silu(v[i], true);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = lt_silu(v[i], false);
  }
}
__device__ __forceinline__ void lt_gate32(float* v, const float* z, bool exact) {
  if (exact) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= lt_silu(z[i], true);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= lt_silu(z[i], false);
  }
}
// Stores of a warp's 32 rows go through shared memory: a lane holds a row, so
// direct stores touch 32 lines with 16 bytes each, and a tile's epilogue took
// longer than a short contraction (71 us for the gate's fp32 input gradient).
// Boxes of 32 rows by 32 columns: bf16 ones leave by TMA, which fetches the
// residual's boxes too and cuts off what lies past the matrix; fp32 ones are
// copied out in whole 128-byte lines, because a TMA store queues behind the
// producer's loads and a warp has room for one fp32 box only (42 us against 33).
__device__ __forceinline__ void lt_stage_f32(uint8_t* box, const float* v, int lane) {       // 128-byte swizzle
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<float4*>(box + lane * 128 + ((i ^ (lane & 7)) << 4)) =
        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
// `rows` rows and `cols` columns of the staged box to dst (16-byte aligned rows `ld` floats apart).
__device__ __forceinline__ void lt_copy_f32(const uint8_t* box, float* dst, int64_t ld, int rows, int64_t cols, int lane) {
  __syncwarp();
  const int p = lane & 7;
  dst += 4 * p;
  cols -= 4 * p;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    const float4 v = *reinterpret_cast<const float4*>(box + r * 128 + ((p ^ (r & 7)) << 4));
    float* d = dst + r * ld;
    if (r >= rows || cols <= 0) continue;
    if (cols >= 4) {
      *reinterpret_cast<float4*>(d) = v;
    } else {
      d[0] = v.x;
      if (cols > 1) d[1] = v.y;
      if (cols > 2) d[2] = v.z;
    }
  }
  __syncwarp();
}
// The same for rows that 16-byte accesses cannot reach: a row of the box per
// store, a column per lane, the residual read the same way. Bound by its
// instructions: pointers that walk, instead of an index per element, 17.4 instead of
// 24.9 us (residual: 32.8 instead of 43.7) at 4096 x 1024 x 2049. Eight rows at a
// time: 16 or 32 took longer (53 and more with the residual).
template <typename T>
__device__ __forceinline__ void lt_copy_rows(const uint8_t* box, T* y, int64_t ldy, const __nv_bfloat16* res, int64_t ldr,
                                             int rows, bool in, int lane) {
  __syncwarp();
  uint32_t at = smem_u32(box) + (lane & 3) * 4;
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += 8, at += 1024) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(at + i * 128 + (((lane >> 2) ^ i) << 4)) : "memory");
    if (res != nullptr) {
      __nv_bfloat16 f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = __float2bfloat16_rn(0.f);
        if (in && r0 + i < rows) f[i] = *res;
        res += ldr;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += __bfloat162float(f[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (in && r0 + i < rows) *y = (T)v[i];
      y += ldy;
    }
  }
  __syncwarp();
}
__device__ __forceinline__ uint4* lt_bf16_piece(uint8_t* box, int i, int lane) {             // 64-byte swizzle
  return reinterpret_cast<uint4*>(box + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4));
}
__device__ __forceinline__ void lt_stage_bf16(uint8_t* box, const float* v, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *lt_bf16_piece(box, i, lane) = make_uint4(pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                                              pack_bf16(v[8 * i + 4], v[8 * i + 5]), pack_bf16(v[8 * i + 6], v[8 * i + 7]));
}
__device__ __forceinline__ void lt_box_out(const CUtensorMap* m, const uint8_t* box, int x, int64_t y, int lane) {
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(m, smem_u32(box), x, (int)y);
    bulk_commit();
  }
}
// Waits until at most N of the warp's stores still read their boxes.
template <int N>
__device__ __forceinline__ void lt_boxes_free(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
  __syncwarp();
}
// Largest magnitude (as bits) of the columns below `end`.
__device__ __forceinline__ uint32_t lt_amax32(const float* v, int64_t c, int64_t end, uint32_t amax) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (c + i < end) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  return amax;
}
__device__ __forceinline__ void lt_store_z32(uint8_t* z, int64_t c, int64_t end, const float* v, uint32_t code) {
  const float inv = e8m0_inverse(code);
  const bool hold = code == kTopScaleCode;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = v[4 * i + j] * inv;
    if (hold) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = hold_finite(s[j]);
    }
    w[i] = e4m3x4(s[0], s[1], s[2], s[3]);
  }
  if (c + 16 <= end) *reinterpret_cast<uint4*>(z + c) = make_uint4(w[0], w[1], w[2], w[3]);     // end: a multiple of 16
  if (c + 32 <= end) *reinterpret_cast<uint4*>(z + c + 16) = make_uint4(w[4], w[5], w[6], w[7]);
}

template <bool A_MN, bool B_MN, bool GATED, bool KEEP, bool CHAIN, bool FLIP>
__global__ void __launch_bounds__(kLtThreads, 1)
    linear_tile_kernel(const __grid_constant__ LinearTileMaps maps, const LinearTileArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + kLtStages * kLtStageBytes;
  LinearTileSmem& S = *reinterpret_cast<LinearTileSmem*>(staging + kLtEpiWarps * kLtStaging);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int crank = (int)cluster_rank();
  const int64_t wid = cluster_id(), G = gridDim.x / 2;
  const int NT = a.n_tile, H = NT / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kLtStages; ++s) {
      mbar_init(smem_u32(&S.full[s]), 1);
      mbar_init(smem_u32(&S.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&S.tfull[b]), 1);
      mbar_init(smem_u32(&S.tempty[b]), 2 * kLtEpiWarps);      // both CTAs' epilogues (the leader's copy)
    }
    for (int w = 0; w < kLtEpiWarps; ++w)
      for (int b = 0; b < 2; ++b) mbar_init(smem_u32(&S.res[w][b]), 1);
    S.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.a);
    tma_prefetch_desc(&maps.b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem_base)),
                 "r"(kLtTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  if (!a.early) pdl_wait();
  pdl_trigger();
  const uint32_t tmem_base = S.tmem_base;
  volatile int* abort_flag = &S.abort_flag;

  if (warp < 4) {
    if constexpr (CHAIN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLtRegsIssue));
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      int s = 0;
      uint32_t parity = 1;
      bool ok = true;
      const uint32_t bytes = 2 * (kLtTileA + H * 128);
      const uint32_t full0 = smem_u32(&S.full[0]), empty0 = smem_u32(&S.empty[0]), stage0 = smem_u32(smem);
      const uint32_t leader0 = mapa_shared(full0, 0);      // both CTAs' loads complete on the leader's barriers
      const int k_end = a.term_blocks * 64;
      for (int64_t u = wid; u < a.units && ok && !__shfl_sync(0xffffffffu, *abort_flag, 0); u += G) {
        const LtUnit x = lt_unit<FLIP>(a, u);
        const int m0 = FLIP && GATED ? crank * a.gate_rows + x.mt * 128 : x.mt * 256 + crank * 128;
        // B rows of this CTA's half: the next H columns of the tile, or for a gated tile its first-half
        // (leader) and second-half (peer) rows
        const int n0 = GATED && !FLIP ? crank * a.gate_rows + x.nt * H : x.nt * NT + crank * H;
        // the small terms first: the chain's truncation is relative to the running sum
        int term = a.terms - 1 - x.kb0 / a.term_blocks;
        int kt = (x.kb0 % a.term_blocks) * 64;
        for (int kb = x.kb0; kb < x.kb1; ++kb) {
          if (!warp_wait(empty0 + 8 * s, parity)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          const uint32_t sa = stage0 + s * kLtStageBytes, sb = sa + kLtTileA, bar = leader0 + 8 * s;
          if (elect_one()) {
            if (crank == 0) mbar_arrive_expect_tx(full0 + 8 * s, bytes);
            if constexpr (A_MN) {
              tma_load_3d_pair(sa, &maps.a, bar, m0, kt, term);
              tma_load_3d_pair(sa + 8192, &maps.a, bar, m0 + 64, kt, term);
            } else {
              tma_load_3d_pair(sa, &maps.a, bar, kt, m0, term);
            }
            if constexpr (B_MN) {
              tma_load_2d_pair(sb, &maps.b, bar, n0, kt);
              if (H == 128) tma_load_2d_pair(sb + 8192, &maps.b, bar, n0 + 64, kt);
            } else {
              tma_load_2d_pair(sb, &maps.b, bar, kt, n0);
            }
          }
          kt += 64;
          if (kt == k_end) {
            kt = 0;
            --term;
          }
          if (++s == kLtStages) {
            s = 0;
            parity ^= 1;
          }
        }
      }
    } else if (warp == 1 && crank == 0) {
      // ------------------------------------------------------------ MMA issuer (leader)
      const uint32_t idesc = idesc_bf16(NT, A_MN, B_MN);
      // test hook: a non-zero value withholds the accumulators, so that the epilogue's wait runs out
      const bool withhold = *reinterpret_cast<const volatile int*>(&g_gate_extra) != 0;
      int s = 0, tt = 0;                                   // stage, accumulator
      uint32_t parity = 0;
      bool ok = true;
      const uint32_t full0 = smem_u32(&S.full[0]), empty0 = smem_u32(&S.empty[0]);
      // descriptors of stage 0; an address step of n bytes is n / 16 in their low word
      const uint64_t a0 = A_MN ? sdesc_sw128_mn(smem_u32(smem)) : sdesc_sw128(smem_u32(smem));
      const uint64_t b0 = B_MN ? sdesc_sw128_mn(smem_u32(smem) + kLtTileA) : sdesc_sw128(smem_u32(smem) + kLtTileA);
      for (int64_t u = wid; u < a.units && ok && !__shfl_sync(0xffffffffu, *abort_flag, 0); u += G) {
        const LtUnit x = lt_unit<FLIP>(a, u);
        for (int kb = x.kb0; kb < x.kb1 && ok; ++tt) {
          const int b = tt & 1, end = CHAIN ? min(kb + a.chain, x.kb1) : x.kb1;
          if (!warp_wait(smem_u32(&S.tempty[b]), ((tt >> 1) & 1) ^ 1)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + (uint32_t)(b * 256);
          uint32_t more = 0;
          for (; kb < end; ++kb, more = 1) {
            if (!warp_wait(full0 + 8 * s, parity)) {
              *abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t da = a0 + (uint32_t)(s * (kLtStageBytes / 16)), db = b0 + (uint32_t)(s * (kLtStageBytes / 16));
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_bf16_pair(d, da + kk * (A_MN ? 128 : 2), db + kk * (B_MN ? 128 : 2), idesc, kk ? 1u : more);
              mma_commit_pair(empty0 + 8 * s);
            }
            if (++s == kLtStages) {
              s = 0;
              parity ^= 1;
            }
          }
          if (ok && !withhold && elect_one()) mma_commit_pair(smem_u32(&S.tfull[b]));
          __syncwarp();
        }
      }
    }
  } else {
    if constexpr (CHAIN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLtRegsEpi));
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, g = (warp - 4) >> 2, ew = warp - 4;
    const int r = 32 * q + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(32 * q) << 16);
    const LinearEpilogue& ep = a.ep;
    const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(ep.bias);
    const int64_t O = a.out_cols;
    const int64_t z_blocks = (O + 127) / 128;
    uint8_t* stage = staging + ew * kLtStaging;
    const uint32_t stage_addr = smem_u32(stage);
    // y as bf16 in whole boxes with a residual: the residual's boxes are fetched into the boxes y leaves from
    const bool res_boxes = ep.residual != nullptr && !ep.y_f32 && a.vec;
    constexpr int CHUNKS_H = GATED ? 4 : 2;              // this warp's columns: NT / CHUNKS_H
    bool ok = true, res_ok = true;
    int tt = 0;
    uint32_t res_count = 0;                              // residual boxes waited for
    uint32_t out_box = 0;                                // without a residual: the box of the next store, across tiles
    for (int64_t u = wid; u < a.units; u += G) {
      const LtUnit x = lt_unit<FLIP>(a, u);
      const int64_t row0 = (int64_t)x.mt * 256 + crank * 128 + 32 * q, row = row0 + lane;
      const bool valid = row < a.m;
      const int warp_rows = (int)max((int64_t)0, min((int64_t)32, a.m - row0));
      const int w = NT / CHUNKS_H;                       // columns of y per warp
      const int64_t c0 = (int64_t)x.nt * (GATED ? H : NT) + g * w;     // the first of them
      const int chunks = (int)min((int64_t)(w / 32), (O - c0 + 31) / 32);
      const bool live = warp_rows > 0 && chunks > 0;
      auto fetch_residual = [&](int j) {                 // chunk j into box j & 1, whose last store has been read
        if (lane == 0 && res_ok) {                       // a box that never came may not be armed again
          const uint32_t bar = smem_u32(&S.res[ew][j & 1]);
          mbar_arrive_expect_tx(bar, 2048);
          tma_load_2d(stage_addr + (j & 1) * 2048, &maps.res, bar, (int)c0 + 32 * j, (int)row0);
        }
      };
      auto fetch_first = [&] {
        if (res_boxes && live && x.slice < 0) {
          lt_boxes_free<0>(lane);
          fetch_residual(0);
          if (chunks > 1) fetch_residual(1);
        }
      };
      if constexpr (!(GATED && KEEP)) fetch_first();     // ahead of the product
      // the accumulator at hand (CHAIN: the one whose partial sums are taken)
      auto wait_acc = [&] {
        const int b = tt & 1;
        if (ok && (*abort_flag || !mbar_wait(smem_u32(&S.tfull[b]), (tt >> 1) & 1))) {
          *abort_flag = 1;
          ok = false;
        }
        tc_fence_after();
      };
      auto release = [&] {                               // back to the leader's MMA
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&S.tempty[tt & 1]), 0));
        ++tt;
      };
      auto acc_at = [&](int col) { return lane_addr + (uint32_t)((tt & 1) * 256 + col); };
      auto from_tmem = [&](int col, float* v) {          // 32 columns
        tmem_ld32(acc_at(col), v);
        tmem_ld_wait();
        if (!ok) {                                       // a wait ran out: NaN instead of sums
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = NAN;
        }
      };
      // CHAIN: the thread's sums, columns g H + i of the tile (gated: g w + i of the first half, and from sum[64]
      // on those of the second half)
      float sum[CHAIN ? 128 : 1];
      if constexpr (CHAIN) {
        for (int kb = x.kb0; kb < x.kb1; kb += a.chain) {
          wait_acc();
          // two loads of up to 64 columns (gated: a half each); columns past w are not used
          const int col1 = GATED ? H + g * w : g * w + 64;
          const bool two = GATED || w > 64;
          if (kb == x.kb0) {
            tmem_ld64(acc_at(g * w), sum);
            if (two) tmem_ld64(acc_at(col1), sum + 64);
            tmem_ld_wait();
          } else {
            float v[64];
            tmem_ld64(acc_at(g * w), v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 64; ++e) sum[e] += v[e];
            if (two) {
              tmem_ld64(acc_at(col1), v);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 64; ++e) sum[64 + e] += v[e];
            }
          }
          release();
        }
        if (!ok) {
#pragma unroll
          for (int e = 0; e < 128; ++e) sum[e] = NAN;
        }
      } else {
        wait_acc();
      }
      if constexpr (FLIP) {                              // always a slice: fp32 [token][column], a lane holds a column
        const int first = g * H;                         // of this warp's tokens
        float* dst = a.partial + ((x.tile * a.splits + x.slice) * NT + first) * 256 + crank * 128 + r;
        const int tokens = (int)min((int64_t)H, a.m - first);
#pragma unroll 1
        for (int i = 0; i < tokens; i += 32) {
          float v[32];
          from_tmem(first + i, v);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (i + e < tokens) __stcg(dst + (i + e) * 256, v[e]);
        }
        release();
        continue;
      }
      if (x.slice >= 0) {                                // fp32 partial tile, [row][column]
        if (warp_rows > 0) {
          const int64_t y0 = ((x.tile - a.full_tiles) * a.splits + x.slice) * 256 + crank * 128 + 32 * q;
          lt_boxes_free<0>(lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int lc = GATED && i >= 2 ? 32 * (i - 2) : 32 * i;
            if (lc >= w) continue;
            const int col = g * w + lc + (GATED && i >= 2 ? H : 0);
            if constexpr (CHAIN) {
              lt_stage_f32(stage, sum + 32 * i, lane);
            } else {
              float v[32];
              from_tmem(col, v);
              lt_stage_f32(stage, v, lane);
            }
            lt_copy_f32(stage, a.partial + y0 * NT + col, NT, warp_rows, 32, lane);
          }
        }
        if constexpr (!CHAIN) release();
        continue;
      }
      // y's columns [c0 + 32 j, + 32)
      auto store = [&](int j, float* v) {
        const int64_t c = c0 + 32 * j;
        if (!KEEP && !a.vec) {
          lt_stage_f32(stage, v, lane);
          const bool in = lane < O - c;
          const __nv_bfloat16* res =
              ep.residual != nullptr ? static_cast<const __nv_bfloat16*>(ep.residual) + row0 * ep.ldr + c + lane : nullptr;
          const int64_t at = row0 * ep.ldy + c + lane;
          if (ep.y_f32) lt_copy_rows(stage, static_cast<float*>(ep.y) + at, ep.ldy, res, ep.ldr, warp_rows, in, lane);
          else lt_copy_rows(stage, static_cast<__nv_bfloat16*>(ep.y) + at, ep.ldy, res, ep.ldr, warp_rows, in, lane);
        } else if (ep.y_f32) {
          if (ep.residual != nullptr && valid) {
            const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(ep.residual) + row * ep.ldr;
            lt_bias32(r, c, O, v);
          }
          lt_stage_f32(stage, v, lane);
          lt_copy_f32(stage, static_cast<float*>(ep.y) + row0 * ep.ldy + c, ep.ldy, warp_rows, O - c, lane);
        } else {
          // without a residual the boxes alternate over all of the warp's stores: a tile may end on either one (NT of
          // 192, one chunk per tile, a cut-off last column tile), and the wait below leaves the last store reading
          uint8_t* box = stage + (res_boxes ? j & 1 : out_box) * 2048;
          if (res_boxes) {
            // waited for in a failed call too: a box that arrives later would cover the NaN staged here
            if (res_ok && !mbar_wait(smem_u32(&S.res[ew][j & 1]), (res_count >> (j & 1)) & 1)) {
              *abort_flag = 1;
              ok = res_ok = false;
            }
            if (!res_ok) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = NAN;
            }
            res_count ^= 1u << (j & 1);                  // each box's phase flips with every use
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 p = *lt_bf16_piece(box, i, lane);
              const uint32_t pw[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack_bf16(pw[e]);
                v[8 * i + 2 * e] += f.x;
                v[8 * i + 2 * e + 1] += f.y;
              }
            }
          } else {
            lt_boxes_free<1>(lane);
            out_box ^= 1;
          }
          lt_stage_bf16(box, v, lane);
          lt_box_out(&maps.out, box, (int)c, row0, lane);
          if (res_boxes && j + 2 < chunks) {
            lt_boxes_free<0>(lane);
            fetch_residual(j + 2);
          }
        }
      };

      if constexpr (CHAIN) {
        if (bias)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int jj = GATED ? j & 1 : j, h = GATED ? j >> 1 : 0;
            if (jj < chunks) lt_bias32(bias + h * O, c0 + 32 * jj, O, sum + 32 * j);
          }
      }
      uint32_t code[2] = {0, 0};
      if constexpr (KEEP) {                              // NT = 256: not gated, a warp's half is one block of the row
        uint32_t amax[2] = {0, 0};
        if constexpr (CHAIN) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int jj = GATED ? j & 1 : j, h = GATED ? j >> 1 : 0;
            if (jj < chunks) amax[h] = lt_amax32(sum + 32 * j, c0 + 32 * jj, O, amax[h]);
          }
        } else {
#pragma unroll 1
          for (int j = 0; j < chunks; ++j)
#pragma unroll
            for (int h = 0; h < (GATED ? 2 : 1); ++h) {
              float v[32];
              from_tmem(g * w + 32 * j + h * H, v);
              if (bias) lt_bias32(bias + h * O, c0 + 32 * j, O, v);
              amax[h] = lt_amax32(v, c0 + 32 * j, O, amax[h]);
            }
        }
        if constexpr (GATED) {                           // a block of each half per tile, shared by two warps:
          lt_boxes_free<0>(lane);                        // the maxima pass through the warps' staging boxes
          uint32_t* mine = reinterpret_cast<uint32_t*>(stage) + lane;
          const uint32_t* other = reinterpret_cast<const uint32_t*>(stage + (g ? -4 : 4) * kLtStaging) + lane;
          mine[0] = amax[0];
          mine[32] = amax[1];
          fence_proxy_async_smem();                      // the residual's boxes come after these words
          named_barrier_sync(2 + q, 64);
          amax[0] = max(amax[0], other[0]);
          amax[1] = max(amax[1], other[32]);
          named_barrier_sync(2 + q, 64);
          fetch_first();
        }
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h) {
          code[h] = e8m0_of_amax(amax[h]);
          if (valid && chunks > 0 && (!GATED || g == 0)) ep.z_scale[(h * z_blocks + (c0 >> 7)) * a.m + row] = (uint8_t)code[h];
        }
      }
      if constexpr (CHAIN) {
        if (live) {
          if constexpr (GATED) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (j < chunks) {
                if constexpr (KEEP)
                  if (valid) {
                    lt_store_z32(ep.z8 + row * O, c0 + 32 * j, O, sum + 32 * j, code[0]);
                    lt_store_z32(ep.z8 + (a.m + row) * O, c0 + 32 * j, O, sum + 64 + 32 * j, code[1]);
                  }
                lt_gate32(sum + 32 * j, sum + 64 + 32 * j, ep.y_f32);
                store(j, sum + 32 * j);
              }
          } else {
#pragma unroll 1
            for (int j = 0; j < chunks; ++j) {           // one body for the chunks: the sums move down
              if constexpr (KEEP)
                if (valid) lt_store_z32(ep.z8 + row * O, c0 + 32 * j, O, sum, code[0]);
              lt_act32(sum, ep.act, ep.y_f32);
              store(j, sum);
#pragma unroll
              for (int e = 0; e < 96; ++e) sum[e] = sum[e + 32];
            }
          }
        }
      } else {
        if (live) {
          float v[GATED ? 64 : 32];                      // gated: 32 of each half
#pragma unroll 1
          for (int j = 0; j < chunks; ++j) {
            const int64_t c = c0 + 32 * j;
            if constexpr (GATED) {
              tmem_ld32(acc_at(g * w + 32 * j), v);
              tmem_ld32(acc_at(g * w + 32 * j + H), v + 32);
              tmem_ld_wait();
              if (!ok) {
#pragma unroll
                for (int e = 0; e < 64; ++e) v[e] = NAN;
              }
            } else {
              from_tmem(g * w + 32 * j, v);
            }
            if (bias) {
              lt_bias32(bias, c, O, v);
              if constexpr (GATED) lt_bias32(bias + O, c, O, v + 32);
            }
            if constexpr (KEEP)
              if (valid) {
                lt_store_z32(ep.z8 + row * O, c, O, v, code[0]);
                if constexpr (GATED) lt_store_z32(ep.z8 + (a.m + row) * O, c, O, v + 32, code[1]);
              }
            if constexpr (GATED) {
              lt_gate32(v, v + 32, ep.y_f32);
            } else {
              lt_act32(v, ep.act, ep.y_f32);
            }
            store(j, v);
          }
        }
        release();
      }
    }
    if (lane == 0) bulk_wait_all();                      // stores complete before the CTA exits
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  cluster_sync_all();      // neither CTA leaves while the other may still signal its barriers
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kLtTmemCols) : "memory");
  }
  if (a.early) pdl_wait();
}

// A warp takes 512 columns of a row, as 4-byte words: where the row starts at an
// odd element, a word's halves come from two neighbouring aligned words (the
// second one from L1, or from L2 in an early launch). Words that reach past the row are read in halves.
template <bool EARLY>
__global__ void __launch_bounds__(256) pad_kernel(PadArgs a) {
  if (!EARLY) pdl_wait();
  pdl_trigger();
  const int j = blockIdx.z, lane = threadIdx.x & 31, w0 = 256 * blockIdx.y + lane, cols = a.cols[j];
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < a.rows[j]; row += (int64_t)gridDim.x * 8) {
    const uint16_t* s = static_cast<const uint16_t*>(a.src[j]) + row * a.lds[j];
    uint32_t* d = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.dst[j]) + row * a.ldd[j]);
    const bool odd = reinterpret_cast<uintptr_t>(s) & 2;
    uint32_t v[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = 2 * (w0 + 32 * e);
      v[e] = load_pair<EARLY>(s, odd ? c - 1 : c, 0, cols);
      if (odd) u[e] = load_pair<EARLY>(s, c + 1, 0, cols);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = 2 * (w0 + 32 * e);
      if (c < cols) d[w0 + 32 * e] = odd ? v[e] >> 16 | u[e] << 16 : v[e];
    }
  }
  if (EARLY) pdl_wait();
}
cudaError_t launch_pad(const PadArgs& a, cudaStream_t st) {
  if (a.count == 0) return cudaSuccess;
  int64_t rows = 1;
  int cols = 1;
  for (int j = 0; j < a.count; ++j) {
    rows = rows > a.rows[j] ? rows : a.rows[j];
    cols = cols > a.cols[j] ? cols : a.cols[j];
  }
  const int segments = (cols + 511) / 512;                 // cols <= 2^23
  int64_t blocks = (rows + 7) / 8;
  if (blocks * segments > 148 * 32) blocks = (148 * 32 + segments - 1) / segments;
  const dim3 grid((unsigned)blocks, segments, a.count);
  return a.early ? launch_kernel(pad_kernel<true>, grid, dim3(256), 0, st, true, a)
                 : launch_kernel(pad_kernel<false>, grid, dim3(256), 0, st, true, a);
}

// Adds the K slices' partial rows in slice order and runs the epilogue. A warp
// takes a block of 128 output columns of R rows, so a block of the 8-bit
// pre-activation is one warp's; the partial rows come from L2, where the product
// has just left them, those of up to four rows in flight together. VEC: 4 neighbouring
// columns per lane and 16-byte rows; else columns lane + 32 j, one by one.
template <bool GATED, bool KEEP, bool VEC, int R>
__global__ void __launch_bounds__(256) linear_join_kernel(LinearTileArgs a) {
  const int lane = threadIdx.x & 31;
  if (!a.join_early) pdl_wait();
  pdl_trigger();
  const int cols = a.flip ? 256 : a.n_tile, H = GATED ? cols / 2 : cols, col_blocks = (H + 127) / 128;
  const uint32_t per_tile = a.tile_rows / (8 * R) * col_blocks;                    // blocks of 8 R rows and 128 columns
  const uint32_t i = blockIdx.x / per_tile, in = blockIdx.x - i * per_tile;
  const int r0 = (int)(in / col_blocks) * 8 * R + (threadIdx.x >> 5) * R, cb = (int)(in % col_blocks);
  int mt, nt;
  lt_place(a, a.full_tiles + i, mt, nt);
  const int64_t row0 = (int64_t)mt * 256 + r0;
  const int64_t O = a.out_cols, c0 = (int64_t)nt * H + 128 * cb;          // the warp's first column
  if (row0 >= a.m || c0 >= O) {                                           // warp-uniform
    if (a.join_early) pdl_wait();
    return;
  }
  const int rows = (int)min((int64_t)R, a.m - row0);
  const int width = (int)min((int64_t)min(128, H - 128 * cb), O - c0);    // its columns
  const int64_t kb = c0 / 128, blocks = (O + 127) / 128, step = (int64_t)a.tile_rows * cols;
  const LinearEpilogue& ep = a.ep;
  const __nv_bfloat16* bias = static_cast<const __nv_bfloat16*>(ep.bias);
  auto col = [&](int j) { return VEC ? 4 * lane + j : lane + 32 * j; };
  constexpr int HALVES = GATED ? 2 : 1, U = R < 4 ? R : 4;
  float b[HALVES][4];
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) b[h][j] = bias && col(j) < width ? __bfloat162float(bias[h * O + c0 + col(j)]) : 0.f;
  const float* tile = a.partial + (int64_t)i * a.splits * step + (int64_t)r0 * cols + 128 * cb;
#pragma unroll 1
  for (int rb = 0; rb < rows; rb += U) {
    float v[U][HALVES][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u][h][j] = 0.f;
#pragma unroll(R == 1 ? 4 : 2)
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          if (rb + u >= rows) continue;
          const float* q = tile + s * step + (int64_t)(rb + u) * cols + h * H;
          if constexpr (VEC) {
            if (col(0) >= width) continue;                                // a tile's width is a multiple of 32
            const float4 f = __ldcg(reinterpret_cast<const float4*>(q) + lane);
            v[u][h][0] += f.x;
            v[u][h][1] += f.y;
            v[u][h][2] += f.z;
            v[u][h][3] += f.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col(j) < width) v[u][h][j] += __ldcg(q + lane + 32 * j);
          }
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (rb + u >= rows) continue;
      const int64_t row = row0 + rb + u;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[u][h][j] += b[h][j];
      if constexpr (KEEP) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          uint32_t amax = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col(j) < width) amax = max(amax, __float_as_uint(v[u][h][j]) & 0x7fffffffu);
          const uint32_t code = e8m0_of_amax(__reduce_max_sync(0xffffffffu, amax));
          const float inv = e8m0_inverse(code);
          if (lane == 0) ep.z_scale[(h * blocks + kb) * a.m + row] = (uint8_t)code;
          float s[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) s[j] = code == kTopScaleCode ? hold_finite(v[u][h][j] * inv) : v[u][h][j] * inv;
          const uint32_t w = e4m3x4(s[0], s[1], s[2], s[3]);
          uint8_t* z = ep.z8 + (h * a.m + row) * O + c0;
          if constexpr (VEC) {
            if (col(0) < width) *reinterpret_cast<uint32_t*>(z + col(0)) = w;   // O is a multiple of 16
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col(j) < width) z[col(j)] = (uint8_t)(w >> (8 * j));
          }
        }
      }
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        y[j] = GATED ? v[u][0][j] * lt_silu(v[u][HALVES - 1][j], ep.y_f32)
                     : ep.act == kActSilu ? lt_silu(v[u][0][j], ep.y_f32) : act_value(v[u][0][j], ep.act);
      const __nv_bfloat16* r = static_cast<const __nv_bfloat16*>(ep.residual) + row * ep.ldr + c0;
      float* yf = static_cast<float*>(ep.y) + row * ep.ldy + c0;
      __nv_bfloat16* yb = static_cast<__nv_bfloat16*>(ep.y) + row * ep.ldy + c0;
      if (VEC && col(3) < width) {
        if (ep.residual) {
          const uint2 w = *reinterpret_cast<const uint2*>(r + col(0));
          const float2 f0 = unpack_bf16(w.x), f1 = unpack_bf16(w.y);
          y[0] += f0.x;
          y[1] += f0.y;
          y[2] += f1.x;
          y[3] += f1.y;
        }
        if (ep.y_f32) *reinterpret_cast<float4*>(yf + col(0)) = make_float4(y[0], y[1], y[2], y[3]);
        else *reinterpret_cast<uint2*>(yb + col(0)) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col(j) < width) {
          if (ep.residual) y[j] += __bfloat162float(r[col(j)]);
          if (ep.y_f32) yf[col(j)] = y[j];
          else yb[col(j)] = __float2bfloat16_rn(y[j]);
        }
    }
  }
  if (a.join_early) pdl_wait();
}

template <bool GATED, bool KEEP>
static cudaError_t launch_join(const LinearTileArgs& a, cudaStream_t st) {
  const int64_t tail = (a.units - a.full_tiles) / a.splits, cols = a.flip ? 256 : a.n_tile;
  const int64_t col_blocks = ((GATED ? cols / 2 : cols) + 127) / 128, rows = a.m < a.tile_rows ? a.m : a.tile_rows;
  // 8 rows per warp once that leaves 16 warps per SM, else one
  const bool many = tail * col_blocks * rows / 8 >= 148 * 16;
  const dim3 grid((unsigned)(tail * col_blocks * (a.tile_rows / (many ? 64 : 8)))), block(256);
#define MOE_JOIN(V, R) launch_kernel(linear_join_kernel<GATED, KEEP, V, R>, grid, block, 0, st, true, a)
  if (many) return a.vec ? MOE_JOIN(true, 8) : MOE_JOIN(false, 8);
  return a.vec ? MOE_JOIN(true, 1) : MOE_JOIN(false, 1);
#undef MOE_JOIN
}

// Tile width and K slices of the last, partial round. Cycles per 64 of K and
// pair, measured: 2.1 NT for a pair alone (the MMA), 174 + 2.3 NT with all pairs
// at work (758 at NT = 256, 590 at 192, 466 at 128), and no less than the
// operands' way from HBM (3.4 KB per cycle); 800 for a change of tile. A tile's
// epilogue hides behind the next tile's products except for the last one, which
// is long where rows are written element-wise. (Joining the one tile of a small
// product whose pre-activation is kept, 64 x 256 x 256 with gelu, takes 9.1 instead
// of 14.5 us on the device, but one launch more costs a host-bound step more: 25.7
// instead of 21.7 us with the checkpoint and both restores.)
// Slices are at least 4 K-blocks deep; joining them costs a launch and moves 8
// bytes per value and slice through L2 (about 3 KB per cycle).
LinearTilePlan plan_linear_tile(int64_t m, int64_t n, int64_t k_blocks, bool gated, bool grad, bool vec,
                                const LinearEpilogue& ep, int pairs) {
  LinearTilePlan best{};
  double best_cost = 1e300;
  const bool keep = ep.z8 != nullptr;
  const int64_t mt = (m + 255) / 256;
  const double hbm = 128.0 * k_blocks * (m + (gated ? 2 : 1) * n) / 3400;
  // the last tile's epilogue, cycles per column of the tile
  const double last = keep ? 20 : vec ? 12 : ep.residual ? 80 : ep.y_f32 ? 45 : 20;
  static const int widths[] = {256, 192, 128, 64};
  for (int nt : widths) {
    if (keep && nt != 256) continue;
    if ((gated || grad) && nt % 128) continue;       // epilogue warps take 32 columns; boxes of 64
    const int64_t cols = gated ? nt / 2 : nt;
    const int64_t tiles = mt * ((n + cols - 1) / cols);
    const double alone = 2.1 * nt, crowded = 174 + 2.3 * nt;
    const double rows = m < 256 ? m : 256;
    for (int s = 0; s <= 16; ++s) {                  // 0: every tile whole
      if (s == 0 && keep && !vec) continue;
      const int64_t tail = s == 0 ? tiles % pairs : keep && !vec ? tiles : tiles % pairs, full = tiles - tail;
      const int slices = s ? s : 1;
      if (s > 0 && tail == 0) break;
      if (s > 1 && k_blocks < 4 * s) break;
      const int64_t units = tail * slices, rounds = (units + pairs - 1) / pairs;
      const double busy = units < pairs ? (double)units / pairs : 1.0;
      double cost = (double)(full / pairs) * (k_blocks * crowded + 800) +
                    (double)rounds * ((k_blocks + slices - 1) / slices * (alone + busy * (crowded - alone)) + 800);
      cost = (cost > hbm ? cost : hbm) + 1500 + (s ? 12 * nt + 4000 + 8.0 * s * tail * rows * nt / 3000 : last * nt);
      if (cost < best_cost) {
        best_cost = cost;
        best = {nt, slices, 0, s ? full : tiles, s ? tail : 0};
      }
    }
  }
  // Few tokens and a long contraction: the weights' rows become the tile's, which pads 64 or 128 columns instead of 256
  // rows, but always needs the join. At 64 (128) tokens and K = 7168 16.2 (18.3) instead of 19.2 (22.8) us for N = 4096
  // gated, 25.8 instead of 29.3 for N = 7168, 10.2 instead of 12.8 for N = 256; at K = 5120 14.0 (15.1) instead of 16.2 (19.0), at
  // 4096 12.8 (13.9) instead of 16.1 (17.2), at 2048 11.8 (11.4) instead of 12.8 (12.0) but 12.9 instead of 11.8 for
  // N = 7168 (weights that change, in a graph). The limit was set when the slices left HBM idle below it.
  if (m <= 128 && k_blocks >= 96 && !keep && !grad) {
    best_cost = 1e300;
    const int nt = m <= 64 ? 64 : 128;
    const int64_t tail = (n + (gated ? 127 : 255)) / (gated ? 128 : 256);
    for (int s = 1; s <= 16; ++s) {
      const int64_t depth = (k_blocks + s - 1) / s;
      if (s > 1 && k_blocks < 4 * s) break;
      if (depth > linear_chain(gated, ep.y_f32, false, k_blocks)) continue;                // longer chains drift
      const int64_t units = tail * s, rounds = (units + pairs - 1) / pairs;
      // 52 pairs reach what HBM gives (32 of them 5 of 6.5 TB/s), fewer a part of it, those of the last round too; a
      // slice more is also a load more, one after the other, in the join
      const int64_t rest = units % pairs;
      const double stream = hbm / units * (units - rest + (rest > 52 ? rest : rest ? 52 : 0));
      double cost = (double)rounds * (depth * (200.0 + 1.4 * nt) + 800);
      cost = (cost > stream ? cost : stream) + 1500 + 12.0 * nt + 4000 + 500.0 * s + 8.0 * s * tail * m * 256 / 3000;
      if (cost < best_cost) {
        best_cost = cost;
        best = {nt, s, 1, 0, tail};
      }
    }
  }
  return best;
}

template <bool A_MN, bool B_MN, bool GATED, bool KEEP, bool CHAIN, bool FLIP = false>
static cudaError_t launch_c(const LinearTileMaps& maps, const LinearTileArgs& a, int num_sms, cudaStream_t st) {
  static int clusters_of[64];
  auto kern = linear_tile_kernel<A_MN, B_MN, GATED, KEEP, CHAIN, FLIP>;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kLtThreads);
  cfg.dynamicSmemBytes = kLtSmem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = dev < 64 ? clusters_of[dev] : 0;
  if (clusters == 0) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kLtSmem);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(num_sms & ~1);
    e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg);
    if (e != cudaSuccess || clusters < 1) return e != cudaSuccess ? e : cudaErrorInvalidConfiguration;
    if (clusters > num_sms / 2) clusters = num_sms / 2;
    if (dev < 64) clusters_of[dev] = clusters;
  }
  const int64_t want = a.units < clusters ? a.units : clusters;
  cfg.gridDim = dim3((unsigned)(2 * want));
  cfg.stream = st;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, maps, a);
}

template <bool A_MN, bool B_MN, bool GATED, bool KEEP>
static cudaError_t launch_t(const LinearTileMaps& maps, const LinearTileArgs& a, int num_sms, cudaStream_t st) {
  // cut the chain where a unit is longer than one piece
  const int unit = a.full_tiles > 0 ? a.k_blocks : (a.k_blocks + a.splits - 1) / a.splits;
  if (unit > a.chain) return launch_c<A_MN, B_MN, GATED, KEEP, true>(maps, a, num_sms, st);
  return launch_c<A_MN, B_MN, GATED, KEEP, false>(maps, a, num_sms, st);
}

cudaError_t launch_linear_tile(bool a_mn, bool b_mn, bool gated, bool keep, const LinearTileMaps& maps,
                               const LinearTileArgs& a, int num_sms, cudaStream_t st) {
  if (a.flip) return gated ? launch_c<false, false, true, false, false, true>(maps, a, num_sms, st)
                           : launch_c<false, false, false, false, false, true>(maps, a, num_sms, st);
  if (a_mn && b_mn) return launch_t<true, true, false, false>(maps, a, num_sms, st);
  if (b_mn) return launch_t<false, true, false, false>(maps, a, num_sms, st);
  if (gated) return keep ? launch_t<false, false, true, true>(maps, a, num_sms, st)
                         : launch_t<false, false, true, false>(maps, a, num_sms, st);
  return keep ? launch_t<false, false, false, true>(maps, a, num_sms, st)
              : launch_t<false, false, false, false>(maps, a, num_sms, st);
}

cudaError_t launch_linear_join(bool gated, bool keep, const LinearTileArgs& a, cudaStream_t st) {
  if (a.units == a.full_tiles) return cudaSuccess;
  if (gated) return keep ? launch_join<true, true>(a, st) : launch_join<true, false>(a, st);
  return keep ? launch_join<false, true>(a, st) : launch_join<false, false>(a, st);
}

static const bool g_debug_waits_added = (add_debug_waits(set_debug_waits_here), true);

}  // namespace moe
