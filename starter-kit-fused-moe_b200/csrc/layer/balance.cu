// The router's balance loss with its per-expert counts, and the gradient of the
// routing logits.
//
// For every sequence q (tokens [cu[q], cu[q+1])), with T_q its tokens that
// select at least one expert, E experts and k picks per token:
//   p_te    = s_te / (sum_j s_tj + 1e-20), s = sigmoid(logit)   (or softmax)
//   f_qe    = E / (k T_q) * (times expert e was picked in q)
//   P_qe    = 1 / T_q * sum_t p_te
//   loss    = alpha * mean over non-empty sequences of sum_e f_qe P_qe
// A pick outside [0, E) selects nothing; a token all of whose picks do so is
// padding (the exchange buffers of expert parallelism mark rows past a rank's
// tokens this way) and counts nowhere, whatever its logits hold. Gradient
// (f does not depend on the logits):
//   c_e = g alpha E / (k n_seq T_q^2) * count_qe
//   d loss / d logit_te = (c_e - sum_j c_j p_tj) / (sum_j s_tj + 1e-20) * s_te (1 - s_te)
//   (softmax: p_te (c_e - sum_j c_j p_tj)),
// and, with the gradient dw of the combine weights w_k = s_k / (sum_sel s + 1e-20) * scale,
//   d / d logit_k += (dw_k scale - sum_j dw_j scale s_j / S) / S * s_k (1 - s_k), S = sum_sel s + 1e-20.
//
// Forward: blocks of consecutive tokens, a warp per token, the sums of a
// (block, sequence) pair in registers and shared memory, stored to slot
// block + sequence (unique: along the tokens one of the two grows with every
// new pair, so no list is needed and nothing is added atomically); a second
// kernel adds a sequence's slots in order, fp64, one block per sequence and 32
// experts, and its last block adds up the loss in order. The result does not
// depend on the order in which blocks run. Backward: one pass, a warp per
// token. Both read the logits once and are bound by latency at a few hundred
// tokens and by HBM (or L2, which holds the logits of 16k tokens) above.
#include "train_common.cuh"

namespace moe {

constexpr int kBalWarps = 8;
constexpr float kScoreEps = 1e-20f;

static int balance_chunk(int t) {   // tokens per block: about three blocks per SM, a multiple of the warps
  const int c = align_up(ceil_div(t, 3 * 148), kBalWarps);
  return c < kBalWarps ? kBalWarps : c;
}

struct BalanceWs {
  float* p;        // [blocks + s, e]
  int32_t* c;      // [blocks + s, e]
  int32_t* t;      // [blocks + s]
  double* loss;    // [s * groups]
  int32_t* state;  // [1]: finished blocks of the second kernel
};
static size_t up(size_t x) { return (x + 255) & ~size_t(255); }
static size_t balance_ws(int t, int e, int s, uint8_t* base, BalanceWs* w) {
  const size_t slots = (size_t)ceil_div(t, balance_chunk(t)) + s;
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o += up(bytes); return base + at; };
  uint8_t* p = take(slots * e * 4);
  uint8_t* c = take(slots * e * 4);
  uint8_t* tt = take(slots * 4);
  uint8_t* l = take((size_t)s * ceil_div(e, 32) * 8);
  uint8_t* st = take(4);
  if (w) *w = {reinterpret_cast<float*>(p), reinterpret_cast<int32_t*>(c), reinterpret_cast<int32_t*>(tt),
               reinterpret_cast<double*>(l), reinterpret_cast<int32_t*>(st)};
  return o;
}
size_t balance_workspace_bytes(int t, int e, int s) { return balance_ws(t, e, s, nullptr, nullptr); }

// Bounds of sequence q, held inside [0, t] whatever cu contains.
__device__ __forceinline__ void seq_bounds(const int32_t* cu, int q, int t, int& a, int& b) {
  if (cu == nullptr) {
    a = 0;
    b = t;
    return;
  }
  a = min(max(__ldg(cu + q), 0), t);
  b = min(max(__ldg(cu + q + 1), a), t);
}
// The last sequence that starts at or before token x (0 if none does): every
// round looks at 32 boundaries at once, one per lane.
__device__ __forceinline__ int seq_of(const int32_t* cu, int s, int x, int lane) {
  int lo = 0, hi = cu == nullptr ? 1 : s;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, i = lo + lane * step;
    const uint32_t m = __ballot_sync(0xffffffffu, lane == 0 || (i < hi && __ldg(cu + i) <= x));
    lo += (31 - __clz(m)) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// The experts of a lane: lane + 32 j, or (VEC: E = 32 ITEMS, a multiple of 128,
// 16-byte aligned rows) groups of four, 128 apart.
template <bool VEC>
__device__ __forceinline__ int expert_of(int lane, int j) {
  return VEC ? 4 * lane + (j & 3) + 128 * (j >> 2) : lane + 32 * j;
}
template <int ITEMS, bool VEC>
__device__ __forceinline__ void load_logits(const float* row, int e, int lane, float* x) {
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < ITEMS; j += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(row + 32 * j) + lane);
      x[j] = v.x;
      x[j + 1] = v.y;
      x[j + 2] = v.z;
      x[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) x[j] = lane + 32 * j < e ? __ldg(row + lane + 32 * j) : -INFINITY;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// Unnormalised scores of a token (experts past E: 0) and the inverse of their
// sum. The hardware exponential and reciprocal are good to 2^-21 of a score at
// |logit| = 8, and the kernels are bound by their instructions with the exact ones.
template <int ITEMS>
__device__ __forceinline__ float scores(const float* x, int scoring, float* s) {
  float sum = 0.f;
  if (scoring == 0) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      s[j] = sigmoid_fast(x[j]);
      sum += s[j];
    }
    return 1.0f / (warp_sum(sum) + kScoreEps);
  }
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    m = fmaxf(m, x[j]);
    nan |= x[j] != x[j];
  }
  m = warp_max(m);
  if (__any_sync(0xffffffffu, nan)) m = NAN;
  if (m == -INFINITY) {          // nothing to choose from: no scores
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) s[j] = 0.f;
    return 0.f;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    s[j] = __expf(x[j] - m);
    sum += s[j];
  }
  return 1.0f / warp_sum(sum);
}

template <int ITEMS, bool VEC>
__global__ void __launch_bounds__(kBalWarps * 32, ITEMS <= 8 ? 4 : 1) balance_partial_kernel(BalanceArgs a, BalanceWs w, int chunk) {
  __shared__ float psum[kBalWarps][32 * ITEMS > 256 ? 256 : 32 * ITEMS];
  __shared__ int hist[32 * ITEMS];
  __shared__ int tok;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *w.state = 0;
  const int b0 = blockIdx.x * chunk, b1 = min(b0 + chunk, a.t);
  for (int q = seq_of(a.cu, a.s, b0, lane); q < a.s; ++q) {
    int qa, qb;
    seq_bounds(a.cu, q, a.t, qa, qb);
    if (qa >= b1) break;
    const int s0 = max(qa, b0), s1 = min(qb, b1);
    if (s0 >= s1) continue;                                  // block-uniform
    for (int i = threadIdx.x; i < a.e; i += blockDim.x) hist[i] = 0;
    if (threadIdx.x == 0) tok = 0;
    __syncthreads();
    float acc[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) acc[j] = 0.f;
    int mine = 0;
    float next[ITEMS];                                       // the next token's logits are on their way
    int id_next = -1;
    if (s0 + warp < s1) {
      load_logits<ITEMS, VEC>(a.logits + (int64_t)(s0 + warp) * a.e, a.e, lane, next);
      if (lane < a.k) id_next = __ldg(a.idx + (int64_t)(s0 + warp) * a.k + lane);
    }
    for (int t = s0 + warp; t < s1; t += kBalWarps) {
      const int id = id_next;
      float x[ITEMS], s[ITEMS];
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) x[j] = next[j];
      if (t + kBalWarps < s1) {
        load_logits<ITEMS, VEC>(a.logits + (int64_t)(t + kBalWarps) * a.e, a.e, lane, next);
        if (lane < a.k) id_next = __ldg(a.idx + (int64_t)(t + kBalWarps) * a.k + lane);
      }
      const bool hit = id >= 0 && id < a.e;
      if (!__any_sync(0xffffffffu, hit)) continue;           // padding
      if (hit) atomicAdd(&hist[id], 1);
      ++mine;
      const float inv = scores<ITEMS>(x, a.scoring, s);
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) acc[j] += s[j] * inv;
    }
    if (lane == 0) atomicAdd(&tok, mine);
    const int64_t slot = (int64_t)blockIdx.x + q;
    // 8 experts' columns (256 experts) at a time through shared memory
#pragma unroll
    for (int j0 = 0; j0 < ITEMS; j0 += 8) {
      __syncthreads();
#pragma unroll
      for (int j = j0; j < j0 + 8 && j < ITEMS; ++j) psum[warp][expert_of<VEC>(lane, j - j0)] = acc[j];
      __syncthreads();
      const int i = threadIdx.x, e = 32 * j0 + i;
      if (i < 32 * ITEMS && e < a.e) {
        float t = 0.f;
#pragma unroll
        for (int v = 0; v < kBalWarps; ++v) t += psum[v][i];
        w.p[slot * a.e + e] = t;
        w.c[slot * a.e + e] = hist[e];
      }
    }
    if (threadIdx.x == 0) w.t[slot] = tok;
    __syncthreads();                                         // hist, tok and psum are reused
  }
}

__global__ void __launch_bounds__(256) balance_reduce_kernel(BalanceArgs a, BalanceWs w, int chunk) {
  __shared__ double rp[8][32];
  __shared__ int rc[8][32];
  __shared__ int rt[8];
  __shared__ int last;
  pdl_wait();
  pdl_trigger();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int groups = gridDim.x, g = blockIdx.x;
  const int q = blockIdx.y;
  const int e = 32 * g + tx;
  int qa, qb;
  seq_bounds(a.cu, q, a.t, qa, qb);
  // a decreasing or out-of-range boundary: a NaN loss, no tokens and no counts anywhere (see the last block below)
  bool bad = false;
  if (a.cu != nullptr) {
    const int c0 = __ldg(a.cu + q), c1 = __ldg(a.cu + q + 1);
    bad = c0 < 0 || c1 < c0 || c1 > a.t;
  }
  const int blo = qa / chunk, bhi = qb > qa ? (qb - 1) / chunk + 1 : blo;
  double p = 0.0;
  int c = 0, n = 0;
  if (!bad) {
    if (e < a.e)
#pragma unroll 4
      for (int b = blo + ty; b < bhi; b += 8) {
        const int64_t slot = (int64_t)b + q;
        p += (double)w.p[slot * a.e + e];
        c += w.c[slot * a.e + e];
      }
    for (int b = blo + (int)threadIdx.x; b < bhi; b += 256) n += w.t[(int64_t)b + q];
  }
  rp[ty][tx] = p;
  rc[ty][tx] = c;
  n = __reduce_add_sync(0xffffffffu, n);
  if (tx == 0) rt[ty] = n;
  __syncthreads();
  if (ty == 0) {
    int tq = 0;
    for (int i = 0; i < 8; ++i) tq += rt[i];
    for (int i = 1; i < 8; ++i) {
      p += rp[i][tx];
      c += rc[i][tx];
    }
    double term = 0.0;
    if (e < a.e) {
      const double mean = tq > 0 ? p / tq : 0.0;
      a.mean_scores[(int64_t)q * a.e + e] = bad ? NAN : (float)mean;
      a.counts[(int64_t)q * a.e + e] = c;
      if (tq > 0) term = mean * ((double)c * a.e / ((double)a.k * tq));
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) term += __shfl_xor_sync(0xffffffffu, term, d);
    __syncwarp();                                            // the warp's outputs come before lane 0's fence
    if (tx == 0) {
      w.loss[(int64_t)q * groups + g] = bad ? (double)NAN : term;
      if (g == 0) a.tokens[q] = bad ? -1 : tq;
      __threadfence();
      last = atomicAdd(w.state, 1) == (int)(gridDim.x * gridDim.y) - 1;
    }
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double l = 0.0;                                            // fixed order: strided sums, then two trees
  int live = 0, wrong = 0;
  const int64_t parts = (int64_t)a.s * groups;
  for (int64_t i = threadIdx.x; i < parts; i += 256) l += __ldcg(w.loss + i);
  for (int i = threadIdx.x; i < a.s; i += 256) {
    const int n_i = __ldcg(a.tokens + i);
    live += n_i > 0;
    wrong |= n_i < 0;
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  live = __reduce_add_sync(0xffffffffu, live);
  const bool any_wrong = __syncthreads_or(wrong);
  if (tx == 0) {
    rp[0][ty] = l;
    rt[ty] = live;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) {
      l += rp[0][i];
      live += rt[i];
    }
    *a.loss = (float)(live > 0 ? (double)a.alpha * l / live : l);   // l is 0 (or NaN) without sequences
    *a.live = any_wrong ? -1 : live;
  }
  // One wrong boundary leaves the tokens of others unassigned too (the search for a block's first sequence expects
  // them in order), so no sequence of the call has counts.
  if (any_wrong) {
    for (int64_t i = threadIdx.x; i < (int64_t)a.s * a.e; i += 256) {
      a.counts[i] = 0;
      a.mean_scores[i] = NAN;
    }
    for (int i = threadIdx.x; i < a.s; i += 256) a.tokens[i] = -1;
  }
}

// t = 0: no tokens anywhere, and every boundary has to be 0.
__global__ void balance_empty_kernel(BalanceArgs a) {
  bool wrong = false;
  if (a.cu != nullptr)
    for (int i = threadIdx.x; i <= a.s; i += blockDim.x) wrong |= a.cu[i] != 0;
  wrong = __syncthreads_or(wrong);
  for (int64_t i = threadIdx.x; i < (int64_t)a.s * a.e; i += blockDim.x) {
    a.counts[i] = 0;
    a.mean_scores[i] = wrong ? NAN : 0.f;
  }
  for (int i = threadIdx.x; i < a.s; i += blockDim.x) a.tokens[i] = wrong ? -1 : 0;
  if (threadIdx.x == 0) {
    *a.loss = wrong ? NAN : 0.f;
    *a.live = wrong ? -1 : 0;
  }
}

// A block takes `chunk` consecutive tokens, a warp every eighth of them; the
// coefficients c_e of the sequence at hand are in the warp's registers.
template <int ITEMS, bool VEC>
__global__ void __launch_bounds__(kBalWarps * 32, ITEMS <= 8 ? 4 : 1) balance_grad_kernel(BalanceGradArgs a, int chunk) {
  __shared__ alignas(16) float scatter[kBalWarps][32 * ITEMS];           // a warp's row of combine-weight gradients, else zero
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) scatter[warp][lane + 32 * j] = 0.f;
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const int b1 = (int)min((int64_t)(blockIdx.x + 1) * chunk, (int64_t)a.t);
  const bool with_loss = a.counts != nullptr;
  const float g = a.grad_loss != nullptr ? __ldg(a.grad_loss) : 1.f;
  const int live = with_loss ? __ldg(a.live) : 0;
  for (int pos = blockIdx.x * chunk; pos < b1;) {
    int end = b1;
    float next[ITEMS];                                       // the next token's logits are on their way
    int id_next = -1;
    if (pos + warp < b1) {
      load_logits<ITEMS, VEC>(a.logits + (int64_t)(pos + warp) * a.e, a.e, lane, next);
      if (lane < a.k) id_next = __ldg(a.idx + (int64_t)(pos + warp) * a.k + lane);
    }
    // c_e less the first expert's: p adds up to 1 (sigmoid: 1 - 1e-20 / (sum + 1e-20)), so c_e - sum_j c_j p_j does not
    // see what all experts have in common but for that share, and balanced counts leave no remainder of rounding
    float coef[ITEMS], common = 0.f;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) coef[j] = live < 0 ? NAN : 0.f;        // wrong boundaries: no gradient either
    if (with_loss && live >= 0) {
      const int q = seq_of(a.cu, a.s, pos, lane);
      int qa, qb;
      seq_bounds(a.cu, q, a.t, qa, qb);
      if (pos < qa) {
        end = min(qa, b1);                                   // before the first sequence
      } else if (pos < qb) {
        end = min(qb, b1);
        const int tq = __ldg(a.tokens + q);
        const double f = tq > 0 && live > 0 ? (double)g * a.alpha * a.e / ((double)a.k * live * tq * tq) : 0.0;
        const int32_t* count = a.counts + (int64_t)q * a.e;
        const int first = __ldg(count);
        common = a.scoring == 0 ? (float)(f * first) * kScoreEps : 0.f;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
          if (VEC || lane + 32 * j < a.e) coef[j] = (float)(f * (__ldg(count + expert_of<VEC>(lane, j)) - first));
      }                                                      // else: behind the last sequence
    }
    for (int t = pos + warp; t < end; t += kBalWarps) {
      const int id = id_next;
      float x[ITEMS], dx[ITEMS];
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) x[j] = next[j];
      if (t + kBalWarps < end) {
        load_logits<ITEMS, VEC>(a.logits + (int64_t)(t + kBalWarps) * a.e, a.e, lane, next);
        if (lane < a.k) id_next = __ldg(a.idx + (int64_t)(t + kBalWarps) * a.k + lane);
      }
      const bool hit = id >= 0 && id < a.e;
      const bool token = __any_sync(0xffffffffu, hit);
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) dx[j] = 0.f;
      if (token && with_loss) {
        // s and its slope (sigmoid: s (1 - s), from one exponential; softmax: s)
        float s[ITEMS], slope[ITEMS], inv;
        if (a.scoring == 0) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < ITEMS; ++j) {
            const float e = __expf(-fabsf(x[j])), r = __fdividef(1.0f, 1.0f + e);
            s[j] = x[j] >= 0.f ? r : e * r;                  // NaN: e is NaN
            slope[j] = e * r * r;
            sum += s[j];
          }
          inv = 1.0f / (warp_sum(sum) + kScoreEps);
        } else {
          inv = scores<ITEMS>(x, 1, s);
#pragma unroll
          for (int j = 0; j < ITEMS; ++j) slope[j] = s[j];
        }
        float inner = 0.f;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) inner += coef[j] * s[j];
        inner = (warp_sum(inner) - common) * inv;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) dx[j] = (coef[j] - inner) * inv * slope[j];
      }
      if (token && a.grad_weights != nullptr) {
        const float xs = hit ? __ldg(a.logits + (int64_t)t * a.e + id) : 0.f;
        const float e = __expf(-fabsf(xs)), r = __fdividef(1.0f, 1.0f + e);
        const float top = hit ? (xs >= 0.f ? r : e * r) : 0.f;
        const float dw = hit ? __ldg(a.grad_weights + (int64_t)t * a.k + lane) : 0.f;
        const float share = 1.0f / (warp_sum(top) + kScoreEps);
        // dw_k - sum_j dw_j s_j / S from the first pick's dw on (the shares s_j / S add up to 1 - 1e-20 / S): what all picks
        // have in common cancels exactly, all of it with one pick, whose weight does not depend on its logit
        const float c = __shfl_sync(0xffffffffu, dw, __ffs(__ballot_sync(0xffffffffu, hit)) - 1);
        const float dot = warp_sum(hit ? (dw - c) * top : 0.f);
        const float d = hit ? ((dw - c) + (c * kScoreEps - dot) * share) * share * (e * r * r) * a.route_scale : 0.f;
        // scattered through shared memory; repeated picks (rare) are added by their first lane in pick order
        const uint32_t same = __match_any_sync(0xffffffffu, hit ? id : -1 - lane);
        float sum = d;
        if (__any_sync(0xffffffffu, same & (same - 1))) {
          sum = 0.f;
          for (int i = 0; i < a.k; ++i) {
            const float v = __shfl_sync(0xffffffffu, d, i);
            if (same >> i & 1) sum += v;
          }
        }
        const bool first = hit && (same & ((1u << lane) - 1)) == 0;
        if (first) scatter[warp][id] = sum;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) dx[j] += scatter[warp][expert_of<VEC>(lane, j)];
        __syncwarp();
        if (first) scatter[warp][id] = 0.f;
        __syncwarp();                                        // the warp's next token may pick it in another lane
      }
      float* out = a.grad_logits + (int64_t)t * a.e;
      if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < ITEMS; j += 4)
          reinterpret_cast<float4*>(out + 32 * j)[lane] = make_float4(dx[j], dx[j + 1], dx[j + 2], dx[j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
          if (lane + 32 * j < a.e) out[lane + 32 * j] = dx[j];
      }
    }
    pos = end;
  }
}

cudaError_t launch_balance(const BalanceArgs& a, cudaStream_t st) {
  if (a.t == 0) {
    balance_empty_kernel<<<1, 256, 0, st>>>(a);
    return cudaGetLastError();
  }
  BalanceWs w;
  balance_ws(a.t, a.e, a.s, static_cast<uint8_t*>(a.workspace), &w);
  const int chunk = balance_chunk(a.t), grid = ceil_div(a.t, chunk);
  const bool vec = a.e % 128 == 0 && (a.e & (a.e - 1)) == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
  const dim3 block(kBalWarps * 32);
  cudaError_t e;
#define MOE_BAL(I, V) e = launch_kernel(balance_partial_kernel<I, V>, dim3(grid), block, 0, st, true, a, w, chunk)
  if (a.e <= 32) MOE_BAL(1, false);
  else if (a.e <= 64) MOE_BAL(2, false);
  else if (a.e <= 128) { if (vec) MOE_BAL(4, true); else MOE_BAL(4, false); }
  else if (a.e <= 256) { if (vec) MOE_BAL(8, true); else MOE_BAL(8, false); }
  else if (a.e <= 512) { if (vec) MOE_BAL(16, true); else MOE_BAL(16, false); }
  else { if (vec) MOE_BAL(32, true); else MOE_BAL(32, false); }
#undef MOE_BAL
  if (e != cudaSuccess) return e;
  return launch_kernel(balance_reduce_kernel, dim3((unsigned)ceil_div(a.e, 32), (unsigned)a.s), dim3(256), 0, st, true, a,
                       w, chunk);
}

cudaError_t launch_balance_grad(const BalanceGradArgs& a, cudaStream_t st) {
  if (a.t == 0) return cudaSuccess;
  int chunk = align_up(ceil_div(a.t, 4 * 148), kBalWarps);     // about four blocks per SM
  if (chunk < kBalWarps) chunk = kBalWarps;
  const int grid = ceil_div(a.t, chunk);
  const bool vec = a.e % 128 == 0 && (a.e & (a.e - 1)) == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.grad_logits) % 16 == 0;
  const dim3 block(kBalWarps * 32);
#define MOE_BALG(I, V) return launch_kernel(balance_grad_kernel<I, V>, dim3(grid), block, 0, st, true, a, chunk)
  if (a.e <= 32) MOE_BALG(1, false);
  if (a.e <= 64) MOE_BALG(2, false);
  if (a.e <= 128) { if (vec) MOE_BALG(4, true); MOE_BALG(4, false); }
  if (a.e <= 256) { if (vec) MOE_BALG(8, true); MOE_BALG(8, false); }
  if (a.e <= 512) { if (vec) MOE_BALG(16, true); MOE_BALG(16, false); }
  if (vec) MOE_BALG(32, true);
  MOE_BALG(32, false);
#undef MOE_BALG
}

}  // namespace moe
