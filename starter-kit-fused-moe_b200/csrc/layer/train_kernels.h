// Launchers of the kernels around the routed experts: dense products, 8-bit
// activation checkpoints, gradients, and the router's balance loss.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace moe {

// activation codes (MOE_ACT_* of moe_fp8.h)
constexpr int kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActSwiglu = 4;

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Epilogue of a dense product z = x W^T: y = act(z + b) + r, optionally with the
// pre-activation kept in 8 bits. O = n / 2 for SwiGLU, n otherwise.
struct LinearEpilogue {
  const void* bias;        // bf16 [n] or NULL
  const void* residual;    // bf16 [m, O] or NULL, row stride ldr
  void* y;                 // bf16 / f32 [m, O], row stride ldy
  uint8_t* z8;             // e4m3 [m, n] ([2, m, O] for SwiGLU) or NULL
  uint8_t* z_scale;        // e8m0 [ceil(n / 128), m] ([2, ceil(O / 128), m])
  int64_t ldr, ldy;
  int act;
  int y_f32;
};

// Every kernel here is launched with programmatic stream serialization: its
// blocks may become resident while the preceding kernel of the stream ends, and
// wait for that kernel's completion before they touch global memory.
//
// Kernels of one call that do not need each other's results run side by side:
// one launched `early` does not wait at its start but before it exits. It starts
// when every block of its predecessor has run launch_dependents, which blocks do
// after their own wait (or, early ones, at once), so whatever that wait stood for
// is complete; and as no block leaves before its predecessor has completed, a
// later kernel's wait covers the whole chain. An early kernel reads what other
// kernels wrote through L2 only (TMA, ld.cg): it has not run the wait that would
// order its L1.
cudaError_t launch_checkpoint(const void* x, bool bf16, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q,
                              uint8_t* scale, cudaStream_t st);
cudaError_t launch_restore(const uint8_t* q, const uint8_t* scale, int64_t batch, int64_t rows, int64_t cols, void* out,
                           bool f32, cudaStream_t st);
// To bf16 rows of stride ldo (out 16-byte aligned, ldo a multiple of 8, what lies between cols and ldo is overwritten).
cudaError_t launch_restore_rows(const uint8_t* q, const uint8_t* scale, int64_t rows, int64_t cols, void* out, int64_t ldo,
                                bool early, cudaStream_t st);

// Products of few tokens without a kept pre-activation run on linear_small.cu,
// the others on linear_tile.cu. Up to 16 tokens the small kernel wins
// (16 tokens: 5.2 against 9 us at K, N = 7168, 256; 10.9 against 12.5 at 2048, 7168;
// 17.5 against 16 at 7168, 4096 gated, the one size tried where it does not); beyond, it loads the tokens' values too
// often unless the weights are small (32 tokens: 7.9 against 9.1, 37 against 16, 19.3 against 11.3).
constexpr bool small_product(int64_t m, int64_t k, int64_t n) { return m <= 16 || (m <= 32 && k * n <= 1 << 22); }
cudaError_t launch_linear_small(const void* x, int64_t ldx, const void* w, int64_t ldw, int m, int k, int n,
                                const LinearEpilogue& ep, cudaStream_t st);

// Gradient of the pre-activation: dz = dy * act'(z), written as bf16 [terms][m][ldz]
// (terms = 3: the roundings' remainders follow), and per-chunk column sums.
struct ActGradArgs {
  const void* dy;          // bf16 / f32 [m, O], row stride ldg
  const uint8_t* z8;       // as LinearEpilogue; NULL when act is none
  const uint8_t* z_scale;
  void* dz;                // NULL: column sums only
  float* colsum;           // [chunks, n] or NULL
  int64_t ldg, ldz;
  int m, n, act, dy_f32, terms;
};
int act_grad_chunks(int m, int n);
cudaError_t launch_act_grad(const ActGradArgs& a, cudaStream_t st);
cudaError_t launch_colsum_finish(const float* colsum, int chunks, int n, void* out, bool f32, bool early, cudaStream_t st);

struct BalanceArgs {
  const float* logits;     // [t, e]
  const int32_t* idx;      // [t, k]
  const int32_t* cu;       // [s + 1] or NULL (one sequence)
  int t, e, k, s, scoring; // scoring 0 sigmoid, 1 softmax
  float alpha;
  float* loss; int32_t* counts; int32_t* tokens; float* mean_scores; int32_t* live;
  void* workspace;
};
size_t balance_workspace_bytes(int t, int e, int s);
cudaError_t launch_balance(const BalanceArgs& a, cudaStream_t st);

struct BalanceGradArgs {
  const float* logits; const int32_t* idx; const int32_t* cu;
  int t, e, k, s, scoring;
  float alpha, route_scale;
  const int32_t* counts; const int32_t* tokens; const int32_t* live;
  const float* grad_loss;      // device scalar or NULL (1); counts NULL: no balance part
  const float* grad_weights;   // [t, k] or NULL
  float* grad_logits;          // [t, e]
};
cudaError_t launch_balance_grad(const BalanceGradArgs& a, cudaStream_t st);

}  // namespace moe
