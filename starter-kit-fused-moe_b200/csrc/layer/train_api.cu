// C-ABI layer of the dense products, 8-bit activation checkpoints, gradients
// and the balance loss: argument checks, workspace carving, launches. Nothing
// here allocates, synchronises or keeps state between calls.
#include <cstdio>

#include "moe_fp8.h"
#include "linear_tile.h"
#include "moe_kernels.h"
#include "train_kernels.h"

namespace {

int bad(const char* msg) {
  moe::set_last_error(msg);
  return MOE_ERR_INVALID_ARGUMENT;
}
int workspace_error(const char* what, size_t need, size_t got) {
  char buf[160];
  snprintf(buf, sizeof(buf), "%s: workspace missing, misaligned or too small (need %zu bytes, got %zu)", what, need, got);
  moe::set_last_error(buf);
  return MOE_ERR_WORKSPACE;
}
int done(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return MOE_OK;
  char buf[160];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
  moe::set_last_error(buf);
  return MOE_ERR_CUDA;
}
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
int64_t up8(int64_t x) { return (x + 7) & ~int64_t(7); }

constexpr int64_t kMaxDim = 1 << 30, kMaxWidth = 1 << 23;

int check_sizes(int64_t m, int64_t k, int64_t n, int act) {
  if (m < 0 || k < 1 || n < 1 || m > kMaxDim || k > kMaxWidth || n > kMaxWidth)
    return bad("m must be in [0, 2^30], k and n in [1, 2^23]");
  if (act < MOE_ACT_NONE || act > MOE_ACT_SWIGLU) return bad("unknown activation");
  if (act == MOE_ACT_SWIGLU && n % 2) return bad("SwiGLU needs an even n");
  return MOE_OK;
}

int pairs() {
  const int n = moe::current_device_sms();
  return n >= 2 ? n / 2 : 74;
}
// TMA reads a matrix in place if its base and row stride are multiples of 16 bytes.
bool tma_ready(const void* p, int64_t ld) { return aligned(p, 16) && ld % 8 == 0; }

// One tensor-core product: its tile plan and the workspace of its K slices.
struct Product {
  moe::LinearTilePlan plan;
  bool vec;
  int64_t term_blocks;
  int terms;
  size_t partial;      // bytes
};
// Whether 16-byte accesses reach every row of y, the residual and the kept z.
bool vec_rows(const moe::LinearEpilogue& ep, int64_t out_cols) {
  return aligned(ep.y, 16) && ep.ldy * (ep.y_f32 ? 4 : 2) % 16 == 0 &&
         (!ep.residual || (aligned(ep.residual, 16) && ep.ldr % 8 == 0 && ep.ldr > 0)) &&
         (!ep.z8 || (aligned(ep.z8, 16) && out_cols % 16 == 0));
}
Product plan_product(int64_t m, int64_t out_cols, int64_t k, int terms, bool gated, const moe::LinearEpilogue& ep, bool grad) {
  Product p{};
  p.vec = vec_rows(ep, out_cols);
  p.term_blocks = (k + 63) / 64;
  p.terms = terms;
  p.plan = moe::plan_linear_tile(m, out_cols, p.term_blocks * terms, gated, grad, p.vec, ep, pairs());
  p.partial = (size_t)p.plan.tail * p.plan.splits * 256 * p.plan.n_tile * sizeof(float);
  return p;
}
// A: [terms][rows][..], term stride in elements. `t` is left for the join.
int run_product(const Product& p, bool a_mn, bool b_mn, bool gated, bool keep, int64_t m, int64_t out_cols, int64_t k,
                const void* A, int64_t lda, int64_t term_stride, const void* B, int64_t ldb, int64_t b_rows,
                const moe::LinearEpilogue& ep, uint8_t* partial, bool early, cudaStream_t st, const char* what,
                moe::LinearTileArgs& t) {
  t = {};
  t.early = early;
  t.m = m;
  t.out_cols = out_cols;
  t.gate_rows = gated ? (int)out_cols : 0;
  t.n_tile = p.plan.n_tile;
  t.flip = p.plan.flip;
  t.tile_rows = t.flip ? t.n_tile : 256;
  const int width = t.flip ? 256 : t.n_tile, cols = gated ? width / 2 : width;
  t.m_tiles = moe::ceil_div(m, t.tile_rows);
  t.n_tiles = moe::ceil_div(out_cols, cols);
  t.term_blocks = (int)p.term_blocks;
  t.terms = p.terms;
  t.k_blocks = t.term_blocks * p.terms;
  t.splits = p.plan.splits;
  t.chain = moe::linear_chain(gated, ep.y_f32, keep, t.k_blocks);
  t.full_tiles = p.plan.full;
  t.units = p.plan.full + p.plan.tail * t.splits;
  t.ep = ep;
  t.vec = p.vec;
  t.partial = reinterpret_cast<float*>(partial);
  moe::LinearTileMaps maps{};
  const uint32_t half = (uint32_t)t.n_tile / 2;
  bool ok;
  if (t.flip)      // the weights' rows are the tile's, the tokens its columns
    ok = moe::encode_bf16(&maps.a, B, k, b_rows, ldb, 1, b_rows * ldb, 64, 128) &&
         moe::encode_bf16(&maps.b, A, k, m, lda, 0, 0, 64, half);
  else
    ok = (a_mn ? moe::encode_bf16(&maps.a, A, m, k, lda, p.terms, term_stride, 64, 64)
               : moe::encode_bf16(&maps.a, A, k, m, lda, p.terms, term_stride, 64, 128)) &&
         (b_mn ? moe::encode_bf16(&maps.b, B, out_cols, k, ldb, 0, 0, 64, 64)
               : moe::encode_bf16(&maps.b, B, k, b_rows, ldb, 0, 0, 64, half));
  if (t.vec && !ep.y_f32 && t.full_tiles > 0) {
    ok = ok && moe::encode_bf16(&maps.out, ep.y, out_cols, m, ep.ldy, 0, 0, 32, 32);
    if (ep.residual) ok = ok && moe::encode_bf16(&maps.res, ep.residual, out_cols, m, ep.ldr, 0, 0, 32, 32);
  }
  if (!ok) {
    moe::set_last_error("cuTensorMapEncodeTiled failed");
    return MOE_ERR_CUDA;
  }
  return done(moe::launch_linear_tile(a_mn, b_mn, gated, keep, maps, t, 2 * pairs(), st), what);
}

// Workspace of a forward product.
struct LinearPlan {
  Product prod;
  bool small, pad_x, pad_w;
  int64_t ldp;
  size_t x, w, total;
};
moe::LinearEpilogue epilogue_of(const MoeLinearArgs& a) {
  return {a.bias, a.residual, a.y, static_cast<uint8_t*>(a.z8), static_cast<uint8_t*>(a.z_scale),
          a.ldr, a.ldy, a.activation, a.y_f32};
}
moe::LinearEpilogue plain_epilogue(void* y, int64_t ldy, int f32) {
  return {nullptr, nullptr, y, nullptr, nullptr, 0, ldy, MOE_ACT_NONE, f32};
}
LinearPlan linear_plan(const MoeLinearArgs& a) {
  LinearPlan p{};
  p.small = a.z8 == nullptr && moe::small_product(a.m, a.k, a.n);
  if (p.small) return p;
  const bool gated = a.activation == MOE_ACT_SWIGLU;
  p.prod = plan_product(a.m, gated ? a.n / 2 : a.n, a.k, 1, gated, epilogue_of(a), false);
  p.pad_x = !tma_ready(a.x, a.ldx);
  p.pad_w = !tma_ready(a.weight, a.ldw);
  p.ldp = up8(a.k);
  size_t o = up256(p.prod.partial);
  p.x = o;
  if (p.pad_x) o += up256((size_t)a.m * p.ldp * 2);
  p.w = o;
  if (p.pad_w) o += up256((size_t)a.n * p.ldp * 2);
  p.total = o;
  return p;
}

// Workspace of the gradient entry: the products' K-slice partials, dz, x^, the padded weights, column sums.
struct GradPlan {
  bool need_dz, direct, pad_w;
  int terms, chunks;
  int64_t ldz, ldk;
  Product px, pw;
  size_t part_w, dz, xhat, w, colsum, total;      // the input gradient's partials come first
};
GradPlan grad_plan(const MoeLinearGradArgs& a) {
  GradPlan p{};
  p.ldz = up8(a.n);
  p.ldk = up8(a.k);
  p.terms = a.grad_f32 && (a.activation != MOE_ACT_NONE || a.grad_y_f32) ? 3 : 1;
  // without an activation bf16 gradients are dz themselves
  p.direct = a.activation == MOE_ACT_NONE && !a.grad_y_f32 && tma_ready(a.grad_y, a.ldg) && a.ldg >= a.n;
  p.need_dz = (a.grad_x || a.grad_weight) && !p.direct;
  p.chunks = moe::act_grad_chunks(a.m, a.n);
  size_t o = 0;
  if (a.grad_x) {
    p.px = plan_product(a.m, a.k, a.n, p.terms, false, plain_epilogue(a.grad_x, a.k, a.grad_f32), true);
    o = up256(p.px.partial);
    p.pad_w = !tma_ready(a.weight, a.ldw);
  }
  p.part_w = o;
  if (a.grad_weight) {
    p.pw = plan_product(a.n, a.k, a.m, p.terms, false, plain_epilogue(a.grad_weight, a.k, a.grad_f32), true);
    o += up256(p.pw.partial);
  }
  p.dz = o;
  if (p.need_dz) o += up256((size_t)a.m * p.ldz * 2 * p.terms);
  p.xhat = o;
  if (a.grad_weight) o += up256((size_t)a.m * p.ldk * 2);
  p.w = o;
  if (p.pad_w) o += up256((size_t)a.n * p.ldk * 2);
  p.colsum = o;
  if (a.grad_bias) o += up256((size_t)p.chunks * a.n * 4);
  p.total = o;
  return p;
}

}  // namespace

extern "C" {

size_t moe_linear_workspace_bytes(const MoeLinearArgs* a) {
  if (!a || a->m <= 0 || a->n <= 0 || a->k <= 0) return 0;
  return linear_plan(*a).total;
}

int moe_linear_run(const MoeLinearArgs* a, void* stream) {
  if (!a) return bad("args is NULL");
  if (int rc = check_sizes(a->m, a->k, a->n, a->activation)) return rc;
  if (a->m == 0) return MOE_OK;
  const int64_t O = a->activation == MOE_ACT_SWIGLU ? a->n / 2 : a->n;
  if (!a->x || !a->weight || !a->y) return bad("linear: x, weight and y must not be NULL");
  if ((a->z8 == nullptr) != (a->z_scale == nullptr)) return bad("linear: z8 and z_scale go together");
  if (!aligned(a->x, 2) || !aligned(a->weight, 2) || !aligned(a->bias, 2) || !aligned(a->residual, 2) ||
      !aligned(a->y, a->y_f32 ? 4 : 2))
    return bad("linear: a pointer is not aligned to its type");
  if (a->ldx < a->k || a->ldw < a->k || a->ldy < O || (a->residual && a->ldr < 0))
    return bad("linear: a row stride is smaller than the row");
  if (a->residual == a->y && (a->y_f32 || a->ldr != a->ldy))
    return bad("linear: y may be the residual itself only as bf16 and with its row stride");
  const LinearPlan p = linear_plan(*a);
  if (p.total && (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < p.total))
    return workspace_error("linear", p.total, a->workspace_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  const moe::LinearEpilogue ep = epilogue_of(*a);
  if (p.small) return done(moe::launch_linear_small(a->x, a->ldx, a->weight, a->ldw, a->m, a->k, a->n, ep, st), "linear product");
  moe::PadArgs pads{};
  if (p.pad_x) pads.add(a->x, a->ldx, a->m, a->k, ws + p.x, p.ldp);
  if (p.pad_w) pads.add(a->weight, a->ldw, a->n, a->k, ws + p.w, p.ldp);
  cudaError_t e = moe::launch_pad(pads, st);
  if (e != cudaSuccess) return done(e, "linear: preparing the operands");
  const void* x = p.pad_x ? ws + p.x : a->x;
  const void* w = p.pad_w ? ws + p.w : a->weight;
  const int64_t ldx = p.pad_x ? p.ldp : a->ldx;
  const bool gated = a->activation == MOE_ACT_SWIGLU, keep = a->z8 != nullptr;
  moe::LinearTileArgs t;
  if (int rc = run_product(p.prod, false, false, gated, keep, a->m, O, a->k, x, ldx, a->m * ldx, w,
                           p.pad_w ? p.ldp : a->ldw, a->n, ep, ws, false, st, "linear product", t))
    return rc;
  return done(moe::launch_linear_join(gated, keep, t, st), "linear product");
}

size_t moe_linear_grad_workspace_bytes(const MoeLinearGradArgs* a) {
  if (!a || a->m <= 0 || a->n <= 0 || a->k <= 0) return 0;
  return grad_plan(*a).total;
}

int moe_linear_grad(const MoeLinearGradArgs* a, void* stream) {
  if (!a) return bad("args is NULL");
  if (int rc = check_sizes(a->m, a->k, a->n, a->activation)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t gsize = a->grad_f32 ? 4 : 2;
  if (!aligned(a->grad_x, gsize) || !aligned(a->grad_weight, gsize) || !aligned(a->grad_bias, gsize))
    return bad("linear gradient: a pointer is not aligned to its type");
  if (a->m == 0) {           // sums over no tokens
    cudaError_t e = cudaSuccess;
    if (a->grad_weight) e = cudaMemsetAsync(a->grad_weight, 0, (size_t)a->n * a->k * gsize, st);
    if (e == cudaSuccess && a->grad_bias) e = cudaMemsetAsync(a->grad_bias, 0, (size_t)a->n * gsize, st);
    return done(e, "clearing the gradients");
  }
  if (!a->grad_x && !a->grad_weight && !a->grad_bias) return MOE_OK;
  const int64_t O = a->activation == MOE_ACT_SWIGLU ? a->n / 2 : a->n;
  const bool act = a->activation != MOE_ACT_NONE;
  if (!a->grad_y || (act && (!a->z8 || !a->z_scale)) || (a->grad_x && !a->weight) ||
      (a->grad_weight && (!a->x8 || !a->x_scale)))
    return bad("linear gradient: an input that the requested gradients need is NULL");
  if (!aligned(a->grad_y, a->grad_y_f32 ? 4 : 2) || !aligned(a->weight, 2))
    return bad("linear gradient: a pointer is not aligned to its type");
  if (a->ldg < 0 || (a->grad_x && a->ldw < a->k)) return bad("linear gradient: a row stride is smaller than the row");
  const GradPlan p = grad_plan(*a);
  if (p.total && (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < p.total))
    return workspace_error("linear gradient", p.total, a->workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  // Three steps: what the products need, the products, what finishes them. A step's kernels run side by side (the
  // first of them waits for the step before, see train_kernels.h).
  cudaError_t e = cudaSuccess;
  bool begun = false;
  if (p.need_dz || a->grad_bias) {
    moe::ActGradArgs g{};
    g.dy = a->grad_y;
    g.z8 = act ? static_cast<const uint8_t*>(a->z8) : nullptr;
    g.z_scale = static_cast<const uint8_t*>(a->z_scale);
    g.dz = p.need_dz ? ws + p.dz : nullptr;
    g.colsum = a->grad_bias ? reinterpret_cast<float*>(ws + p.colsum) : nullptr;
    g.ldg = a->ldg;
    g.ldz = p.ldz;
    g.m = a->m;
    g.n = a->n;
    g.act = a->activation;
    g.dy_f32 = a->grad_y_f32;
    g.terms = p.terms;
    e = moe::launch_act_grad(g, st);
    if (e != cudaSuccess) return done(e, "activation gradient");
    begun = true;
  }
  if (a->grad_weight) {
    e = moe::launch_restore_rows(static_cast<const uint8_t*>(a->x8), static_cast<const uint8_t*>(a->x_scale), a->m, a->k,
                                 ws + p.xhat, p.ldk, begun, st);
    if (e != cudaSuccess) return done(e, "restoring the input checkpoint");
    begun = true;
  }
  if (p.pad_w) {
    moe::PadArgs pads{};
    pads.early = begun;
    pads.add(a->weight, a->ldw, a->n, a->k, ws + p.w, p.ldk);
    e = moe::launch_pad(pads, st);
    if (e != cudaSuccess) return done(e, "linear gradient: preparing the operands");
  }
  const void* dz = p.direct ? a->grad_y : ws + p.dz;
  const int64_t ldz = p.direct ? a->ldg : p.ldz, term_stride = a->m * ldz;
  moe::LinearTileArgs tx{}, tw{};
  if (a->grad_x) {
    const void* w = p.pad_w ? ws + p.w : a->weight;
    const int64_t ldw = p.pad_w ? p.ldk : a->ldw;
    const moe::LinearEpilogue ep = plain_epilogue(a->grad_x, a->k, a->grad_f32);
    if (int rc = run_product(p.px, false, true, false, false, a->m, a->k, a->n, dz, ldz, term_stride, w, ldw, a->n, ep,
                             ws, false, st, "input gradient", tx))
      return rc;
  }
  if (a->grad_weight) {
    const moe::LinearEpilogue ep = plain_epilogue(a->grad_weight, a->k, a->grad_f32);
    if (int rc = run_product(p.pw, true, true, false, false, a->n, a->k, a->m, dz, ldz, term_stride, ws + p.xhat, p.ldk,
                             a->m, ep, ws + p.part_w, a->grad_x != nullptr, st, "weight gradient", tw))
      return rc;
  }
  if (a->grad_bias) {
    e = moe::launch_colsum_finish(reinterpret_cast<float*>(ws + p.colsum), p.chunks, a->n, a->grad_bias,
                                  a->grad_f32 != 0, a->grad_x || a->grad_weight, st);
    if (e != cudaSuccess) return done(e, "bias gradient");
  }
  if (a->grad_x && (e = moe::launch_linear_join(false, false, tx, st)) != cudaSuccess) return done(e, "input gradient");
  tw.join_early = a->grad_x && tx.units != tx.full_tiles;
  if (a->grad_weight && (e = moe::launch_linear_join(false, false, tw, st)) != cudaSuccess) return done(e, "weight gradient");
  return MOE_OK;
}

int moe_checkpoint_activations(const void* x, int32_t x_is_bf16, int64_t rows, int64_t cols, int64_t ldx, void* q,
                               void* scale, void* stream) {
  if (rows < 0 || cols < 0 || rows > kMaxDim || cols > (int64_t)65535 * 1024)
    return bad("checkpoint: rows must be in [0, 2^30], cols in [0, 65535 * 1024]");
  if (rows == 0 || cols == 0) return MOE_OK;
  if (!x || !q || !scale || !aligned(x, x_is_bf16 ? 2 : 4)) return bad("checkpoint: NULL or misaligned pointer");
  if (ldx < 0) return bad("checkpoint: negative row stride");
  return done(moe::launch_checkpoint(x, x_is_bf16 != 0, rows, cols, ldx, static_cast<uint8_t*>(q),
                                     static_cast<uint8_t*>(scale), static_cast<cudaStream_t>(stream)),
              "checkpoint");
}

int moe_restore_activations(const void* q, const void* scale, int64_t batch, int64_t rows, int64_t cols, void* out,
                            int32_t out_f32, void* stream) {
  if (batch < 0 || batch > 65535 || rows < 0 || cols < 0 || rows > kMaxDim || cols > (int64_t)65535 * 1024)
    return bad("restore: batch must be in [0, 65535], rows in [0, 2^30], cols in [0, 65535 * 1024]");
  if (batch == 0 || rows == 0 || cols == 0) return MOE_OK;
  if (!q || !scale || !out || !aligned(out, out_f32 ? 4 : 2)) return bad("restore: NULL or misaligned pointer");
  return done(moe::launch_restore(static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale), batch, rows, cols,
                                  out, out_f32 != 0, static_cast<cudaStream_t>(stream)),
              "restore");
}

static int check_balance(int t, int e, int k, int s, int scoring) {
  if (t < 0 || t > kMaxDim || e < 1 || e > 1024 || k < 1 || k > 32 || s < 1 || s > 65535)
    return bad("balance: need T in [0, 2^30], E in [1, 1024], k in [1, 32], S in [1, 65535]");
  if (scoring != 0 && scoring != 1) return bad("balance: scoring must be 0 (sigmoid) or 1 (softmax)");
  return MOE_OK;
}

size_t moe_balance_workspace_bytes(int32_t t, int32_t e, int32_t s) {
  if (t <= 0 || e < 1 || e > 1024 || s < 1 || s > 65535) return 0;
  return moe::balance_workspace_bytes(t, e, s);
}

int moe_balance_loss(const MoeBalanceArgs* a, void* stream) {
  if (!a) return bad("args is NULL");
  if (int rc = check_balance(a->num_tokens, a->num_experts, a->top_k, a->num_sequences, a->scoring)) return rc;
  if (!a->loss || !a->counts || !a->tokens || !a->mean_scores || !a->sequences) return bad("balance: an output is NULL");
  if (a->num_tokens > 0 && (!a->routing_logits || !a->topk_idx || !aligned(a->routing_logits, 4) || !aligned(a->topk_idx, 4)))
    return bad("balance: NULL or misaligned input");
  if (!aligned(a->cu_seqlens, 4) || !aligned(a->loss, 4) || !aligned(a->counts, 4) || !aligned(a->tokens, 4) ||
      !aligned(a->mean_scores, 4) || !aligned(a->sequences, 4))
    return bad("balance: a pointer is not aligned to its type");
  if (!a->cu_seqlens && a->num_sequences != 1) return bad("balance: one sequence without cu_seqlens");
  const size_t need = moe_balance_workspace_bytes(a->num_tokens, a->num_experts, a->num_sequences);
  if (need && (!a->workspace || !aligned(a->workspace, 256) || a->workspace_bytes < need))
    return workspace_error("balance", need, a->workspace_bytes);
  moe::BalanceArgs b{a->routing_logits, a->topk_idx, a->cu_seqlens, a->num_tokens, a->num_experts, a->top_k,
                     a->num_sequences, a->scoring, a->alpha, a->loss, a->counts, a->tokens, a->mean_scores,
                     a->sequences, a->workspace};
  return done(moe::launch_balance(b, static_cast<cudaStream_t>(stream)), "balance loss");
}

int moe_balance_loss_grad(const MoeBalanceGradArgs* a, void* stream) {
  if (!a) return bad("args is NULL");
  if (int rc = check_balance(a->num_tokens, a->num_experts, a->top_k, a->num_sequences, a->scoring)) return rc;
  if (a->num_tokens == 0) return MOE_OK;
  if (!a->routing_logits || !a->topk_idx || !a->grad_logits || !aligned(a->routing_logits, 4) ||
      !aligned(a->topk_idx, 4) || !aligned(a->grad_logits, 4) || !aligned(a->grad_topk_weights, 4) ||
      !aligned(a->cu_seqlens, 4) || !aligned(a->counts, 4) || !aligned(a->tokens, 4) || !aligned(a->sequences, 4) ||
      !aligned(a->grad_loss, 4))
    return bad("balance gradient: NULL or misaligned pointer");
  if ((a->grad_loss || a->counts || a->tokens || a->sequences) && (!a->counts || !a->tokens || !a->sequences))
    return bad("balance gradient: the loss's part needs counts, tokens and sequences");
  if (!a->cu_seqlens && a->num_sequences != 1) return bad("balance gradient: one sequence without cu_seqlens");
  moe::BalanceGradArgs b{a->routing_logits, a->topk_idx, a->cu_seqlens, a->num_tokens, a->num_experts, a->top_k,
                         a->num_sequences, a->scoring, a->alpha, a->routed_scaling_factor, a->counts, a->tokens,
                         a->sequences, a->grad_loss, a->grad_topk_weights, a->grad_logits};
  return done(moe::launch_balance_grad(b, static_cast<cudaStream_t>(stream)), "balance gradient");
}

}  // extern "C"
