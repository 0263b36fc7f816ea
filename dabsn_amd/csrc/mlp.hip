// The block's MLP as a whole, forward and backward, and one layer's backward: norm, products and sums of
// norm.hip and linear.hip one after the other, with what lies between them in the caller's workspace.
// One call from the host instead of three to nine, and one buffer for all that the backward needs,
// which is what small steps wait for (2048 x 256 x 1024 fp32, forward and backward: 235 us with a
// call and a tensor each, 180 to 188 so, of which 131 are kernels).
//
// Rounded to bf16 on the way, where the operands are bf16, is what the matrix cores read: the normed
// rows, h and dz. (Weights' gradients of the branch are 0.3% off in the norm by these, a single rounding
// of the result 0.17%.) Sums stay fp32, and so does dn, which only the norm's backward reads: rounded
// too it left dx 0.28% off and the norm's weight 0.33%, now 0.25% and 0.29%, for 1.1% of the time
// (65536 x 2048 x 8192). b1's gradient sums dz as the products have it, in a pass of its own (190 us
// there): dz before its rounding is in no memory. The roundings of the terms have independent signs and
// add up to 0.17% of the root of the terms' squares, which is the size of a sum of gradients of
// either sign, and as much as the result's own rounding.
#include "common.hpp"
#include "norm.hpp"

#include <algorithm>
#include <initializer_list>
#include <utility>

namespace dabsn {
namespace mlp {

static size_t up(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// Places in the workspace; with `base` not the workspace, a walk for the sizes alone.
struct Space {
  char* base;
  size_t at = 0;
  void* take(size_t bytes) {
    void* p = base + at;
    at += up(bytes);
    return p;
  }
};

static int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }

static dabsn_linear_call product(int dtype, int64_t M, int64_t N, int64_t K, const void* A, int64_t lda,
                                 const void* B, int64_t ldb, void* C, int64_t ldc) {
  dabsn_linear_call l = {};
  l.dtype = dtype;
  l.M = M; l.N = N; l.K = K;
  l.A = A; l.lda = lda;
  l.B = B; l.ldb = ldb;
  l.C = C; l.ldc = ldc;
  return l;
}
// The gradients of a layer's rows (without slope) and weight from those of its results.
static dabsn_linear_call rows_grad(int dtype, int64_t M, int64_t N, int64_t K, const void* dz, int64_t ldz,
                                   const void* w, int64_t ldw, void* dx, int64_t ldx) {
  dabsn_linear_call l = product(dtype, M, K, N, dz, ldz, w, ldw, dx, ldx);
  l.transB = 1;
  return l;
}
static dabsn_linear_call weight_grad(int dtype, int64_t M, int64_t N, int64_t K, const void* dz, int64_t ldz,
                                     const void* x, int64_t ldx, void* dw) {
  dabsn_linear_call l = product(dtype, N, K, M, dz, ldz, x, ldx, dw, K);
  l.transA = l.transB = 1;
  return l;
}

static int run(dabsn_linear_call l, void* scratch, size_t bytes, hipStream_t s) {
  l.workspace = scratch;
  l.workspace_bytes = bytes;
  return dabsn_hip_linear(&l, s);
}

// What the forward leaves for the backward.
struct Saved {
  float* stats;
  void *normed, *h, *keep;
  int64_t ldh;
};
static Saved saved(const dabsn_mlp_call& c, Space& s) {
  const size_t size = c.dtype == kF32 ? 4 : 2, M = static_cast<size_t>(c.M);
  Saved v = {};
  v.ldh = padded(c.F);
  v.stats = static_cast<float*>(s.take(M * 2 * sizeof(float)));
  v.normed = s.take(M * c.H * size);
  v.h = s.take(M * v.ldh * size);
  if (c.act > 1) v.keep = s.take(M * v.ldh * size);
  return v;
}

struct Forward {
  Saved v;
  dabsn_linear_call first, second;
  size_t scratch_at, scratch, total;
};
static Forward forward(const dabsn_mlp_call& c, char* base) {
  const size_t size = c.dtype == kF32 ? 4 : 2;
  Space s{base};
  Forward f = {};
  if (c.train) {
    Space kept{static_cast<char*>(c.saved)};
    f.v = saved(c, kept);
  } else {
    f.v.ldh = padded(c.F);
    f.v.normed = s.take(static_cast<size_t>(c.M) * c.H * size);
    f.v.h = s.take(static_cast<size_t>(c.M) * f.v.ldh * size);
  }
  f.first = product(c.dtype, c.M, c.F, c.H, f.v.normed, c.H, c.w1, c.ldw1, f.v.h, f.v.ldh);
  f.first.bias = c.b1;
  f.first.act = c.act;
  f.first.keep = f.v.keep; f.first.ldk = f.v.ldh;
  f.first.padC = 1;
  f.second = product(c.dtype, c.M, c.H, c.F, f.v.h, f.v.ldh, c.w2, c.ldw2, c.out, c.H);
  f.second.bias = c.b2;
  f.second.residual = c.x; f.second.ldr = c.ldx;
  f.second.padA = 1;
  f.scratch = std::max(dabsn_hip_linear_workspace_bytes(&f.first), dabsn_hip_linear_workspace_bytes(&f.second));
  f.scratch_at = s.at;
  f.total = s.at + f.scratch;
  return f;
}

struct Backward {
  Saved v;
  void *dz, *dx;
  void* dn;  // [M][ldn] in fp32
  int64_t ldn;
  dabsn_linear_call dz_call, dn_call, dw1_call, dw2_call;
  bool rows, inner;  // whether dz, and what lies before it, is asked for
  size_t scratch_at, scratch, total;
};
static Backward backward(const dabsn_mlp_call& c, char* base) {
  const size_t size = c.dtype == kF32 ? 4 : 2, M = static_cast<size_t>(c.M);
  Space s{base}, kept{static_cast<char*>(c.saved)};
  Backward b = {};
  b.v = saved(c, kept);
  const int64_t ldh = b.v.ldh;
  b.inner = c.dx || c.dnorm_weight || c.dnorm_bias;
  b.rows = b.inner || c.dw1 || c.db1;
  b.dz = b.rows ? s.take(M * ldh * size) : nullptr;
  b.ldn = c.dtype == kF32 ? c.H : padded(c.H);
  b.dn = b.inner ? s.take(M * b.ldn * sizeof(float)) : nullptr;
  b.dx = c.dx || !b.inner ? c.dx : s.take(M * c.H * size);
  const auto need = [&](const dabsn_linear_call& l) {
    b.scratch = std::max(b.scratch, dabsn_hip_linear_workspace_bytes(&l));
  };
  if (c.dw2) need(b.dw2_call = weight_grad(c.dtype, c.M, c.H, c.F, c.grad, c.H, b.v.h, ldh, c.dw2));
  if (b.rows) {
    b.dz_call = rows_grad(c.dtype, c.M, c.H, c.F, c.grad, c.H, c.w2, c.ldw2, b.dz, ldh);
    b.dz_call.padC = 1;
    if (c.act) {  // the squared ReLU's slope is its output's
      b.dz_call.slope = c.act == 1 ? b.v.h : b.v.keep;
      b.dz_call.slope_kind = c.act == 1 ? 2 : 1;
      b.dz_call.lds = ldh;
    }
    need(b.dz_call);
  }
  if (c.dw1) need(b.dw1_call = weight_grad(c.dtype, c.M, c.F, c.H, b.dz, ldh, b.v.normed, c.H, c.dw1));
  if (b.inner) {
    b.dn_call = rows_grad(c.dtype, c.M, c.F, c.H, b.dz, ldh, c.w1, c.ldw1, b.dn, b.ldn);
    b.dn_call.padA = 1;
    b.dn_call.wideC = c.dtype == kBF16;
    need(b.dn_call);
    b.scratch = std::max(b.scratch, dabsn_hip_norm_workspace_bytes(c.dtype, c.M, c.H));
  }
  if (c.db1) b.scratch = std::max(b.scratch, dabsn_hip_linear_slope_workspace_bytes(c.dtype, c.M, c.F));
  if (c.db2) b.scratch = std::max(b.scratch, dabsn_hip_linear_slope_workspace_bytes(c.dtype, c.M, c.H));
  b.scratch_at = s.at;
  b.total = s.at + b.scratch;
  return b;
}

// One layer's gradients.
struct Layer {
  void* dz;  // grad * slope, or NULL: grad itself
  int64_t ldz;
  dabsn_linear_call dx_call, dw_call;
  size_t scratch_at, scratch, total;
};
static Layer layer(const dabsn_linear_grads_call& c, char* base) {
  Space s{base};
  Layer l = {};
  if (c.slope && (c.dx || c.dw)) {
    l.ldz = padded(c.N);
    l.dz = s.take(static_cast<size_t>(c.M) * l.ldz * (c.dtype == kF32 ? 4 : 2));
  }
  const void* dz = c.slope ? l.dz : c.grad;
  const int64_t ldz = c.slope ? l.ldz : c.ldg;
  if (c.dx) {
    l.dx_call = rows_grad(c.dtype, c.M, c.N, c.K, dz, ldz, c.w, c.ldw, c.dx, c.K);
    l.dx_call.padA = c.slope != nullptr;
    l.scratch = std::max(l.scratch, dabsn_hip_linear_workspace_bytes(&l.dx_call));
  }
  if (c.dw) {
    l.dw_call = weight_grad(c.dtype, c.M, c.N, c.K, dz, ldz, c.x, c.ldx, c.dw);
    l.scratch = std::max(l.scratch, dabsn_hip_linear_workspace_bytes(&l.dw_call));
  }
  if (c.db) l.scratch = std::max(l.scratch, dabsn_hip_linear_slope_workspace_bytes(c.dtype, c.M, c.N));
  l.scratch_at = s.at;
  l.total = s.at + l.scratch;
  return l;
}

// The products' limits, so that nothing has been launched when one refuses its call.
constexpr int64_t WIDTH = 1 << 21, ROWS = (1ll << 31) - 65536;
static bool strides(std::initializer_list<std::pair<int64_t, int64_t>> of) {
  for (const auto& s : of)
    if (s.first < s.second || s.first >= WIDTH) return false;
  return true;
}
static bool fits(const void* workspace, size_t bytes, size_t need) {
  return need == 0 || (workspace && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
}
static char* anywhere() { return reinterpret_cast<char*>(static_cast<uintptr_t>(4096)); }

static int check(const dabsn_mlp_call& c) {
  DABSN_REQUIRE((c.dtype == kF32 || c.dtype == kBF16) && (c.wdtype == c.dtype || c.wdtype == kF32),
                "mlp: bad type %d, norm's weight %d", c.dtype, c.wdtype);
  DABSN_REQUIRE(c.M >= 0 && c.M < ROWS && c.H > 0 && c.H <= 16384 && c.F > 0 && c.F <= WIDTH - 8,
                "mlp: bad shape M=%lld H=%lld F=%lld", (long long)c.M, (long long)c.H, (long long)c.F);
  DABSN_REQUIRE(c.act >= 0 && c.act <= 3, "mlp: bad activation %d", c.act);
  DABSN_REQUIRE(strides({{c.ldx, c.H}, {c.ldw1, c.H}, {c.ldw2, c.F}}), "mlp: bad row strides %lld, %lld, %lld",
                (long long)c.ldx, (long long)c.ldw1, (long long)c.ldw2);
  return DABSN_OK;
}
static int check(const dabsn_linear_grads_call& c) {
  DABSN_REQUIRE(c.dtype == kF32 || c.dtype == kBF16, "linear gradients: bad dtype %d", c.dtype);
  DABSN_REQUIRE(c.M >= 0 && c.M < ROWS && c.N > 0 && c.N <= WIDTH - 8 && c.K > 0 && c.K < WIDTH,
                "linear gradients: bad shape M=%lld N=%lld K=%lld", (long long)c.M, (long long)c.N,
                (long long)c.K);
  DABSN_REQUIRE(strides({{c.ldx, c.K}, {c.ldw, c.K}, {c.ldg, c.N}, {c.slope ? c.lds : c.N, c.N}}),
                "linear gradients: bad row strides %lld, %lld, %lld, %lld", (long long)c.ldx,
                (long long)c.ldw, (long long)c.ldg, (long long)c.lds);
  DABSN_REQUIRE(!c.slope || c.slope_kind == 1 || c.slope_kind == 2, "linear gradients: bad slope kind %d",
                c.slope_kind);
  return DABSN_OK;
}

}  // namespace mlp
}  // namespace dabsn

using namespace dabsn;
using namespace dabsn::mlp;

#define DABSN_STEP(expr)             \
  do {                               \
    const int rc_ = (expr);          \
    if (rc_ != DABSN_OK) return rc_; \
  } while (0)

extern "C" {

int dabsn_hip_mlp_plan(dabsn_mlp_call* call, int back) {
  DABSN_REQUIRE(call, "mlp: null call");
  DABSN_STEP(check(*call));
  Space all{anywhere()};
  if (call->train) saved(*call, all);
  call->saved_bytes = all.at;
  call->workspace_bytes = back ? backward(*call, anywhere()).total : forward(*call, anywhere()).total;
  return DABSN_OK;
}

int dabsn_hip_mlp_fwd(const dabsn_mlp_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "mlp: null call");
  const dabsn_mlp_call& c = *call;
  DABSN_STEP(check(c));
  if (c.M == 0) return DABSN_OK;
  DABSN_REQUIRE(c.x && c.w1 && c.w2 && c.out, "mlp: null pointer");
  Space all{anywhere()};
  if (c.train) saved(c, all);
  char* ws = static_cast<char*>(c.workspace);
  const Forward f = forward(c, ws);
  DABSN_REQUIRE(fits(c.saved, c.saved_bytes, all.at) && fits(ws, c.workspace_bytes, f.total),
                "mlp: %zu bytes to save and a workspace of %zu, %zu and %zu needed", c.saved_bytes,
                c.workspace_bytes, all.at, f.total);
  DABSN_STEP(dabsn_hip_norm_fwd(c.dtype, c.wdtype, c.layer, c.M, c.H, c.x, c.ldx, c.norm_weight, c.norm_bias,
                                c.eps, f.v.normed, f.v.stats, stream));
  DABSN_STEP(run(f.first, ws + f.scratch_at, f.scratch, stream));
  return run(f.second, ws + f.scratch_at, f.scratch, stream);
}

int dabsn_hip_mlp_bwd(const dabsn_mlp_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "mlp backward: null call");
  const dabsn_mlp_call& c = *call;
  DABSN_STEP(check(c));
  DABSN_REQUIRE(c.train && c.w1 && c.w2 && (c.M == 0 || (c.x && c.grad)), "mlp backward: null pointer");
  Space all{anywhere()};
  saved(c, all);
  char* ws = static_cast<char*>(c.workspace);
  const Backward b = backward(c, ws);
  DABSN_REQUIRE(fits(c.saved, c.saved_bytes, all.at) && fits(ws, c.workspace_bytes, b.total),
                "mlp backward: %zu bytes saved and a workspace of %zu, %zu and %zu needed", c.saved_bytes,
                c.workspace_bytes, all.at, b.total);
  void* scratch = ws + b.scratch_at;
  if (c.db2)
    DABSN_STEP(dabsn_hip_linear_slope(c.dtype, c.M, c.H, c.grad, c.H, nullptr, 0, 0, nullptr, 0, c.db2, scratch,
                                      b.scratch, stream));
  if (c.dw2) DABSN_STEP(run(b.dw2_call, scratch, b.scratch, stream));
  if (b.rows) DABSN_STEP(run(b.dz_call, scratch, b.scratch, stream));
  if (c.db1)
    DABSN_STEP(dabsn_hip_linear_slope(c.dtype, c.M, c.F, b.dz, b.v.ldh, nullptr, 0, 0, nullptr, 0, c.db1,
                                      scratch, b.scratch, stream));
  if (c.dw1) DABSN_STEP(run(b.dw1_call, scratch, b.scratch, stream));
  if (!b.inner) return DABSN_OK;
  DABSN_STEP(run(b.dn_call, scratch, b.scratch, stream));
  return norm::backward(c.dtype, c.wdtype, kF32, c.layer, c.M, c.H, c.x, c.ldx, c.norm_weight, b.v.stats, b.dn,
                        b.ldn, c.grad, b.dx, c.dnorm_weight, c.dnorm_bias, scratch, b.scratch, stream);
}

size_t dabsn_hip_linear_grads_workspace_bytes(const dabsn_linear_grads_call* call) {
  return call && check(*call) == DABSN_OK ? layer(*call, anywhere()).total : 0;
}

int dabsn_hip_linear_grads(const dabsn_linear_grads_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "linear gradients: null call");
  const dabsn_linear_grads_call& c = *call;
  DABSN_STEP(check(c));
  DABSN_REQUIRE(c.M == 0 || (c.grad && (!c.dx || c.w) && (!c.dw || c.x)), "linear gradients: null pointer");
  char* ws = static_cast<char*>(c.workspace);
  const Layer l = layer(c, ws);
  DABSN_REQUIRE(fits(ws, c.workspace_bytes, l.total), "linear gradients: workspace of %zu bytes, %zu needed",
                c.workspace_bytes, l.total);
  void* scratch = ws + l.scratch_at;
  if (c.db || l.ldz)
    DABSN_STEP(dabsn_hip_linear_slope(c.dtype, c.M, c.N, c.grad, c.ldg, c.slope, c.lds, c.slope_kind,
                                      l.ldz ? l.dz : nullptr, l.ldz, c.db, scratch, l.scratch, stream));
  if (c.dx) DABSN_STEP(run(l.dx_call, scratch, l.scratch, stream));
  return c.dw ? run(l.dw_call, scratch, l.scratch, stream) : DABSN_OK;
}

}  // extern "C"
