// The block's MLP as a whole, forward and backward: norm, products and sums of norm.hip and linear.hip
// one after the other, with what lies between them in the caller's workspace. One call from the host
// instead of three to nine, which is what small steps wait for (2048 x 256 x 1024 fp32, forward and
// backward: 235 us with a call each, 140 so).
#include "capi.hpp"
#include "common.hpp"

#include <algorithm>

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

static dabsn_linear_call product(const dabsn_mlp_call& c, int64_t M, int64_t N, int64_t K, const void* A,
                                 int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc) {
  dabsn_linear_call l = {};
  l.dtype = c.dtype;
  l.M = M; l.N = N; l.K = K;
  l.A = A; l.lda = lda;
  l.B = B; l.ldb = ldb;
  l.C = C; l.ldc = ldc;
  return l;
}

static int run(dabsn_linear_call l, void* scratch, size_t bytes, hipStream_t s) {
  l.workspace = scratch;
  l.workspace_bytes = bytes;
  return dabsn_hip_linear(&l, s);
}

struct Forward {
  void *normed, *h;
  int64_t ldh;
  dabsn_linear_call first, second;
  size_t scratch_at, scratch, total;
};
static Forward forward(const dabsn_mlp_call& c, char* base) {
  const size_t size = c.dtype == kF32 ? 4 : 2;
  Space s{base};
  Forward f = {};
  f.ldh = c.h ? c.ldh : padded(c.F);
  f.normed = c.normed ? c.normed : s.take(static_cast<size_t>(c.M) * c.H * size);
  f.h = c.h ? c.h : s.take(static_cast<size_t>(c.M) * f.ldh * size);
  f.first = product(c, c.M, c.F, c.H, f.normed, c.H, c.w1, c.ldw1, f.h, f.ldh);
  f.first.bias = c.b1;
  f.first.act = c.act;
  if (c.act > 1) f.first.keep = c.keep, f.first.ldk = c.ldk;
  f.first.padC = 1;
  f.second = product(c, c.M, c.H, c.F, f.h, f.ldh, c.w2, c.ldw2, c.out, c.H);
  f.second.bias = c.b2;
  f.second.residual = c.x; f.second.ldr = c.ldx;
  f.second.padA = 1;
  f.scratch = std::max(dabsn_hip_linear_workspace_bytes(&f.first), dabsn_hip_linear_workspace_bytes(&f.second));
  f.scratch_at = s.at;
  f.total = s.at + f.scratch;
  return f;
}

struct Backward {
  void *dz, *dn, *dx;
  int64_t ldz;
  dabsn_linear_call dz_call, dn_call, dw1_call, dw2_call;
  bool rows, inner;  // whether dz, and what lies before it, is asked for
  size_t scratch_at, scratch, total;
};
static Backward backward(const dabsn_mlp_call& c, char* base) {
  const size_t size = c.dtype == kF32 ? 4 : 2;
  Space s{base};
  Backward b = {};
  b.ldz = padded(c.F);
  b.inner = c.dx || c.dnorm_weight || c.dnorm_bias;
  b.rows = b.inner || c.dw1 || c.db1;
  b.dz = b.rows ? s.take(static_cast<size_t>(c.M) * b.ldz * size) : nullptr;
  b.dn = b.inner ? s.take(static_cast<size_t>(c.M) * c.H * size) : nullptr;
  b.dx = c.dx || !b.inner ? c.dx : s.take(static_cast<size_t>(c.M) * c.H * size);
  const auto need = [&](const dabsn_linear_call& l) {
    b.scratch = std::max(b.scratch, dabsn_hip_linear_workspace_bytes(&l));
  };
  if (c.dw2) {
    b.dw2_call = product(c, c.H, c.F, c.M, c.grad, c.H, c.h, c.ldh, c.dw2, c.F);
    b.dw2_call.transA = b.dw2_call.transB = 1;
    need(b.dw2_call);
  }
  if (b.rows) {
    b.dz_call = product(c, c.M, c.F, c.H, c.grad, c.H, c.w2, c.ldw2, b.dz, b.ldz);
    b.dz_call.transB = 1;
    b.dz_call.padC = 1;
    if (c.act) {  // the squared ReLU's slope is its output's
      b.dz_call.slope = c.act == 1 ? c.h : c.keep;
      b.dz_call.lds = c.act == 1 ? c.ldh : c.ldk;
      b.dz_call.slope_kind = c.act == 1 ? 2 : 1;
    }
    need(b.dz_call);
  }
  if (c.dw1) {
    b.dw1_call = product(c, c.F, c.H, c.M, b.dz, b.ldz, c.normed, c.H, c.dw1, c.H);
    b.dw1_call.transA = b.dw1_call.transB = 1;
    need(b.dw1_call);
  }
  if (b.inner) {
    b.dn_call = product(c, c.M, c.H, c.F, b.dz, b.ldz, c.w1, c.ldw1, b.dn, c.H);
    b.dn_call.transB = 1;
    b.dn_call.padA = 1;
    need(b.dn_call);
    b.scratch = std::max(b.scratch, dabsn_hip_norm_workspace_bytes(c.dtype, c.M, c.H));
  }
  if (c.db1) b.scratch = std::max(b.scratch, dabsn_hip_linear_slope_workspace_bytes(c.dtype, c.M, c.F));
  if (c.db2) b.scratch = std::max(b.scratch, dabsn_hip_linear_slope_workspace_bytes(c.dtype, c.M, c.H));
  b.scratch_at = s.at;
  b.total = s.at + b.scratch;
  return b;
}

static int check(const dabsn_mlp_call& c) {
  DABSN_REQUIRE(c.dtype == kF32 || c.dtype == kBF16, "mlp: bad dtype %d", c.dtype);
  const int64_t width = (1 << 21) - 8;
  DABSN_REQUIRE(c.M >= 0 && c.M < (1ll << 31) - 65536 && c.H > 0 && c.H <= 16384 && c.F > 0 && c.F < width,
                "mlp: bad shape M=%lld H=%lld F=%lld", (long long)c.M, (long long)c.H, (long long)c.F);
  DABSN_REQUIRE(c.act >= 0 && c.act <= 3 && !(c.keep && c.act == 0), "mlp: bad activation %d", c.act);
  DABSN_REQUIRE(c.ldx >= c.H && c.ldw1 >= c.H && c.ldw2 >= c.F && (!c.h || c.ldh >= padded(c.F)) &&
                    (!c.keep || c.ldk >= c.F),
                "mlp: a row stride is shorter than its row");
  // The products' limits, so that nothing has been launched when one refuses its call.
  for (const int64_t ld : {c.ldx, c.ldw1, c.ldw2, c.ldh, c.ldk})
    DABSN_REQUIRE(ld < width + 8, "mlp: a row stride of %lld values", (long long)ld);
  DABSN_REQUIRE(c.wdtype == c.dtype || c.wdtype == kF32, "mlp: bad type %d of the norm's weight", c.wdtype);
  return DABSN_OK;
}

}  // namespace mlp
}  // namespace dabsn

using namespace dabsn;
using namespace dabsn::mlp;

#define DABSN_STEP(expr)                \
  do {                                  \
    const int rc_ = (expr);             \
    if (rc_ != DABSN_OK) return rc_;    \
  } while (0)

extern "C" {

size_t dabsn_hip_mlp_workspace_bytes(const dabsn_mlp_call* call, int back) {
  if (!call || check(*call) != DABSN_OK || (call->M == 0 && !back)) return 0;
  char* somewhere = reinterpret_cast<char*>(static_cast<uintptr_t>(4096));
  return back ? backward(*call, somewhere).total : forward(*call, somewhere).total;
}

int dabsn_hip_mlp_fwd(const dabsn_mlp_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "mlp: null call");
  const dabsn_mlp_call& c = *call;
  DABSN_STEP(check(c));
  if (c.M == 0) return DABSN_OK;
  DABSN_REQUIRE(c.x && c.w1 && c.w2 && c.out, "mlp: null pointer");
  char* ws = static_cast<char*>(c.workspace);
  const Forward f = forward(c, ws);
  DABSN_REQUIRE(f.total == 0 || (ws && c.workspace_bytes >= f.total && (reinterpret_cast<uintptr_t>(ws) & 15u) == 0),
                "mlp: workspace of %zu bytes, %zu needed", c.workspace_bytes, f.total);
  DABSN_STEP(dabsn_hip_norm_fwd(c.dtype, c.wdtype, c.layer, c.M, c.H, c.x, c.ldx, c.norm_weight, c.norm_bias,
                                c.eps, f.normed, c.stats, stream));
  DABSN_STEP(run(f.first, ws + f.scratch_at, f.scratch, stream));
  return run(f.second, ws + f.scratch_at, f.scratch, stream);
}

int dabsn_hip_mlp_bwd(const dabsn_mlp_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "mlp backward: null call");
  const dabsn_mlp_call& c = *call;
  DABSN_STEP(check(c));
  DABSN_REQUIRE(c.w1 && c.w2 && (c.M == 0 || (c.x && c.grad && c.normed && c.stats && c.h)),
                "mlp backward: null pointer");
  DABSN_REQUIRE(c.act <= 1 || c.keep || c.M == 0, "mlp backward: no slope");
  char* ws = static_cast<char*>(c.workspace);
  const Backward b = backward(c, ws);
  DABSN_REQUIRE(b.total == 0 || (ws && c.workspace_bytes >= b.total && (reinterpret_cast<uintptr_t>(ws) & 15u) == 0),
                "mlp backward: workspace of %zu bytes, %zu needed", c.workspace_bytes, b.total);
  void* scratch = ws + b.scratch_at;
  if (c.db2)
    DABSN_STEP(dabsn_hip_linear_slope(c.dtype, c.M, c.H, c.grad, c.H, nullptr, 0, 0, nullptr, 0, c.db2, scratch,
                                      b.scratch, stream));
  if (c.dw2) DABSN_STEP(run(b.dw2_call, scratch, b.scratch, stream));
  if (b.rows) DABSN_STEP(run(b.dz_call, scratch, b.scratch, stream));
  if (c.db1)
    DABSN_STEP(dabsn_hip_linear_slope(c.dtype, c.M, c.F, b.dz, b.ldz, nullptr, 0, 0, nullptr, 0, c.db1, scratch,
                                      b.scratch, stream));
  if (c.dw1) DABSN_STEP(run(b.dw1_call, scratch, b.scratch, stream));
  if (!b.inner) return DABSN_OK;
  DABSN_STEP(run(b.dn_call, scratch, b.scratch, stream));
  return dabsn_hip_norm_bwd(c.dtype, c.wdtype, c.layer, c.M, c.H, c.x, c.ldx, c.norm_weight, c.stats, b.dn, c.H,
                            c.grad, b.dx, c.dnorm_weight, c.dnorm_bias, scratch, b.scratch, stream);
}

}  // extern "C"
