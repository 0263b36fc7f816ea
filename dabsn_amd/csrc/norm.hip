// Layer norm and RMS norm of rows, forward and backward.
//
//   u = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = u * w + b
//   (RMS norm: mean = 0, no b)
//   dx = rstd * (gw - mean(gw) - u * mean(gw u)) [+ add],  gw = g * w;  dw = sum g u;  db = sum g
//
// HBM bound: the forward reads a row and writes one, the backward reads two and writes one. A
// row is held in the registers of T threads (64: a wave, four rows a workgroup; 256 or 1024: a
// workgroup), NV vectors of 16 bytes each, so that the mean, the squares around it and the
// result come from one reading: 65536 x 4096 bf16 in 211 us, backward 312 to 322 (5.1 and 5.0 TB/s; a
// copy reaches 5.2; 332 and 534 before the next row was loaded ahead). Sums are fp32: a thread's, then a wave's, then the workgroup's.
//
// The backward's workgroups walk over the rows with a column's dw and db in the registers of the
// thread that holds the column, and leave one partial row each; join_kernel adds these in order.
// The same inputs give the same bits.
#include "norm.hpp"

#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace dabsn {
namespace norm {

constexpr int64_t MAX_WIDTH = 16384;

template <typename E>
constexpr int vec_of() { return 16 / static_cast<int>(sizeof(E)); }

// A thread's vector of a row as it is stored, at any alignment; elements beyond `left` are 0.
template <typename E, int VEC = vec_of<E>()>
struct Raw {
  static constexpr int PER = vec_of<E>();
  u32x4 q[VEC / PER];
  __device__ __forceinline__ void load(const E* p, int left) {
    if (left >= VEC) {
      __builtin_memcpy(q, p, sizeof(q));
    } else {
      E e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = i < left ? p[i] : static_cast<E>(0);
      __builtin_memcpy(q, e, sizeof(q));
    }
  }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w = q[e / PER][sizeof(E) == 4 ? e % PER : e % PER / 2];
    if constexpr (sizeof(E) == 4) return __builtin_bit_cast(float, w);
    else return __builtin_bit_cast(float, e % 2 ? w & 0xffff0000u : w << 16);
  }
};

// VEC elements of a weight or bias; those beyond `left` are 0.
template <typename E, int VEC>
__device__ __forceinline__ void load_row(const E* p, int left, float (&v)[VEC]) {
  if (left >= VEC) {
    E raw[VEC];
    __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = to_f(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = e < left ? to_f(p[e]) : 0.0f;
  }
}

template <typename E, int VEC>
__device__ __forceinline__ void store_row(E* p, int left, const float (&v)[VEC]) {
  if (left >= VEC) {
    E raw[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) raw[e] = from_f<E>(v[e]);
    __builtin_memcpy(p, raw, sizeof(raw));
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e < left) p[e] = from_f<E>(v[e]);
  }
}

// The sum over a row's threads; `part` has a slot a wave and must not be in use.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = wave_sum(v);
  if constexpr (T == 64) return v;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) total += part[w];
  return total;
}

// Workgroup `blockIdx.x` of `gridDim.x` takes rows blockIdx.x * R + (its row slot), and so on by
// gridDim.x * R, the next row on its way while one is worked on.
template <typename E, typename W, int T, int NV>
__global__ void __launch_bounds__(T < 256 ? 256 : T)
    fwd_kernel(int64_t rows, int H, const E* x, int64_t ldx, const W* weight, const W* bias,
               float eps, int center, E* out, float* stats) {
  constexpr int VEC = vec_of<E>(), R = T < 256 ? 256 / T : 1;
  __shared__ float part[2][2][T / 64];
  const int t = threadIdx.x % T;
  const float inv = 1.0f / static_cast<float>(H);
  Raw<E> next[NV];
  auto fetch = [&](int64_t row) {
    if (row >= rows) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * VEC;
      next[i].load(x + row * ldx + c, H - c);
    }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * R + threadIdx.x / T;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * R;
  fetch(row);
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * T + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[i][e] = 1.0f;
      b[i][e] = 0.0f;
    }
    if (weight && c < H) load_row<W, VEC>(weight + c, H - c, w[i]);
    if (bias && c < H) load_row<W, VEC>(bias + c, H - c, b[i]);
  }
  int turn = 0;
  for (; row < rows; row += stride, turn ^= 1) {  // a row of several waves is the workgroup's
    float v[NV][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = next[i].get(e);
        sum += v[i][e];
      }
    fetch(row + stride);
    // The slots alternate: a wave that is still adding the last row's finds them untouched.
    const float mean = center ? row_sum<T>(sum, part[turn][0]) * inv : 0.0f;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = c + e < H ? v[i][e] - mean : 0.0f;
        sq = fmaf(v[i][e], v[i][e], sq);
      }
    }
    const float rstd = 1.0f / sqrtf(fmaf(row_sum<T>(sq, part[turn][1]), inv, eps));
    if (stats && t == 0) {
      stats[2 * row] = mean;
      stats[2 * row + 1] = rstd;
    }
    E* o = out + row * H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * VEC;
      if (c >= H) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = v[i][e] * rstd * w[i][e] + b[i][e];
      store_row<E, VEC>(o + c, H - c, v[i]);
    }
  }
}

// Rows as in fwd_kernel; parts [gridDim.x][2][H] (dw, db; NULL: not needed). G: type of the gradient's
// rows, which the block's MLP leaves in fp32 beside bf16 (65536 x 2048 with ADD: 252 us, 5.3 TB/s). With
// ADD the rows to add are on their way with the next row too (loaded where they are used they waited for it: 65536 x 2048
// bf16 299 us, 200 so; without ADD their registers cost 77 -> 95 us at 30011 x 1001 fp32).
template <typename E, typename W, typename G, int T, int NV, bool ADD>
__global__ void __launch_bounds__(T < 256 ? 256 : T)
    bwd_kernel(int64_t rows, int H, const E* x, int64_t ldx, const W* weight, const float* stats,
               int center, const G* grad, int64_t ldg, const E* add, E* dx, float* parts) {
  constexpr int VEC = vec_of<E>(), R = T < 256 ? 256 / T : 1;
  __shared__ float part[2][2][T / 64];
  __shared__ float lds[R > 1 ? R : 1][R > 1 ? 2 * T * VEC : 1];
  const int t = threadIdx.x % T, slot = threadIdx.x / T;
  const float inv = 1.0f / static_cast<float>(H);
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * T + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[i][e] = 1.0f;
      dw[i][e] = db[i][e] = 0.0f;
    }
    if (weight && c < H) load_row<W, VEC>(weight + c, H - c, w[i]);
  }
  Raw<E> nextx[NV], nexta[NV];
  Raw<G, VEC> nextg[NV];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
    if (row >= rows) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * VEC;
      nextx[i].load(x + row * ldx + c, H - c);
      nextg[i].load(grad + row * ldg + c, H - c);
      if constexpr (ADD) nexta[i].load(add + row * H + c, H - c);
    }
    next_mean = stats[2 * row];
    next_rstd = stats[2 * row + 1];
  };
  int turn = 0;
  int64_t row = static_cast<int64_t>(blockIdx.x) * R + slot;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * R;
  fetch(row);
  for (; row < rows; row += stride, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    float u[NV][VEC], g[NV][VEC];
    Raw<E> a[NV];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (ADD) a[i] = nexta[i];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        u[i][e] = (nextx[i].get(e) - mean) * rstd;  // beyond H: g = 0, and u meets nothing else
        g[i][e] = nextg[i].get(e);
        dw[i][e] = fmaf(g[i][e], u[i][e], dw[i][e]);
        db[i][e] += g[i][e];
        g[i][e] *= w[i][e];
        s1 += g[i][e];
        s2 = fmaf(g[i][e], u[i][e], s2);
      }
    }
    fetch(row + stride);
    s1 = center ? row_sum<T>(s1, part[turn][0]) * inv : 0.0f;
    s2 = row_sum<T>(s2, part[turn][1]) * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * VEC;
      if (c >= H) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        u[i][e] = rstd * (g[i][e] - fmaf(u[i][e], s2, s1));
        if constexpr (ADD) u[i][e] += a[i].get(e);
      }
      store_row<E, VEC>(dx + row * H + c, H - c, u[i]);
    }
  }
  if (!parts) return;
  float* pw = parts + static_cast<int64_t>(blockIdx.x) * 2 * H;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * T + t) * VEC;
    if constexpr (R > 1) {
      // The workgroup's row slots, added in order.
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        lds[slot][t * VEC + e] = dw[i][e];
        lds[slot][(T + t) * VEC + e] = db[i][e];
      }
      __syncthreads();
      for (int j = threadIdx.x; j < 2 * T * VEC; j += 256) {
        const int col = i * T * VEC + j % (T * VEC);
        if (col >= H) continue;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < R; ++k) s += lds[k][j];
        pw[(j < T * VEC ? 0 : H) + col] = s;
      }
    } else if (c < H) {
      store_row<float, VEC>(pw + c, H - c, dw[i]);
      store_row<float, VEC>(pw + H + c, H - c, db[i]);
    }
  }
}

// out0 [n0] and out1 [n - n0] = the sums of parts' columns [P][n]: a thread a column and a
// sixteenth of the partial rows, joined in order. Either output may be NULL.
template <typename W>
__global__ void __launch_bounds__(1024) join_kernel(int P, int n, int n0, const float* parts,
                                                    W* out0, W* out1) {
  __shared__ float lds[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), slot = threadIdx.x >> 6;
  float s = 0.0f;
  if (col < n)
#pragma unroll 4
    for (int p = slot; p < P; p += 16) s += parts[static_cast<int64_t>(p) * n + col];
  lds[slot][threadIdx.x & 63] = s;
  __syncthreads();
  if (slot || col >= n) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += lds[k][threadIdx.x];
  if (col < n0) {
    if (out0) st(out0, col, s);
  } else if (out1) {
    st(out1, col - n0, s);
  }
}

// Threads a row and vectors a thread. A wave takes a row of up to four vectors a lane: no barrier,
// four rows a workgroup; wider rows, or few of them (a row a workgroup finishes sooner), take
// more threads.
struct Plan {
  int T, NV;
};
static Plan plan_of(int64_t rows, int64_t H, int vec) {
  const int64_t v = (H + vec - 1) / vec;  // vectors a row
  Plan p;
  if (v <= 64 || (v <= 256 && rows > 1024)) {
    p.T = 64;
  } else {
    p.T = v <= 1024 ? 256 : 1024;
  }
  const int64_t nv = (v + p.T - 1) / p.T;
  p.NV = nv <= 1 ? 1 : nv <= 2 ? 2 : 4;
  return p;
}

// Partial rows of the backward: workgroups that fill the card once by their registers, each with 4
// rows or more.
static int64_t parts_of(int64_t rows, int64_t H, int vec) {
  const Plan p = plan_of(rows, H, vec);
  const int64_t slots = p.T < 256 ? 256 / p.T : 1;
  const int values = p.NV * vec;
  const int64_t most = 256 * (p.T == 1024 ? 1 : values <= 4 ? 8 : values <= 8 ? 4 : values <= 16 ? 3 : 2);
  return std::max<int64_t>(1, std::min<int64_t>(most, (rows + 4 * slots - 1) / (4 * slots)));
}

template <typename E, typename F>
static int with_plan(const Plan& p, F&& f) {
#define C(T_, NV_) \
  if (p.T == T_ && p.NV == NV_) return f(std::integral_constant<int, T_>{}, std::integral_constant<int, NV_>{})
  C(64, 1); C(64, 2); C(64, 4);
  C(256, 1); C(256, 2); C(256, 4);
  C(1024, 1); C(1024, 2);
  if constexpr (1024 * 2 * vec_of<E>() < MAX_WIDTH) C(1024, 4);
#undef C
  return DABSN_ERR_ARG;
}

template <typename E, typename W>
static int run_fwd(int64_t rows, int H, const void* x, int64_t ldx, const void* w, const void* b,
                   float eps, int center, void* out, float* stats, hipStream_t s) {
  const Plan p = plan_of(rows, H, vec_of<E>());
  return with_plan<E>(p, [&](auto T, auto NV) {
    constexpr int R = T < 256 ? 256 / T : 1;
    // Eight workgroups a unit (two of 1024 threads), or one a row.
    const int64_t most = T == 1024 ? 512 : 2048;
    hipLaunchKernelGGL((fwd_kernel<E, W, T, NV>), dim3((unsigned)std::min((rows + R - 1) / R, most)),
                       dim3(T < 256 ? 256 : T), 0, s, rows, H, (const E*)x, ldx, (const W*)w,
                       (const W*)b, eps, center, (E*)out, stats);
    DABSN_HIP_CHECK(hipGetLastError());
    return DABSN_OK;
  });
}

template <typename E, typename W, typename G>
static int run_bwd(int64_t rows, int H, const void* x, int64_t ldx, const void* w,
                   const float* stats, int center, const void* g, int64_t ldg, const void* add,
                   void* dx, void* dw, void* db, float* parts, hipStream_t s) {
  const Plan p = plan_of(rows, H, vec_of<E>());
  const int64_t P = parts_of(rows, H, vec_of<E>());
  const int rc = with_plan<E>(p, [&](auto T, auto NV) {
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)P), dim3(T < 256 ? 256 : T), 0, s, rows, H, (const E*)x,
                         ldx, (const W*)w, stats, center, (const G*)g, ldg, (const E*)add, (E*)dx, parts);
    };
    if (add) launch(bwd_kernel<E, W, G, T, NV, true>);
    else if constexpr (std::is_same_v<E, G>) launch(bwd_kernel<E, W, G, T, NV, false>);
    DABSN_HIP_CHECK(hipGetLastError());
    return DABSN_OK;
  });
  if (rc != DABSN_OK || !parts) return rc;
  hipLaunchKernelGGL(join_kernel<W>, dim3((unsigned)((2 * H + 63) / 64)), dim3(1024), 0, s, (int)P,
                     2 * H, H, parts, (W*)dw, (W*)db);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

}  // namespace norm
}  // namespace dabsn

using namespace dabsn;
using namespace dabsn::norm;

static int check_norm(const char* what, int dtype, int wdtype, int64_t rows, int64_t H, int64_t ldx) {
  DABSN_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: bad dtype %d", what, dtype);
  DABSN_REQUIRE(wdtype == dtype || wdtype == kF32, "%s: bad weight dtype %d", what, wdtype);
  DABSN_REQUIRE(H > 0 && H <= MAX_WIDTH && rows >= 0 && rows < (1ll << 31) && ldx >= H,
                "%s: bad shape rows=%lld H=%lld ld=%lld", what, (long long)rows, (long long)H,
                (long long)ldx);
  return DABSN_OK;
}

int norm::backward(int dtype, int wdtype, int gdtype, int layer, int64_t rows, int64_t H, const void* x,
                   int64_t ldx, const void* weight, const float* stats, const void* grad, int64_t ldg,
                   const void* add, void* dx, void* dweight, void* dbias, void* workspace,
                   size_t workspace_bytes, hipStream_t stream) {
  const int rc = check_norm("norm backward", dtype, wdtype, rows, H, std::min(ldx, ldg));
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(gdtype == dtype || (gdtype == kF32 && (add || rows == 0)), "norm backward: bad gradient dtype %d", gdtype);
  float* parts = nullptr;
  if (dweight || dbias) {
    parts = static_cast<float*>(workspace);
    const size_t need = dabsn_hip_norm_workspace_bytes(dtype, rows, H);
    DABSN_REQUIRE(rows == 0 || (parts && workspace_bytes >= need),
                  "norm backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  }
  if (rows == 0) {  // no rows: zero sums
    for (void* p : {dweight, dbias})
      if (p) {
        const unsigned blocks = (unsigned)((H + 63) / 64);
        if (wdtype == kF32)
          hipLaunchKernelGGL(join_kernel<float>, dim3(blocks), dim3(1024), 0, stream, 0, (int)H,
                             (int)H, nullptr, (float*)p, (float*)nullptr);
        else
          hipLaunchKernelGGL(join_kernel<bf16>, dim3(blocks), dim3(1024), 0, stream, 0, (int)H,
                             (int)H, nullptr, (bf16*)p, (bf16*)nullptr);
        DABSN_HIP_CHECK(hipGetLastError());
      }
    return DABSN_OK;
  }
  DABSN_REQUIRE(x && stats && grad && dx, "norm backward: null pointer");
  const auto run = [&](auto kernels) {
    return kernels(rows, (int)H, x, ldx, weight, stats, layer != 0, grad, ldg, add, dx, dweight, dbias, parts,
                   stream);
  };
  if (dtype == kF32) return run(run_bwd<float, float, float>);
  if (gdtype == dtype) return wdtype == kF32 ? run(run_bwd<bf16, float, bf16>) : run(run_bwd<bf16, bf16, bf16>);
  return wdtype == kF32 ? run(run_bwd<bf16, float, float>) : run(run_bwd<bf16, bf16, float>);
}

extern "C" {

int dabsn_hip_norm_fwd(int dtype, int wdtype, int layer, int64_t rows, int64_t H, const void* x,
                       int64_t ldx, const void* weight, const void* bias, float eps, void* out,
                       float* stats, hipStream_t stream) {
  const int rc = check_norm("norm", dtype, wdtype, rows, H, ldx);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(eps >= 0.0f, "norm: bad eps");
  if (rows == 0) return DABSN_OK;
  DABSN_REQUIRE(x && out, "norm: null pointer");
  if (dtype == kF32)
    return run_fwd<float, float>(rows, (int)H, x, ldx, weight, bias, eps, layer != 0, out, stats, stream);
  if (wdtype == kF32)
    return run_fwd<bf16, float>(rows, (int)H, x, ldx, weight, bias, eps, layer != 0, out, stats, stream);
  return run_fwd<bf16, bf16>(rows, (int)H, x, ldx, weight, bias, eps, layer != 0, out, stats, stream);
}

size_t dabsn_hip_norm_workspace_bytes(int dtype, int64_t rows, int64_t H) {
  if (rows <= 0 || H <= 0 || H > MAX_WIDTH || (dtype != kF32 && dtype != kBF16)) return 0;
  return static_cast<size_t>(parts_of(rows, H, dtype == kF32 ? 4 : 8)) * 2 * H * sizeof(float);
}

int dabsn_hip_norm_bwd(int dtype, int wdtype, int layer, int64_t rows, int64_t H, const void* x,
                       int64_t ldx, const void* weight, const float* stats, const void* grad,
                       int64_t ldg, const void* add, void* dx, void* dweight, void* dbias,
                       void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return norm::backward(dtype, wdtype, dtype, layer, rows, H, x, ldx, weight, stats, grad, ldg, add, dx,
                        dweight, dbias, workspace, workspace_bytes, stream);
}

}  // extern "C"
