// Matrix products with the work around them in their epilogue, for the block's MLP.
//
//   C(m, n) = act(sum_k A(m, k) B(n, k) + bias(n)) * slope(m, n) + residual(m, n)
//
// in fp32, rounded once to the type of A and B. An operand is K-contiguous, A[m * lda + k], or
// stored as its transpose, A[k * lda + m]: the forward needs neither transposed, the gradient of
// the rows has B = W transposed, that of the weight both. The products are bound by the matrix
// cores once there are a few hundred rows, by the weight's bytes below.
//
// A workgroup of WM x WN waves forms a BM x BN tile, BK deep steps through two buffers in LDS:
// while the matrix instructions take step k from one, the loads of step k + 2 are on their way to
// registers and step k + 1 goes to the other. Operands come at any alignment (unaligned 16-byte
// loads), beyond their edge as zeros.
#include "capi.hpp"
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace dabsn {
namespace linear {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

enum Act : int { kNone = 0, kRelu2 = 1, kGelu = 2, kSilu = 3 };
// Where the factor of the epilogue comes from: none, a stored slope, or the squared ReLU's output
// h, whose slope is 2 sqrt(h).
enum Slope : int { kNoSlope = 0, kStored = 1, kFromSquare = 2 };

template <typename E>
struct Args {
  int M, N, K;
  const E *A, *B;
  int64_t lda, ldb;
  const E* bias;
  int act;
  const E* slope;
  int64_t lds;
  int slope_kind;
  const E* residual;
  int64_t ldr;
  E* C;
  int64_t ldc;
  E* keep;  // act'(z); NULL: not kept
  int64_t ldk;
  int mt, nt, splits, kper;
  float* parts;  // [splits][M][ldp]: the splits' sums, instead of C
  int64_t ldp;
};

// act(z) and its derivative.
template <typename E>
__device__ __forceinline__ float activate(int act, float z, float& slope) {
  if (act == kRelu2) {
    const float r = z > 0.0f || z != z ? z : 0.0f;
    slope = 2.0f * r;
    return r * r;
  }
  if (act == kGelu) {
    const float below = 0.5f * erfcf(z * -0.70710678118654752f);
    slope = fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), below);
    return z * below;
  }
  if (act == kSilu) {
    const float s = 1.0f / (1.0f + expf(-z)), rest = 1.0f / (1.0f + expf(z));
    slope = fmaf(z * s, rest, s);
    return z * s;
  }
  slope = 1.0f;
  return z;
}

__device__ __forceinline__ float factor(int kind, float s) {
  return kind == kFromSquare ? 2.0f * sqrtf(s) : s;
}

template <typename E>
__device__ __forceinline__ void put_one(const Args<E>& a, int m, int n, float v) {
  if (a.bias) v += ld(a.bias, n);
  float slope;
  v = activate<E>(a.act, v, slope);
  if (a.keep) st(a.keep, static_cast<size_t>(m) * a.ldk + n, slope);
  if (a.slope_kind) v *= factor(a.slope_kind, ld(a.slope, static_cast<size_t>(m) * a.lds + n));
  if (a.residual) v += ld(a.residual, static_cast<size_t>(m) * a.ldr + n);
  st(a.C, static_cast<size_t>(m) * a.ldc + n, v);
}

template <typename E, bool T, int BT, int BK, int NTH>
struct Stage {
  static constexpr int VEC = 16 / static_cast<int>(sizeof(E));
  static constexpr int COLS = T ? BT : BK, ROWS = T ? BK : BT;
  static constexpr int CPR = COLS / VEC, NV = ROWS * CPR / NTH;
  static_assert(ROWS * CPR % NTH == 0, "staging must divide evenly");

  // Position of 16-byte chunk c in row r of the tile. K-contiguous rows are 128 bytes: the 16 lanes
  // of one read (a chunk of 16 rows) then touch all 64 banks. Transposed rows are read in pieces of
  // 32 bytes (bf16: four rows by 16 columns a 16 lanes) or 64 (fp32: 16 columns of a row), eight or
  // four of them by different rows at once.
  __device__ static int pos(int c, int r) {
    if constexpr (!T) return c ^ ((r >> 1) & 7);
    if constexpr (sizeof(E) == 2) return c ^ (((r & 3) | ((r >> 1) & 4)) << 1);
    return c ^ (((r >> 2) & 3) << 2);
  }

  // Chunks of the tile at row r0, column c0 of a matrix of `rows` x `cols`, zeros beyond.
  __device__ static void load(const E* p, int64_t ld, int r0, int c0, int rows, int cols, int tid,
                              u32x4 (&v)[NV]) {
    const bool inside = r0 + ROWS <= rows && c0 + COLS <= cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = tid + i * NTH, r = r0 + q / CPR, c = c0 + q % CPR * VEC;
      const E* at = p + static_cast<int64_t>(r) * ld + c;
      if (inside || (r < rows && c + VEC <= cols)) {
        __builtin_memcpy(&v[i], at, 16);
      } else {
        E raw[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) raw[e] = r < rows && c + e < cols ? at[e] : static_cast<E>(0);
        __builtin_memcpy(&v[i], raw, 16);
      }
    }
  }
  __device__ static void store(E* lds, int tid, const u32x4 (&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = tid + i * NTH, r = q / CPR;
      *reinterpret_cast<u32x4*>(lds + r * COLS + pos(q % CPR, r) * VEC) = v[i];
    }
  }
};

// Fragments of a wave's 16-row tiles for the matrix instructions.
template <typename E, bool T, int BT, int BK>
struct Frag;
template <bool T, int BT, int BK>
struct Frag<bf16, T, BT, BK> {
  static constexpr int KSTEP = 32;
  using R = bf16x8;
  // Rows row0 + (lane & 15), k = ks * 32 + (lane >> 4) * 8 + 0..7.
  __device__ static R get(const bf16* lds, int row0, int ks, int lane) {
    const int li = lane & 15, g = lane >> 4;
    if constexpr (!T) {
      const int r = row0 + li;
      return __builtin_bit_cast(
          R, *reinterpret_cast<const u32x4*>(lds + r * BK + ((ks * 4 + g) ^ ((r >> 1) & 7)) * 8));
    } else {
      // Two transposing reads: each takes four k of 16 columns per 16 lanes.
      const int f = (li >> 2) | ((g & 1) << 2);
      const bf16* at = lds + (ks * 32 + g * 8 + (li >> 2)) * BT + ((row0 >> 4) ^ f) * 16 + (li & 3) * 4;
      using L = __attribute__((address_space(3))) s16x4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(at + 4 * BT));
      return __builtin_bit_cast(R, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  __device__ static f32x4 mma(R a, R b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <bool T, int BT, int BK>
struct Frag<float, T, BT, BK> {
  static constexpr int KSTEP = 16;
  using R = f32x4;
  // Rows row0 + (lane & 15), k = ks * 16 + (lane >> 4) * 4 + 0..3: four matrix instructions of
  // four k each, one element of every group at a time.
  __device__ static R get(const float* lds, int row0, int ks, int lane) {
    const int li = lane & 15, g = lane >> 4;
    if constexpr (!T) {
      const int r = row0 + li;
      return *reinterpret_cast<const f32x4*>(lds + r * BK + ((ks * 4 + g) ^ ((r >> 1) & 7)) * 4);
    } else {
      const float* at = lds + (ks * 16 + g * 4) * BT + ((row0 >> 4) ^ g) * 16 + li;
      return (f32x4){at[0], at[BT], at[2 * BT], at[3 * BT]};
    }
  }
  __device__ static f32x4 mma(R a, R b, f32x4 c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};

// The tile and split of workgroup L: consecutive workgroups go round the 8 XCDs, so each XCD gets a
// contiguous range of the order, patches of 8 x 8 tiles whose operands its L2 holds.
__device__ __forceinline__ bool tile_of(int L, int nblk, int splits, int mt_n, int nt_n, int& sp,
                                        int& mt, int& nt) {
  const int g = (L % 8) * (nblk / 8) + L / 8, per = mt_n * nt_n;
  if (g >= splits * per) return false;
  sp = g / per;
  int r = g % per;
  const int band = r / (8 * nt_n);
  r %= 8 * nt_n;
  const int rows = min(8, mt_n - band * 8);
  const int pcol = r / (rows * 8);
  r %= rows * 8;
  const int cols = min(8, nt_n - pcol * 8);
  mt = band * 8 + r / cols;
  nt = pcol * 8 + r % cols;
  return true;
}

template <typename E, bool TA, bool TB, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) product_kernel(Args<E> a, int nblk) {
  constexpr int NTH = WM * WN * 64, BK = 128 / static_cast<int>(sizeof(E));
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  using SA = Stage<E, TA, BM, BK, NTH>;
  using SB = Stage<E, TB, BN, BK, NTH>;
  using FA = Frag<E, TA, BM, BK>;
  using FB = Frag<E, TB, BN, BK>;
  __shared__ __attribute__((aligned(16))) E ldsA[2][BM * BK], ldsB[2][BN * BK];

  int sp, mt, nt;
  if (!tile_of(blockIdx.x, nblk, a.splits, a.mt, a.nt, sp, mt, nt)) return;
  const int m0 = mt * BM, n0 = nt * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int k0 = sp * a.kper, kend = min(a.K, k0 + a.kper);
  const int steps = (kend - k0 + BK - 1) / BK;

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  u32x4 va[SA::NV], vb[SB::NV];
  auto load = [&](int it) {
    const int k = k0 + it * BK;
    if constexpr (TA) SA::load(a.A, a.lda, k, m0, kend, a.M, tid, va);
    else SA::load(a.A, a.lda, m0, k, a.M, kend, tid, va);
    if constexpr (TB) SB::load(a.B, a.ldb, k, n0, kend, a.N, tid, vb);
    else SB::load(a.B, a.ldb, n0, k, a.N, kend, tid, vb);
  };
  auto store = [&](int buf) {
    SA::store(ldsA[buf], tid, va);
    SB::store(ldsB[buf], tid, vb);
  };
  if (steps > 0) {
    load(0);
    store(0);
    if (steps > 1) load(1);
  }
  __syncthreads();
  for (int it = 0; it < steps; ++it) {
    const int buf = it & 1;
    if (it + 1 < steps) {
      store(buf ^ 1);  // released by the barrier that ended step it - 1
      if (it + 2 < steps) load(it + 2);
    }
#pragma unroll
    for (int ks = 0; ks < BK / FA::KSTEP; ++ks) {
      typename FA::R af[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) af[i] = FA::get(ldsA[buf], wm + i * 16, ks, lane);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const typename FB::R bf = FB::get(ldsB[buf], wn + j * 16, ks, lane);
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = FA::mma(bf, af[i], acc[i][j]);
      }
    }
    __syncthreads();
  }

  // B is the instruction's first operand: a lane holds four consecutive columns of a row.
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm + i * 16 + (lane & 15);
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
      if (a.parts) {
        float* p = a.parts + (static_cast<int64_t>(sp) * a.M + m) * a.ldp + n;
        if (n < a.ldp) *reinterpret_cast<f32x4*>(p) = acc[i][j];  // ldp is a multiple of 4
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < a.N) put_one(a, m, n + r, acc[i][j][r]);
      }
    }
  }
}

// The splits' sums in order, then the epilogue: a thread four columns.
template <typename E>
__global__ void __launch_bounds__(256) join_kernel(Args<E> a) {
  const int64_t quads = a.ldp / 4, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= quads * a.M) return;
  const int m = static_cast<int>(i / quads), n = static_cast<int>(i % quads) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s)
    v += *reinterpret_cast<const f32x4*>(a.parts + (static_cast<int64_t>(s) * a.M + m) * a.ldp + n);
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < a.N) put_one(a, m, n + r, v[r]);
}

// Tiles of 128 x 128, and as many splits of K as bring the workgroups to the card's 256 units,
// each of at least 8 steps.
struct Plan {
  int mt, nt, splits, kper;
  int64_t ldp;
};
static Plan plan_of(int64_t M, int64_t N, int64_t K, int size) {
  const int64_t BK = 128 / size;
  Plan p;
  p.mt = static_cast<int>((M + 127) / 128);
  p.nt = static_cast<int>((N + 127) / 128);
  const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt, steps = (K + BK - 1) / BK;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({256 / tiles, steps / 8, 64}));
  const int64_t each = std::max<int64_t>(1, (steps + splits - 1) / splits);
  p.splits = static_cast<int>(std::max<int64_t>(1, (steps + each - 1) / each));
  p.kper = static_cast<int>(each * BK);
  p.ldp = (N + 3) / 4 * 4;
  return p;
}

template <typename E>
static int run(const dabsn_linear_call& c, hipStream_t s) {
  const Plan p = plan_of(c.M, c.N, c.K, sizeof(E));
  Args<E> a = {};
  a.M = (int)c.M; a.N = (int)c.N; a.K = (int)c.K;
  a.A = (const E*)c.A; a.B = (const E*)c.B; a.lda = c.lda; a.ldb = c.ldb;
  a.bias = (const E*)c.bias; a.act = c.act;
  a.slope = (const E*)c.slope; a.lds = c.lds; a.slope_kind = c.slope ? c.slope_kind : kNoSlope;
  a.residual = (const E*)c.residual; a.ldr = c.ldr;
  a.C = (E*)c.C; a.ldc = c.ldc; a.keep = (E*)c.keep; a.ldk = c.ldk;
  a.mt = p.mt; a.nt = p.nt; a.splits = p.splits; a.kper = p.kper; a.ldp = p.ldp;
  a.parts = p.splits > 1 ? (float*)c.workspace : nullptr;
  const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt * p.splits;
  DABSN_REQUIRE(tiles < (1ll << 31) - 8, "linear: too many tiles");
  const int nblk = (int)((tiles + 7) / 8 * 8);
#define L(TA, TB) \
  hipLaunchKernelGGL((product_kernel<E, TA, TB, 128, 128, 2, 2>), dim3(nblk), dim3(256), 0, s, a, nblk)
  if (c.transA) L(true, true);
  else if (c.transB) L(false, true);
  else L(false, false);
#undef L
  DABSN_HIP_CHECK(hipGetLastError());
  if (a.parts) {
    const int64_t blocks = (p.ldp / 4 * c.M + 255) / 256;
    DABSN_REQUIRE(blocks < (1ll << 31), "linear: too many elements to join");
    hipLaunchKernelGGL(join_kernel<E>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    DABSN_HIP_CHECK(hipGetLastError());
  }
  return DABSN_OK;
}

// dz = g * slope (NULL: not written) and partial column sums of it (NULL: none) over a range of rows
// each. A workgroup takes 64 lanes by VEC columns and every fourth row of its range.
template <typename E>
__global__ void __launch_bounds__(256) slope_kernel(int64_t rows, int n, const E* g, int64_t ldg,
                                                    const E* s, int64_t lds, int kind, E* dz,
                                                    int64_t ldz, float* parts) {
  constexpr int VEC = 16 / static_cast<int>(sizeof(E));
  __shared__ float lds_[4][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * VEC;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = std::min(rows, r0 + per);
  float sum[VEC] = {};
  if (c < n) {
    const bool whole = c + VEC <= n;
    for (int64_t r = r0 + wave; r < r1; r += 4) {
      E gv[VEC], sv[VEC], o[VEC];
      if (whole) {
        __builtin_memcpy(gv, g + r * ldg + c, 16);
        if (kind) __builtin_memcpy(sv, s + r * lds + c, 16);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          gv[e] = c + e < n ? g[r * ldg + c + e] : static_cast<E>(0);
          if (kind) sv[e] = c + e < n ? s[r * lds + c + e] : static_cast<E>(0);
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = to_f(gv[e]);
        if (kind) v *= factor(kind, to_f(sv[e]));
        sum[e] += v;
        o[e] = from_f<E>(v);
      }
      if (dz) {
        if (whole) {
          __builtin_memcpy(dz + r * ldz + c, o, 16);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (c + e < n) dz[r * ldz + c + e] = o[e];
        }
      }
    }
  }
  if (!parts) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) lds_[wave][lane * VEC + e] = sum[e];
  __syncthreads();
  for (int j = threadIdx.x; j < 64 * VEC; j += 256) {
    const int col = blockIdx.x * 64 * VEC + j;
    if (col < n)
      parts[static_cast<int64_t>(blockIdx.y) * n + col] =
          (lds_[0][j] + lds_[1][j]) + (lds_[2][j] + lds_[3][j]);
  }
}

// out [n] = the column sums of parts [P][n], in order.
template <typename E>
__global__ void __launch_bounds__(1024) sums_kernel(int P, int n, const float* parts, E* out) {
  __shared__ float lds_[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), slot = threadIdx.x >> 6;
  float s = 0.0f;
  if (col < n)
#pragma unroll 4
    for (int p = slot; p < P; p += 16) s += parts[static_cast<int64_t>(p) * n + col];
  lds_[slot][threadIdx.x & 63] = s;
  __syncthreads();
  if (slot || col >= n) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += lds_[k][threadIdx.x];
  st(out, col, s);
}

// Row ranges of slope_kernel: workgroups that fill the card, each of 16 rows or more.
static int64_t slope_parts(int64_t rows, int64_t n, int size) {
  const int64_t across = (n + 1024 / size - 1) / (1024 / size);
  return std::max<int64_t>(1, std::min<int64_t>({2048 / across, (rows + 15) / 16, 512}));
}

}  // namespace linear
}  // namespace dabsn

using namespace dabsn;
using namespace dabsn::linear;

extern "C" {

size_t dabsn_hip_linear_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || (dtype != kF32 && dtype != kBF16)) return 0;
  const Plan p = plan_of(M, N, K, dtype == kF32 ? 4 : 2);
  return p.splits > 1 ? static_cast<size_t>(p.splits) * M * p.ldp * sizeof(float) : 0;
}

int dabsn_hip_linear(const dabsn_linear_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "linear: null call");
  const dabsn_linear_call& c = *call;
  DABSN_REQUIRE(c.dtype == kF32 || c.dtype == kBF16, "linear: bad dtype %d", c.dtype);
  const int64_t top = (1ll << 31) - 65536;
  DABSN_REQUIRE(c.M >= 0 && c.M < top && c.N > 0 && c.N < top && c.K >= 0 && c.K < top,
                "linear: bad shape M=%lld N=%lld K=%lld", (long long)c.M, (long long)c.N,
                (long long)c.K);
  DABSN_REQUIRE(c.lda >= (c.transA ? c.M : c.K) && c.ldb >= (c.transB ? c.N : c.K) && c.ldc >= c.N &&
                    (!c.residual || c.ldr >= c.N) && (!c.slope || c.lds >= c.N) && (!c.keep || c.ldk >= c.N),
                "linear: a row stride is shorter than its row");
  DABSN_REQUIRE(!c.transA || c.transB, "linear: transA goes with transB");
  DABSN_REQUIRE(c.act >= kNone && c.act <= kSilu, "linear: bad activation %d", c.act);
  DABSN_REQUIRE(!c.slope || c.slope_kind == kStored || c.slope_kind == kFromSquare,
                "linear: bad slope kind %d", c.slope_kind);
  if (c.M == 0) return DABSN_OK;
  DABSN_REQUIRE(c.C && (c.K == 0 || (c.A && c.B)), "linear: null pointer");
  const size_t need = dabsn_hip_linear_workspace_bytes(c.dtype, c.M, c.N, c.K);
  DABSN_REQUIRE(need == 0 || (c.workspace && c.workspace_bytes >= need),
                "linear: workspace of %zu bytes, %zu needed", c.workspace_bytes, need);
  return c.dtype == kF32 ? run<float>(c, stream) : run<bf16>(c, stream);
}

size_t dabsn_hip_linear_slope_workspace_bytes(int dtype, int64_t rows, int64_t n) {
  if (rows <= 0 || n <= 0 || (dtype != kF32 && dtype != kBF16)) return 0;
  return static_cast<size_t>(slope_parts(rows, n, dtype == kF32 ? 4 : 2)) * n * sizeof(float);
}

int dabsn_hip_linear_slope(int dtype, int64_t rows, int64_t n, const void* grad, int64_t ldg,
                           const void* slope, int64_t lds, int slope_kind, void* dz, int64_t ldz,
                           void* dbias, void* workspace, size_t workspace_bytes,
                           hipStream_t stream) {
  DABSN_REQUIRE(dtype == kF32 || dtype == kBF16, "linear slope: bad dtype %d", dtype);
  DABSN_REQUIRE(rows >= 0 && rows < (1ll << 31) && n > 0 && n < (1ll << 31) - 65536 && ldg >= n &&
                    (!slope || lds >= n) && (!dz || ldz >= n),
                "linear slope: bad shape rows=%lld n=%lld", (long long)rows, (long long)n);
  DABSN_REQUIRE(!slope || slope_kind == kStored || slope_kind == kFromSquare,
                "linear slope: bad slope kind %d", slope_kind);
  DABSN_REQUIRE(rows == 0 || grad, "linear slope: null pointer");
  float* parts = dbias ? static_cast<float*>(workspace) : nullptr;
  const size_t need = dabsn_hip_linear_slope_workspace_bytes(dtype, rows, n);
  DABSN_REQUIRE(!dbias || rows == 0 || (parts && workspace_bytes >= need),
                "linear slope: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!dz && !dbias) return DABSN_OK;
  const int size = dtype == kF32 ? 4 : 2;
  const int64_t P = rows ? slope_parts(rows, n, size) : 0;
  const int kind = slope ? slope_kind : kNoSlope;
  if (rows) {
    const dim3 grid((unsigned)((n + 1024 / size - 1) / (1024 / size)), (unsigned)P);
    if (dtype == kF32)
      hipLaunchKernelGGL(slope_kernel<float>, grid, dim3(256), 0, stream, rows, (int)n,
                         (const float*)grad, ldg, (const float*)slope, lds, kind, (float*)dz, ldz, parts);
    else
      hipLaunchKernelGGL(slope_kernel<bf16>, grid, dim3(256), 0, stream, rows, (int)n,
                         (const bf16*)grad, ldg, (const bf16*)slope, lds, kind, (bf16*)dz, ldz, parts);
    DABSN_HIP_CHECK(hipGetLastError());
  }
  if (dbias) {
    const dim3 grid((unsigned)((n + 63) / 64));
    if (dtype == kF32)
      hipLaunchKernelGGL(sums_kernel<float>, grid, dim3(1024), 0, stream, (int)P, (int)n, parts, (float*)dbias);
    else
      hipLaunchKernelGGL(sums_kernel<bf16>, grid, dim3(1024), 0, stream, (int)P, (int)n, parts, (bf16*)dbias);
    DABSN_HIP_CHECK(hipGetLastError());
  }
  return DABSN_OK;
}

}  // extern "C"
