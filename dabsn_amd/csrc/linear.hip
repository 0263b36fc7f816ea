// The products of linear.hpp: how each runs, its operands' packing, the join of its splits, and the
// C ABI; the activations' slopes.
#include "linear.hpp"

#include "capi.hpp"

namespace dabsn {
namespace linear {

// Instantiated in linear_forward_*.hip and linear_gradients_*.hip.
#define DABSN_LINEAR(E, EPI, TA, TB) \
  extern template void launch<E, EPI, TA, TB>(const Args<E>&, int, int, hipStream_t)
#define DABSN_LINEAR_ALL(E)             \
  DABSN_LINEAR(E, kNone, false, false); \
  DABSN_LINEAR(E, kRelu2, false, false); \
  DABSN_LINEAR(E, kGelu, false, false); \
  DABSN_LINEAR(E, kSilu, false, false); \
  DABSN_LINEAR(E, kShare, false, false); \
  DABSN_LINEAR(E, kNone, false, true);  \
  DABSN_LINEAR(E, kShare, false, true); \
  DABSN_LINEAR(E, kShare, true, true);  \
  DABSN_LINEAR(E, kStored, false, true); \
  DABSN_LINEAR(E, kFromSquare, false, true); \
  DABSN_LINEAR(E, kNone, true, true)
DABSN_LINEAR_ALL(float);
DABSN_LINEAR_ALL(bf16);

// An operand [rows][cols] of row stride ld as the products read it: rows of `to` values (a multiple
// of 8) that end in zeros; fp32 as its planes hi, mid, lo, each [rows][to].
template <typename E>
struct Operand {
  int64_t rows;
  int cols, to;
  const E* x;
  int64_t ld;
  bf16* out;
  __host__ __device__ int64_t chunks() const { return rows * (to / 8); }
};
// One operand or both, a thread eight values. Bound by HBM: 1001 columns of 3001 and 777 rows fp32
// 9.5 us.
template <typename E>
__global__ void __launch_bounds__(256) pack_kernel(Operand<E> p, Operand<E> other) {
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.chunks()) {
    i -= p.chunks();
    p = other;
    if (i >= p.chunks()) return;
  }
  const int per = p.to / 8;
  const int64_t r = i / per, plane = p.rows * p.to;
  const int c = static_cast<int>(i - r * per) * 8;
  const E* at = p.x + r * p.ld + c;
  E v[8];
  if (c + 8 <= p.cols) {
    __builtin_memcpy(v, at, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < p.cols ? at[e] : static_cast<E>(0);
  }
  bf16* o = p.out + r * p.to + c;
  if constexpr (sizeof(E) == 2) {
    __builtin_memcpy(o, v, 16);
  } else {
    bf16 part[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float rest = v[e];
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        bf16 h = f2bf(rest);
        // A number that rounds to infinity is cut instead.
        if ((h & 0x7fff) == 0x7f80 && fabsf(rest) < INFINITY)
          h = static_cast<bf16>(__builtin_bit_cast(uint32_t, rest) >> 16);
        part[k][e] = h;
        rest = fabsf(rest) < INFINITY ? rest - bf2f(h) : 0.0f;  // infinity and NaN are in hi alone
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) __builtin_memcpy(o + k * plane, part[k], 16);
  }
}

// The splits' sums in order, then the epilogue: a thread eight columns. Bound by the parts' way from
// L2: 3001 x 777 fp32 of two splits 13 us, 256 x 2048 of four 4 us.
template <typename E, int EPI>
__global__ void __launch_bounds__(256) join_kernel(Args<E> a) {
  const int64_t per = a.ldp / 8, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= per * a.M) return;
  const int64_t m = i / per;
  const int n = static_cast<int>(i % per) * 8;
  float v[8] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.parts + (s * static_cast<int64_t>(a.M) + m) * a.ldp + n;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += lo[e];
      v[4 + e] += hi[e];
    }
  }
  if (n + 8 > a.N) {
#pragma unroll
    for (int e = 0; e < 8; ++e) finish_one<E, EPI>(a, m, n + e, v[e]);
    return;
  }
  Eight<E> x;
  if (a.bias) {
    __builtin_memcpy(&x, a.bias + n, sizeof(x));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x.get(e);
  }
  float kept[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = activate<E, EPI>(v[e], kept[e]);
  if (a.keep) {
    x.template set<HALF<E, EPI>>(kept);
    __builtin_memcpy(a.keep + m * a.ldk + n, &x, sizeof(x));
  }
  if (a.beside) {
    __builtin_memcpy(&x, a.beside + m * a.ldr + n, sizeof(x));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (EPI == kStored || EPI == kFromSquare) v[e] *= factor<E, EPI>(x.template get<HALF<E, EPI>>(e));
      else v[e] += x.get(e);
    }
  }
  x.set(v);
  __builtin_memcpy(a.C + m * a.ldc + n, &x, sizeof(x));
}

// How a product runs.
struct Plan {
  bool packA, packB;
  int64_t lda, ldb, planeA, planeB;  // of the operands the kernel reads
  int tile;
  int mt, nt, splits, kper;
  int64_t ldp;
  size_t atB, atParts, bytes;  // places in the workspace, which starts with A
};

static size_t up16(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// bf16 operands are read where they lie if their chunks of 16 bytes are aligned and whole.
static bool ready(const void* p, int64_t ld, bool trans, int64_t K, bool padded) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && (trans || padded || K % 8 == 0);
}

// The tile and the splits of K are those that take least by these times in us, as measured:
//   256 x 256   1.41 a step of 64 k for all units (8192^3), six times as many steps for fp32
//   128 x 128   0.55 a step with one tile a unit, 0.9 with two
//   deep        the operands' way from L2, 100 KB/us a unit, but at least 0.2 a step
//   direct      2.3 a step of 32 k (128 x 128; 0.62 for 64 x 64, but 0.9) for each tile of a unit
//   besides     4 to 7 a round of tiles; packing 4 and its bytes at 4.5 TB/s; joining splits 6 and
//               their bytes at 7 TB/s
static Plan plan_of(const dabsn_linear_call& c) {
  Plan p = {};
  if (c.M <= 16 && !c.transB && c.K > 0) {
    p.tile = kRows;
    p.splits = 1;
    p.lda = c.lda;
    p.ldb = c.ldb;
    return p;
  }
  const bool f32 = c.dtype == kF32;
  const bool packA = f32 || !ready(c.A, c.lda, c.transA, c.K, c.padA);
  const bool packB = f32 || !ready(c.B, c.ldb, c.transB, c.K, false);
  const int64_t rowsA = c.transA ? c.K : c.M, rowsB = c.transB ? c.K : c.N;
  const int64_t wideA = ((c.transA ? c.M : c.K) + 7) / 8 * 8, wideB = ((c.transB ? c.N : c.K) + 7) / 8 * 8;
  const int64_t lda = packA ? wideA : c.lda, ldb = packB ? wideB : c.ldb;
  p.ldp = (c.N + 7) / 8 * 8;
  const double values = (packA ? 1.0 * rowsA * wideA : 0) + (packB ? 1.0 * rowsB * wideB : 0);
  const double pack = values ? 4 + values * (f32 ? 10 : 4) / 4.5e6 : 0;
  // A transposed operand's rows of a split lie within 2^30 bytes.
  const int64_t ld = std::max<int64_t>(c.transA ? lda : 0, c.transB ? ldb : 0);
  const int64_t least = std::max<int64_t>(1, (c.K * ld * 2 + (1ll << 30) - 1) >> 30);
  double best = 0;
  for (int tile = kBig; tile <= kDirectLow; ++tile) {
    const bool deep = tile == kDeep || tile == kDeepLow, direct = tile >= kDirect;
    if ((deep && (f32 || c.transB)) || (direct && !f32)) continue;
    const TileOf size = tile_size(tile);
    const int64_t mt = (c.M + size.m - 1) / size.m, nt = (c.N + size.n - 1) / size.n;
    const int64_t deepness = direct ? 32 : PK, steps = (c.K + deepness - 1) / deepness;
    const int64_t times = f32 && !direct ? 6 : 1;
    for (int64_t want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256}) {
      if (want > 1 && (want > steps || want < least)) continue;
      const int64_t splits = direct ? want : std::max(want, least);
      const int64_t each = std::max<int64_t>(1, (steps + splits - 1) / splits);
      const int64_t real = std::max<int64_t>(1, (steps + each - 1) / each), wgs = mt * nt * real;
      const int64_t rounds = (wgs + 255) / 256;
      double us = direct ? 0 : pack;
      if (tile == kBig) us += rounds * (each * times * 1.41 + 7);
      else if (tile == kMiddle)
        us += (wgs <= 256 ? each * times * 0.55 : (rounds + 1) / 2 * (each * times * 0.9)) + 4;
      else if (deep) us += rounds * (each * std::max(0.2, (size.m + size.n) * PK * 2 / 100e3) + 4);
      else if (tile == kDirect) us += rounds * each * 2.3 + 4;
      else us += each * std::max(0.9, rounds * 0.62) + 4;
      if (real > 1) us += 6 + (8.0 * real * c.M * p.ldp) / 7e6;
      if (best == 0 || us < best) {
        best = us;
        p.tile = tile;
        p.mt = static_cast<int>(mt);
        p.nt = static_cast<int>(nt);
        p.splits = static_cast<int>(real);
        p.kper = static_cast<int>(each * deepness);
      }
    }
  }
  const bool direct = p.tile >= kDirect;
  p.packA = packA && !direct;
  p.packB = packB && !direct;
  p.lda = p.packA ? lda : c.lda;
  p.ldb = p.packB ? ldb : c.ldb;
  p.planeA = p.packA ? rowsA * p.lda : 0;
  p.planeB = p.packB ? rowsB * p.ldb : 0;
  p.atB = p.packA ? up16(static_cast<size_t>(p.planeA) * (f32 ? 6 : 2)) : 0;
  p.atParts = p.atB + (p.packB ? up16(static_cast<size_t>(p.planeB) * (f32 ? 6 : 2)) : 0);
  p.bytes = p.atParts + (p.splits > 1 ? static_cast<size_t>(p.splits) * c.M * p.ldp * sizeof(float) : 0);
  return p;
}

template <typename F>
static void with_activation(const dabsn_linear_call& c, F&& f) {
  if (c.act == kRelu2) f(std::integral_constant<int, kRelu2>{});
  else if (c.act == kGelu) f(std::integral_constant<int, kGelu>{});
  else if (c.act == kSilu) f(std::integral_constant<int, kSilu>{});
  else f(std::integral_constant<int, kNone>{});
}
template <typename F>
static void with_factor(const dabsn_linear_call& c, F&& f) {
  if (!c.slope) f(std::integral_constant<int, kNone>{});
  else if (c.slope_kind == 1) f(std::integral_constant<int, kStored>{});
  else f(std::integral_constant<int, kFromSquare>{});
}

template <typename E>
static int run(const dabsn_linear_call& c, const Plan& p, hipStream_t s) {
  Args<E> a = {};
  a.M = (int)c.M; a.N = (int)c.N; a.K = (int)c.K;
  char* ws = static_cast<char*>(c.workspace);
  a.A = p.packA ? (const bf16*)ws : (const bf16*)c.A;
  a.B = p.packB ? (const bf16*)(ws + p.atB) : (const bf16*)c.B;
  a.lda = p.lda; a.ldb = p.ldb; a.planeA = p.planeA; a.planeB = p.planeB;
  a.bias = (const E*)c.bias;
  a.beside = (const E*)(c.slope ? c.slope : c.residual);
  a.ldr = c.slope ? c.lds : c.ldr;
  a.C = (E*)c.C; a.ldc = c.ldc; a.keep = (E*)c.keep; a.ldk = c.ldk; a.padC = c.padC;
  a.mt = p.mt; a.nt = p.nt; a.splits = c.K ? p.splits : 0; a.kper = p.kper; a.ldp = p.ldp;
  a.wholeA = (const E*)c.A; a.wholelda = c.lda;
  a.wholeB = (const E*)c.B; a.wholeldb = c.ldb;
  a.parts = p.splits > 1 ? (float*)(ws + p.atParts) : nullptr;
  const bool wide = c.wideC && c.K && p.splits == 1;  // the only share is the result
  if (wide) {
    a.parts = (float*)c.C;
    a.ldp = c.ldc;
  }
  if (c.K) {
    Operand<E> pa = {}, pb = {};
    if (p.packA)
      pa = {c.transA ? c.K : c.M, (int)(c.transA ? c.M : c.K), (int)p.lda, (const E*)c.A, c.lda, (bf16*)ws};
    if (p.packB)
      pb = {c.transB ? c.K : c.N, (int)(c.transB ? c.N : c.K), (int)p.ldb, (const E*)c.B, c.ldb,
            (bf16*)(ws + p.atB)};
    const int64_t blocks = (pa.chunks() + pb.chunks() + 255) / 256;
    DABSN_REQUIRE(blocks < (1ll << 31), "linear: operands of too many elements");
    if (blocks)
      hipLaunchKernelGGL(pack_kernel<E>, dim3((unsigned)blocks), dim3(256), 0, s, pa, pb);
    DABSN_HIP_CHECK(hipGetLastError());
    const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt * p.splits;
    DABSN_REQUIRE(tiles < (1ll << 31) - 8, "linear: too many tiles");
    const int nblk = (int)((tiles + 7) / 8 * 8);
    // The products the MLP has: activations go with the forward, factors with the rows' gradient.
    if (a.parts) {
      if (c.transA) launch<E, kShare, true, true>(a, p.tile, nblk, s);
      else if (c.transB) launch<E, kShare, false, true>(a, p.tile, nblk, s);
      else launch<E, kShare, false, false>(a, p.tile, nblk, s);
    } else if (c.transA) launch<E, kNone, true, true>(a, p.tile, nblk, s);
    else if (c.transB) with_factor(c, [&](auto epi) { launch<E, decltype(epi)::value, false, true>(a, p.tile, nblk, s); });
    else with_activation(c, [&](auto epi) { launch<E, decltype(epi)::value, false, false>(a, p.tile, nblk, s); });
    DABSN_HIP_CHECK(hipGetLastError());
  }
  if ((a.parts && !wide) || !c.K) {
    const int64_t blocks = (p.ldp / 8 * c.M + 255) / 256;
    DABSN_REQUIRE(blocks < (1ll << 31), "linear: too many elements to join");
    auto join = [&](auto epi) {
      hipLaunchKernelGGL((join_kernel<E, decltype(epi)::value>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    };
    if (c.wideC) {
      Args<float> f = {};
      f.M = a.M; f.N = a.N; f.splits = a.splits; f.parts = a.parts; f.ldp = a.ldp;
      f.C = (float*)c.C; f.ldc = c.ldc; f.padC = 1;
      hipLaunchKernelGGL((join_kernel<float, kNone>), dim3((unsigned)blocks), dim3(256), 0, s, f);
    } else if (c.slope) with_factor(c, join);
    else with_activation(c, join);
    DABSN_HIP_CHECK(hipGetLastError());
  }
  return DABSN_OK;
}

// Sixteen bytes of a row. H: fp16 in bf16's place.
template <typename E>
struct Piece {
  static constexpr int VEC = 16 / static_cast<int>(sizeof(E));
  u32x4 q;
  __device__ __forceinline__ void load(const E* p, int left) {
    if (left >= VEC) {
      __builtin_memcpy(&q, p, 16);
    } else {
      E e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = i < left ? p[i] : static_cast<E>(0);
      __builtin_memcpy(&q, e, 16);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    if constexpr (sizeof(E) == 4) {
      __builtin_memcpy(&q, v, 16);
    } else {
      Eight<E> all;
      all.set(v);
      q = all.q[0];
    }
  }
  template <bool H = false>
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w = q[sizeof(E) == 4 ? e : e / 2];
    if constexpr (sizeof(E) == 4) return __builtin_bit_cast(float, w);
    else if constexpr (H) return from_half(static_cast<uint16_t>(e % 2 ? w >> 16 : w));
    else return __builtin_bit_cast(float, e % 2 ? w & 0xffff0000u : w << 16);
  }
};

// dz = g * slope (NULL: not written; KIND kNone: no slope) and partial column sums of it (NULL: none)
// over a range of rows each. A workgroup takes 64 lanes by VEC columns and every fourth row of its
// range, four a wave at once and as many on their way. Bound by HBM: 8192 x 8192 bf16 with slope and
// sums 80 us, 5.1 TB/s, a copy's rate (101 with one set of rows; 121 with both sets as 16-bit values).
template <typename E, int KIND>
__global__ void __launch_bounds__(256) slope_kernel(int64_t rows, int n, const E* g, int64_t ldg,
                                                    const E* s, int64_t lds, E* dz, int64_t ldz,
                                                    float* parts) {
  constexpr int VEC = Piece<E>::VEC, U = 4;
  __shared__ float lds_[4][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * VEC;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = std::min(rows, r0 + per);
  float sum[VEC] = {};
  // dz's rows end in zeros up to a multiple of 8 where their stride has the room.
  const int pad = (n + 7) / 8 * 8 <= ldz ? (n + 7) / 8 * 8 : n;
  if (c < pad) {
    Piece<E> nextg[U], nexts[U];
    const auto fetch = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = r + 4 * u;
        if (row >= r1) break;
        nextg[u].load(g + row * ldg + c, n - c);
        if constexpr (KIND != kNone) nexts[u].load(s + row * lds + c, n - c);
      }
    };
    fetch(r0 + wave);
    for (int64_t r = r0 + wave; r < r1; r += 4 * U) {
      Piece<E> nowg[U], nows[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        nowg[u] = nextg[u];
        nows[u] = nexts[u];
      }
      fetch(r + 4 * U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = r + 4 * u;
        if (row >= r1) break;
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[e] = nowg[u].get(e);
          if constexpr (KIND != kNone) v[e] *= factor<E, KIND>(nows[u].template get<HALF<E, KIND>>(e));
          sum[e] += v[e];
        }
        if (!dz) continue;
        Piece<E> done;
        done.set(v);
        if (c + VEC <= n) {
          __builtin_memcpy(dz + row * ldz + c, &done, 16);
        } else {
          E o[VEC];
          __builtin_memcpy(o, &done, 16);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (c + e < n || c + e < pad) dz[row * ldz + c + e] = o[e];  // o is 0 beyond n
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

static int check_linear(const dabsn_linear_call& c) {
  DABSN_REQUIRE(c.dtype == kF32 || c.dtype == kBF16, "linear: bad dtype %d", c.dtype);
  const int64_t top = (1ll << 31) - 65536, width = 1 << 21;
  DABSN_REQUIRE(c.M >= 0 && c.M < top && c.N > 0 && c.N < top && c.K >= 0 && c.K < top,
                "linear: bad shape M=%lld N=%lld K=%lld", (long long)c.M, (long long)c.N,
                (long long)c.K);
  DABSN_REQUIRE(!c.transA || c.transB, "linear: transA goes with transB");
  DABSN_REQUIRE(c.lda >= (c.transA ? c.M : c.K) && c.ldb >= (c.transB ? c.N : c.K) && c.ldc >= c.N &&
                    (!c.residual || c.ldr >= c.N) && (!c.slope || c.lds >= c.N) &&
                    (!c.keep || c.ldk >= c.N),
                "linear: a row stride is shorter than its row");
  // 256 rows of any matrix lie within 31-bit offsets.
  DABSN_REQUIRE(c.lda < width && c.ldb < width && c.ldc < width && (!c.residual || c.ldr < width) &&
                    (!c.slope || c.lds < width) && (!c.keep || c.ldk < width),
                "linear: rows of at most %lld elements", (long long)width - 1);
  DABSN_REQUIRE(c.act >= kNone && c.act <= kSilu && !(c.keep && c.act == kNone),
                "linear: bad activation %d", c.act);
  DABSN_REQUIRE(!c.slope || c.slope_kind == 1 || c.slope_kind == 2, "linear: bad slope kind %d",
                c.slope_kind);
  // Activations, bias and residual belong to the forward, a slope to the rows' gradient.
  DABSN_REQUIRE(!c.transB || (c.act == kNone && !c.bias && !c.residual),
                "linear: no activation, bias or residual with transB");
  DABSN_REQUIRE(!c.slope || (c.transB && !c.transA), "linear: a slope goes with transB alone");
  DABSN_REQUIRE(!c.wideC || (c.dtype == kBF16 && c.transB && !c.transA && !c.slope && c.ldc % 8 == 0),
                "linear: a wide C goes with bf16, transB alone, no slope and rows of a multiple of 8");
  return DABSN_OK;
}

extern "C" {

size_t dabsn_hip_linear_workspace_bytes(const dabsn_linear_call* call) {
  if (!call || call->M <= 0 || check_linear(*call) != DABSN_OK) return 0;
  return plan_of(*call).bytes;
}

int dabsn_hip_linear(const dabsn_linear_call* call, hipStream_t stream) {
  DABSN_REQUIRE(call, "linear: null call");
  const dabsn_linear_call& c = *call;
  const int rc = check_linear(c);
  if (rc != DABSN_OK || c.M == 0) return rc;
  DABSN_REQUIRE(c.C && (c.K == 0 || (c.A && c.B)), "linear: null pointer");
  const Plan p = plan_of(c);
  DABSN_REQUIRE(p.bytes == 0 || (c.workspace && c.workspace_bytes >= p.bytes &&
                                 (reinterpret_cast<uintptr_t>(c.workspace) & 15u) == 0),
                "linear: workspace of %zu bytes, %zu needed", c.workspace_bytes, p.bytes);
  return c.dtype == kF32 ? run<float>(c, p, stream) : run<bf16>(c, p, stream);
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
  DABSN_REQUIRE(!slope || slope_kind == 1 || slope_kind == 2,
                "linear slope: bad slope kind %d", slope_kind);
  DABSN_REQUIRE(rows == 0 || grad, "linear slope: null pointer");
  float* parts = dbias ? static_cast<float*>(workspace) : nullptr;
  const size_t need = dabsn_hip_linear_slope_workspace_bytes(dtype, rows, n);
  DABSN_REQUIRE(!dbias || rows == 0 || (parts && workspace_bytes >= need),
                "linear slope: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!dz && !dbias) return DABSN_OK;
  const int size = dtype == kF32 ? 4 : 2;
  const int64_t P = rows ? slope_parts(rows, n, size) : 0;
  if (rows) {
    const dim3 grid((unsigned)(((n + 7) / 8 * 8 + 1024 / size - 1) / (1024 / size)), (unsigned)P);
    const auto launch = [&](auto kernel, auto zero) {
      using E = decltype(zero);
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, rows, (int)n, (const E*)grad, ldg,
                         (const E*)slope, lds, (E*)dz, ldz, parts);
    };
    if (dtype == kF32)
      launch(!slope ? slope_kernel<float, kNone> : slope_kind == 1 ? slope_kernel<float, kStored>
                                                                   : slope_kernel<float, kFromSquare>, 0.0f);
    else
      launch(!slope ? slope_kernel<bf16, kNone> : slope_kind == 1 ? slope_kernel<bf16, kStored>
                                                                  : slope_kernel<bf16, kFromSquare>, bf16());
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
