// Matrix products with the work around them in their epilogue, for the block's MLP.
//
//   C(m, n) = act(sum_k A(m, k) B(n, k) + bias(n)) * slope(m, n) + residual(m, n)
//
// in fp32, rounded once to the type of A and B. An operand is K-contiguous, A[m * lda + k], or
// stored as its transpose, A[k * lda + m]: the forward needs neither transposed, the gradient of
// the rows has B = W transposed, that of the weight both. The products are bound by the matrix
// cores once there are a few hundred rows, by the weight's bytes below.
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
  const bf16 *A, *B;  // as they are, or as pack_kernel leaves them
  int64_t lda, ldb, planeA, planeB;
  const E* bias;
  int act;
  const E* slope;
  int64_t lds;
  int slope_kind;
  const E* residual;
  int64_t ldr;
  E* C;
  int64_t ldc;
  int padC;  // rows of C get zeros up to a multiple of 8
  E* keep;  // act'(z); NULL: not kept
  int64_t ldk;
  int mt, nt, splits, kper;
  float* parts;  // [splits][M][ldp]: the splits' sums, instead of C
  int64_t ldp;
};

// act(z) and its derivative. Where they are rounded to bf16, the hardware's exp and reciprocal do
// (2^-22 and 2^-23 of their values), and erfc(x) = exp(-x^2) erfcx(x) with erfcx as a polynomial in
// t = 1 / (1 + 0.46 x), a fit of our own for x >= 0 that is within 1.7e-5 of the value up to x = 60
// (2^-8 is a rounding's): 20 instructions instead of erfcf's 70.
template <typename E>
__device__ __forceinline__ float activate(int act, float z, float& slope) {
  constexpr bool low = sizeof(E) == 2;
  constexpr float LOG2E = 1.44269504088896341f;
  if (act == kRelu2) {
    const float r = z > 0.0f || z != z ? z : 0.0f;
    slope = 2.0f * r;
    return r * r;
  }
  if (act == kGelu) {
    float below, bell;  // the normal distribution function and exp(-z^2 / 2)
    if constexpr (low) {
      const float x = fabsf(z) * 0.70710678118654752f;
      const float t = __builtin_amdgcn_rcpf(fmaf(0.46f, x, 1.0f));
      float q = fmaf(-0.12698957f, t, 0.2432926f);
      q = fmaf(q, t, 0.12421153f);
      q = fmaf(q, t, 0.24096189f);
      q = fmaf(q, t, 0.25897348f);
      q = fmaf(q, t, 0.25953397f);
      bell = __builtin_amdgcn_exp2f(z * z * (-0.5f * LOG2E));
      const float tail = 0.5f * q * t * bell;
      below = z > 0.0f ? 1.0f - tail : tail;
    } else {
      below = 0.5f * erfcf(z * -0.70710678118654752f);
      bell = expf(-0.5f * z * z);
    }
    slope = fmaf(z * 0.39894228040143268f, bell, below);
    return z * below;
  }
  if (act == kSilu) {
    float s, rest;
    if constexpr (low) {
      s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * z));
      rest = 1.0f - s;
    } else {
      s = 1.0f / (1.0f + expf(-z));
      rest = 1.0f / (1.0f + expf(z));
    }
    slope = fmaf(z * s, rest, s);
    return z * s;
  }
  slope = 1.0f;
  return z;
}

__device__ __forceinline__ float factor(int kind, float s) {
  return kind == kFromSquare ? 2.0f * sqrtf(s) : s;
}

// Eight columns of a row, the first `left` of them within it, at any alignment.
template <typename E>
__device__ __forceinline__ void take(const E* p, int left, float (&v)[8]) {
  E raw[8];
  if (left >= 8) {
    __builtin_memcpy(raw, p, sizeof(raw));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) raw[e] = e < left ? p[e] : static_cast<E>(0);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = to_f(raw[e]);
}
template <typename E>
__device__ __forceinline__ void put(E* p, int left, const float (&v)[8]) {
  E raw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) raw[e] = from_f<E>(v[e]);
  if (left >= 8) {
    __builtin_memcpy(p, raw, sizeof(raw));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) p[e] = raw[e];
  }
}

// The epilogue of the sums v at row m, columns n to n + 7 (n < N a multiple of 8).
template <typename E>
__device__ __forceinline__ void finish(const Args<E>& a, int64_t m, int n, float (&v)[8],
                                       const float (&bias)[8]) {
  const int left = a.N - n;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += bias[e];
  if (a.act) {
    float slope[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = activate<E>(a.act, v[e], slope[e]);
    if (a.keep) put(a.keep + m * a.ldk + n, left, slope);
  }
  if (a.slope_kind) {
    float s[8];
    take(a.slope + m * a.lds + n, left, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= factor(a.slope_kind, s[e]);
  }
  if (a.residual) {
    float r[8];
    take(a.residual + m * a.ldr + n, left, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += r[e];
  }
  if (a.padC) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? v[e] : 0.0f;
    put(a.C + m * a.ldc + n, 8, v);
  } else {
    put(a.C + m * a.ldc + n, left, v);
  }
}
template <typename E>
__device__ __forceinline__ void bias_of(const Args<E>& a, int n, float (&b)[8]) {
  if (a.bias) {
    take(a.bias + n, a.N - n, b);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = 0.0f;
  }
}

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

// ---- the products -----------------------------------------------------------------------------
constexpr int PK = 64;
constexpr uint32_t NOWHERE = 0x80000000u;  // an offset beyond every buffer resource

// A tile's way into LDS, BT rows (or columns, where transposed) by PK k a step: 16-byte chunks in
// the order of their positions, K-contiguous rows of 128 bytes (eight lanes read a chunk of eight
// rows at once) or transposed rows of 2 BT bytes (32 lanes read 32 bytes of eight rows), positions
// permuted so that no bank is asked twice (by the counter of conflicts).
template <bool T, int BT, int NTH>
struct Feed {
  static constexpr int NV = BT * PK * 2 / 16 / NTH;
  static constexpr int CPR = T ? BT / 8 : 8, ROWS = NTH / CPR;
  static_assert(BT * PK * 2 % (16 * NTH) == 0 && NTH % CPR == 0 && ROWS % 8 == 0,
                "a thread's chunks lie ROWS rows apart");
  // Chunk i + 1 of a thread comes from the same columns as chunk i, or from 128 bytes on or back.
  static constexpr bool SWAP = T && ROWS % 16 == 8 && BT >= 128;
  const bf16* base;  // the tile's first element
  uint32_t bytes;    // from there to the matrix's end
  u32x4 rsrc;
  uint32_t off, stride;  // of the first chunk in this step, from chunk to chunk
  int32_t flip;  // 128 or -128
  int64_t ld;
  int k0, len;  // the first chunk's k, of `len`

  __host__ __device__ static constexpr int turn(int r) {
    const int f = (r & 3) | ((r >> 1) & 4);
    return BT >= 128 ? f : f >> 1;
  }
  __device__ void init(const bf16* p, int64_t ld_, int r0, int rows, int kbase, int len_, int tid) {
    ld = ld_;
    len = len_;
    base = T ? p + static_cast<int64_t>(kbase) * ld + r0 : p + static_cast<int64_t>(r0) * ld + kbase;
    // K-contiguous rows hold zeros up to a whole chunk.
    const int64_t last = T ? static_cast<int64_t>(len - 1) * ld + (rows - r0)
                           : static_cast<int64_t>(min(BT, rows - r0) - 1) * ld + (len + 7) / 8 * 8;
    bytes = static_cast<uint32_t>((last * 2 + 3) & ~3ll);
    const int r = tid / CPR, c = (tid % CPR) ^ (T ? turn(r) << 1 : r & 7);
    k0 = T ? r : c * 8;
    flip = c & 8 ? -128 : 128;
    off = static_cast<uint32_t>((r * ld + c * 8) * 2);
    stride = static_cast<uint32_t>(ROWS * ld * 2);
  }
  __device__ void plane(int64_t at) {
    const uint64_t p = reinterpret_cast<uint64_t>(base + at);
    rsrc = (u32x4){static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32) & 0xffffu, bytes, 0x00020000u};
  }
  // Where step t's chunks are. Transposed rows beyond the last k lie beyond the resource; of the
  // others' chunks those that start beyond it are sent there. Both load zeros.
  __device__ uint32_t place(int t) const {
    if constexpr (T) return off + static_cast<uint32_t>(t) * static_cast<uint32_t>(PK * ld * 2);
    return t * PK + k0 < len ? off + t * PK * 2 : NOWHERE;
  }
  // Chunk I of the step at `at` to LDS, I * NTH * 16 bytes from `lds` on. Written as assembly, since
  // before a transposing read the compiler would wait for every load under way; the kernel waits for
  // them itself. (They write no register.)
  template <int I>
  __device__ void load(uint32_t lds, uint32_t at) const {
    if constexpr (SWAP && I % 2 == 1) at += flip;
    uint32_t o;
    asm volatile("s_add_u32 m0, %1, %2\n\tv_add_u32 %0, %3, %4\n\tbuffer_load_dwordx4 %0, %5, 0 offen lds"
                 : "=&v"(o)
                 : "s"(lds), "n"(I * NTH * 16), "s"(I * stride), "v"(at), "s"(rsrc)
                 : "memory", "scc");
  }
};

// A wave's fragments: tile i of 16 rows from its first row on, half a step of 32 k, eight k a lane.
// Addresses are bytes of LDS; `at` is made anew for each half (the compiler would keep a register
// for every tile and buffer).
template <bool T, int BT>
struct Reader {
  uint32_t base;
  __device__ void init(uint32_t lds, int row, int lane) {
    const int li = lane & 15, g = lane >> 4, r = g * 8 + (li >> 2);
    base = lds + (T ? r * BT * 2 + ((row / 16) ^ Feed<true, BT, 512>::turn(r)) * 32 + (li & 3) * 8
                    : (row + li) * PK * 2 + (g ^ (li & 7)) * 16);
  }
  __device__ uint32_t at(int bytes, int half) const {
    uint32_t p = (T ? base + half * 32 * BT * 2 : base ^ (half * 64)) + bytes;
    asm volatile("" : "+v"(p));
    return p;
  }
  template <typename V>
  using Lds = __attribute__((address_space(3))) V*;
  __device__ static bf16x8 get(uint32_t at, int i) {
    if constexpr (!T) {
      return __builtin_bit_cast(bf16x8, *(Lds<const u32x4>)(at + i * 16 * PK * 2));
    } else {
      // Two transposing reads, each of four k by 16 columns per 16 lanes. (A wave's rows start at a
      // multiple of its tiles, so adding i to the tile's number is an exclusive or.)
      const uint32_t p = at ^ (i * 32);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds<s16x4>)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds<s16x4>)(p + 8 * BT));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// f(0), f(1), ... f(N - 1), each with its number as a constant.
template <int N, typename F>
__device__ __forceinline__ void each_of(F&& f) {
  if constexpr (N > 0) {
    each_of<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// c += a b. Of a wave that has a SIMD's 512 registers to itself, `PIN` keeps the sums in its
// accumulation registers (left to itself the compiler copies them to and fro). It does not see the
// waits that these need: settle() stands between other writes or reads of the sums and the products.
template <bool PIN>
__device__ __forceinline__ void mma(f32x4& c, bf16x8 a, bf16x8 b) {
  if constexpr (PIN) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <bool PIN>
__device__ __forceinline__ void settle() {
  if constexpr (PIN) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Steps of 64 k through two buffers in LDS, filled by loads that go there without registers, and two
// sets of fragments of 32 k each. A step's first half multiplies its first set while the second is
// read; its second half multiplies that one while the first set of the next step is read and the
// loads of the step after it go out, over the buffer just read. One barrier a step, between the
// halves: before it a wave waits until its own loads of the next step have landed (they had a step's
// time) and its reads have; after it, all of the next step is in LDS and this one's buffer is free.
//
// fp32 operands come as three bf16 planes each (x = hi + mid + lo, 8 bits each, the remainders
// exact): the steps then go through six products of planes, small ones first; the three left out
// are below 2^-24 of the product. At 2.5 PFLOP/s for bf16 against 0.16 for fp32 this is 2.6 times
// the fp32 instructions' rate.
template <typename E, bool TA, bool TB, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) product_kernel(Args<E> a, int nblk) {
  constexpr int NTH = WM * WN * 64, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int PAIRS = sizeof(E) == 4 ? 6 : 1;
  constexpr bool PIN = TM * TN == 64;
  using FA = Feed<TA, BM, NTH>;
  using FB = Feed<TB, BN, NTH>;
  __shared__ __attribute__((aligned(16))) bf16 lds[2][(BM + BN) * PK];

  int sp, mt, nt;
  if (!tile_of(blockIdx.x, nblk, a.splits, a.mt, a.nt, sp, mt, nt)) return;
  const int m0 = mt * BM, n0 = nt * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int k0 = sp * a.kper, len = min(a.K - k0, a.kper);
  const int each = (len + PK - 1) / PK, steps = PAIRS * each;

  FA fa;
  FB fb;
  fa.init(a.A, a.lda, m0, a.M, k0, len, tid);
  fb.init(a.B, a.ldb, n0, a.N, k0, len, tid);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  constexpr int BUF = (BM + BN) * PK * 2;
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) bf16*)lds[0]));
  // The loads' place: step `at` of the pair; steps beyond the last load zeros, without traffic.
  int pair = 0, at = 0;
  auto planes = [&]() __attribute__((always_inline)) {
    // (lo hi) (hi lo) (mid mid) (mid hi) (hi mid) (hi hi), the planes hi, mid, lo in this order.
    constexpr uint32_t PA = 0x001102, PB = 0x010120;
    fa.plane(PAIRS > 1 ? static_cast<int64_t>((PA >> (4 * pair)) & 3) * a.planeA : 0);
    fb.plane(PAIRS > 1 ? static_cast<int64_t>((PB >> (4 * pair)) & 3) * a.planeB : 0);
  };
  planes();
  uint32_t placeA = fa.place(0), placeB = fb.place(0);
  constexpr int LOADS = FA::NV + FB::NV;
  auto feed = [&](auto i, int buf) __attribute__((always_inline)) {
    constexpr int I = decltype(i)::value;
    const uint32_t to = lds0 + buf * BUF + wave * 1024;
    if constexpr (I < FA::NV) fa.template load<I>(to, placeA);
    else fb.template load<I - FA::NV>(to + BM * PK * 2, placeB);
  };
  auto fed = [&]() __attribute__((always_inline)) {
    ++at;
    if (PAIRS > 1 && at == each && pair + 1 < PAIRS) {
      at = 0;
      ++pair;
      planes();
    }
    placeA = fa.place(at);
    placeB = fb.place(at);
  };
  using RA = Reader<TA, BM>;
  using RB = Reader<TB, BN>;
  RA ra;
  RB rb;
  ra.init(lds0, wm, lane);
  rb.init(lds0 + BM * PK * 2, wn, lane);
  bf16x8 fra[2][TM], frb[2][TN];
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Multiplies set SET while the other is read from buffer BUFFER and, with GO, the next loads go to
  // the other buffer. A product takes the matrix unit 16 cycles and the wave 4, so the reads and loads
  // go between the products, one or two at a place, and the last quarter of the places stays free for
  // them to land.
  auto half = [&](auto set, auto buffer, auto go) __attribute__((always_inline)) {
    constexpr int SET = decltype(set)::value, BUFFER = decltype(buffer)::value;
    constexpr bool GO = decltype(go)::value;
    constexpr int ALL = TM * TN, READS = TM + TN, RSTEP = ALL * 3 / 4 / READS, LSTEP = ALL * 3 / 4 / LOADS;
    static_assert(RSTEP >= 1 && LSTEP >= 1, "places for all");
    const uint32_t pa = ra.at(BUFFER * BUF, SET ^ 1), pb = rb.at(BUFFER * BUF, SET ^ 1);
    each_of<ALL>([&](auto place) __attribute__((always_inline)) {
      constexpr int P = decltype(place)::value, I = P / TN, J = P % TN;
      mma<PIN>(acc[I][J], frb[SET][J], fra[SET][I]);
      if constexpr (P % RSTEP == 0 && P / RSTEP < READS) {
        constexpr int R = P / RSTEP;
        if constexpr (R < TN) frb[SET ^ 1][R] = RB::get(pb, R);
        else fra[SET ^ 1][R - TN] = RA::get(pa, R - TN);
      }
      if constexpr (GO && P % LSTEP == LSTEP / 2 && P / LSTEP < LOADS)
        feed(std::integral_constant<int, P / LSTEP>{}, BUFFER ^ 1);
      if constexpr (PIN) __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (!PIN) __builtin_amdgcn_sched_barrier(0);
    if constexpr (GO) fed();
  };
  using N0 = std::integral_constant<int, 0>;
  using N1 = std::integral_constant<int, 1>;
  each_of<LOADS>([&](auto i) __attribute__((always_inline)) { feed(i, 0); });
  fed();
  meet();
  each_of<LOADS>([&](auto i) __attribute__((always_inline)) { feed(i, 1); });
  fed();
  {
    const uint32_t pa = ra.at(0, 0), pb = rb.at(0, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) frb[0][j] = RB::get(pb, j);
#pragma unroll
    for (int i = 0; i < TM; ++i) fra[0][i] = RA::get(pa, i);
  }
  auto step = [&](auto buffer) __attribute__((always_inline)) {
    using Next = std::integral_constant<int, decltype(buffer)::value ^ 1>;
    half(N0{}, buffer, std::false_type{});
    meet();
    half(N1{}, Next{}, std::true_type{});
  };
  settle<PIN>();
  int t = 0;
  for (; t + 2 <= steps; t += 2) {
    step(N0{});
    step(N1{});
  }
  if (t < steps) step(N0{});
  // No load may land after the workgroup has gone, nor in the epilogue's places.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  settle<PIN>();
  __syncthreads();

  // B is the instruction's first operand: a lane holds four consecutive columns of a row. A wave
  // turns HR rows at a time in its own part of LDS, positions of 16 bytes permuted by the row, and
  // takes them back as eight columns a lane: whole lines for every access of the epilogue, and its
  // code once.
  constexpr int CW = TN * 16, HT = TM < 4 ? TM : 4, HR = HT * 16, LPR = CW / 8, RPP = 64 / LPR;
  static_assert(sizeof(lds) >= static_cast<size_t>(WM * WN) * HR * CW * 4, "LDS holds the waves' parts");
  float* mine = reinterpret_cast<float*>(lds) + wave * HR * CW;
  const int n = n0 + wn + lane % LPR * 8, row = lane / LPR;
  float bias[8];
  if (n < a.N && !a.parts) bias_of(a, n, bias);
#pragma unroll
  for (int h = 0; h < TM / HT; ++h) {
#pragma unroll
    for (int i = 0; i < HT; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int r = i * 16 + (lane & 15), c = j * 4 + (lane >> 4);
        *reinterpret_cast<f32x4*>(mine + r * CW + (c ^ (r & (CW / 4 - 1))) * 4) = acc[h * HT + i][j];
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
    for (int p = 0; p < HR; p += RPP) {
      const int r = p + row, m = m0 + wm + h * HR + r;
      if (m >= a.M || n >= a.N) continue;
      const int c = lane % LPR * 2, x = r & (CW / 4 - 1);
      const f32x4 lo = *reinterpret_cast<const f32x4*>(mine + r * CW + (c ^ x) * 4);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(mine + r * CW + ((c + 1) ^ x) * 4);
      if (a.parts) {
        f32x4* q = reinterpret_cast<f32x4*>(a.parts + (static_cast<int64_t>(sp) * a.M + m) * a.ldp + n);
        q[0] = lo;
        q[1] = hi;
      } else {
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        finish(a, m, n, v, bias);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// An operand [rows][cols] of row stride ld as the products read it: rows of `to` values (a multiple
// of 8) that end in zeros; fp32 as its planes hi, mid, lo, each [rows][to].
template <typename E>
__global__ void __launch_bounds__(256) pack_kernel(int64_t rows, int cols, const E* x, int64_t ld,
                                                   int to, bf16* out, int64_t plane) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, per = to / 8;
  if (i >= rows * per) return;
  const int64_t r = i / per;
  const int c = static_cast<int>(i % per) * 8;
  const E* p = x + r * ld + c;
  E v[8];
  if (c + 8 <= cols) {
    __builtin_memcpy(v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? p[e] : static_cast<E>(0);
  }
  bf16* o = out + r * to + c;
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

// The splits' sums in order, then the epilogue: a thread eight columns.
template <typename E>
__global__ void __launch_bounds__(256) join_kernel(Args<E> a) {
  const int64_t per = a.ldp / 8, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= per * a.M) return;
  const int64_t m = i / per;
  const int n = static_cast<int>(i % per) * 8;
  float v[8] = {}, bias[8];
  bias_of(a, n, bias);
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.parts + (s * static_cast<int64_t>(a.M) + m) * a.ldp + n;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += lo[e];
      v[4 + e] += hi[e];
    }
  }
  finish(a, m, n, v, bias);
}

// How a product runs.
struct Plan {
  bool packA, packB;
  int64_t lda, ldb, planeA, planeB;  // of the operands the kernel reads
  bool big;                          // tiles of 256 x 256, else 128 x 128
  int mt, nt, splits, kper;
  int64_t ldp;
  size_t atB, atParts, bytes;  // places in the workspace, which starts with A
};

static size_t up16(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// bf16 operands are read where they lie if their chunks of 16 bytes are aligned and whole.
static bool ready(const void* p, int64_t ld, bool trans, int64_t K, bool padded) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && (trans || padded || K % 8 == 0);
}

static Plan plan_of(const dabsn_linear_call& c) {
  Plan p = {};
  const bool f32 = c.dtype == kF32;
  p.packA = f32 || !ready(c.A, c.lda, c.transA, c.K, c.padA);
  p.packB = f32 || !ready(c.B, c.ldb, c.transB, c.K, c.padB);
  const int64_t rowsA = c.transA ? c.K : c.M, rowsB = c.transB ? c.K : c.N;
  p.lda = p.packA ? ((c.transA ? c.M : c.K) + 7) / 8 * 8 : c.lda;
  p.ldb = p.packB ? ((c.transB ? c.N : c.K) + 7) / 8 * 8 : c.ldb;
  p.planeA = p.packA ? rowsA * p.lda : 0;
  p.planeB = p.packB ? rowsB * p.ldb : 0;
  size_t at = p.packA ? up16(static_cast<size_t>(p.planeA) * (f32 ? 6 : 2)) : 0;
  p.atB = at;
  at += p.packB ? up16(static_cast<size_t>(p.planeB) * (f32 ? 6 : 2)) : 0;
  p.atParts = at;
  const int64_t big = ((c.M + 255) / 256) * ((c.N + 255) / 256);
  p.big = big >= 192;
  const int64_t edge = p.big ? 256 : 128;
  p.mt = static_cast<int>((c.M + edge - 1) / edge);
  p.nt = static_cast<int>((c.N + edge - 1) / edge);
  const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt, steps = (c.K + PK - 1) / PK;
  const int64_t room = p.big ? 256 : 512;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({room / tiles, steps * (f32 ? 6 : 1) / 16, 64}));
  // Offsets of a transposed operand's rows are 32 bits.
  const int64_t ld = std::max<int64_t>(c.transA ? p.lda : 0, c.transB ? p.ldb : 0);
  if (ld) splits = std::max<int64_t>(splits, (c.K * ld * 2 + (1ll << 30) - 1) >> 30);
  const int64_t each = std::max<int64_t>(1, (steps + splits - 1) / splits);
  p.splits = static_cast<int>(std::max<int64_t>(1, (steps + each - 1) / each));
  p.kper = static_cast<int>(each * PK);
  p.ldp = (c.N + 7) / 8 * 8;
  if (p.splits > 1) at += static_cast<size_t>(p.splits) * c.M * p.ldp * sizeof(float);
  p.bytes = at;
  return p;
}

template <typename E>
static int pack(int64_t rows, int64_t cols, const void* x, int64_t ld, int64_t to, bf16* out,
                hipStream_t s) {
  const int64_t blocks = (rows * (to / 8) + 255) / 256;
  DABSN_REQUIRE(blocks < (1ll << 31), "linear: an operand of too many elements");
  hipLaunchKernelGGL(pack_kernel<E>, dim3((unsigned)blocks), dim3(256), 0, s, rows, (int)cols,
                     (const E*)x, ld, (int)to, out, rows * to);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

template <typename E>
static int run(const dabsn_linear_call& c, const Plan& p, hipStream_t s) {
  Args<E> a = {};
  a.M = (int)c.M; a.N = (int)c.N; a.K = (int)c.K;
  char* ws = static_cast<char*>(c.workspace);
  a.A = p.packA ? (const bf16*)ws : (const bf16*)c.A;
  a.B = p.packB ? (const bf16*)(ws + p.atB) : (const bf16*)c.B;
  a.lda = p.lda; a.ldb = p.ldb; a.planeA = p.planeA; a.planeB = p.planeB;
  a.bias = (const E*)c.bias; a.act = c.act;
  a.slope = (const E*)c.slope; a.lds = c.lds; a.slope_kind = c.slope ? c.slope_kind : kNoSlope;
  a.residual = (const E*)c.residual; a.ldr = c.ldr;
  a.C = (E*)c.C; a.ldc = c.ldc; a.keep = (E*)c.keep; a.ldk = c.ldk; a.padC = c.padC;
  a.mt = p.mt; a.nt = p.nt; a.splits = c.K ? p.splits : 0; a.kper = p.kper; a.ldp = p.ldp;
  a.parts = p.splits > 1 ? (float*)(ws + p.atParts) : nullptr;
  if (c.K) {
    int rc = DABSN_OK;
    if (p.packA) rc = pack<E>(c.transA ? c.K : c.M, c.transA ? c.M : c.K, c.A, c.lda, p.lda, (bf16*)ws, s);
    if (rc == DABSN_OK && p.packB)
      rc = pack<E>(c.transB ? c.K : c.N, c.transB ? c.N : c.K, c.B, c.ldb, p.ldb, (bf16*)(ws + p.atB), s);
    if (rc != DABSN_OK) return rc;
    const int64_t tiles = static_cast<int64_t>(p.mt) * p.nt * p.splits;
    DABSN_REQUIRE(tiles < (1ll << 31) - 8, "linear: too many tiles");
    const int nblk = (int)((tiles + 7) / 8 * 8);
#define L(TA, TB)                                                                                     \
  if (p.big)                                                                                          \
    hipLaunchKernelGGL((product_kernel<E, TA, TB, 256, 256, 2, 2>), dim3(nblk), dim3(256), 0, s, a, nblk); \
  else                                                                                                \
    hipLaunchKernelGGL((product_kernel<E, TA, TB, 128, 128, 2, 2>), dim3(nblk), dim3(256), 0, s, a, nblk)
    if (c.transA) { L(true, true); }
    else if (c.transB) { L(false, true); }
    else { L(false, false); }
#undef L
    DABSN_HIP_CHECK(hipGetLastError());
  }
  if (a.parts || !c.K) {
    const int64_t blocks = (p.ldp / 8 * c.M + 255) / 256;
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
  // dz's rows end in zeros up to a multiple of 8 where their stride has the room.
  const int pad = (n + 7) / 8 * 8 <= ldz ? (n + 7) / 8 * 8 : n;
  if (c < pad) {
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
            if (c + e < n || c + e < pad) dz[r * ldz + c + e] = o[e];  // o is 0 beyond n
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
  const int64_t top = (1ll << 31) - 65536, width = 1 << 22;
  DABSN_REQUIRE(c.M >= 0 && c.M < top && c.N > 0 && c.N < top && c.K >= 0 && c.K < top,
                "linear: bad shape M=%lld N=%lld K=%lld", (long long)c.M, (long long)c.N,
                (long long)c.K);
  DABSN_REQUIRE(!c.transA || c.transB, "linear: transA goes with transB");
  DABSN_REQUIRE(c.lda >= (c.transA ? c.M : c.K) && c.ldb >= (c.transB ? c.N : c.K) && c.ldc >= c.N &&
                    (!c.residual || c.ldr >= c.N) && (!c.slope || c.lds >= c.N) &&
                    (!c.keep || c.ldk >= c.N),
                "linear: a row stride is shorter than its row");
  // 256 rows of an operand lie within 32-bit offsets.
  DABSN_REQUIRE(c.lda < width && c.ldb < width, "linear: operands have rows of at most %lld elements",
                (long long)width - 1);
  DABSN_REQUIRE(c.act >= kNone && c.act <= kSilu && !(c.keep && c.act == kNone),
                "linear: bad activation %d", c.act);
  DABSN_REQUIRE(!c.slope || c.slope_kind == kStored || c.slope_kind == kFromSquare,
                "linear: bad slope kind %d", c.slope_kind);
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
    const dim3 grid((unsigned)(((n + 7) / 8 * 8 + 1024 / size - 1) / (1024 / size)), (unsigned)P);
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
