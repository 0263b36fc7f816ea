// Matrix products with the work around them in their epilogue, for the block's MLP.
//
//   C(m, n) = act(sum_k A(m, k) B(n, k) + bias(n)) + residual(m, n)   or   sum * slope(m, n)
//
// in fp32, rounded once to the type of A and B. An operand is K-contiguous, A[m * lda + k], or
// stored as its transpose, A[k * lda + m]: the forward needs neither transposed, the gradient of
// the rows has B = W transposed, that of the weight both. The products are bound by the matrix
// cores once there are a few hundred rows, by the weight's bytes below.
#pragma once

#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace dabsn {
namespace linear {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// What the epilogue does with the sums: an activation (and then the residual is added), or a factor:
// a stored slope, or the squared ReLU's output h, whose slope is 2 sqrt(h).
// Or it leaves them as a split's share.
enum Epi : int { kNone = 0, kRelu2 = 1, kGelu = 2, kSilu = 3, kStored = 4, kFromSquare = 5, kShare = 6 };

template <typename E>
struct Args {
  int M, N, K;
  const bf16 *A, *B;  // as they are, or as pack_kernel leaves them
  int64_t lda, ldb, planeA, planeB;
  const E* bias;
  const E* beside;  // the residual or the factor
  int64_t ldr;
  E* C;
  int64_t ldc;
  int padC;  // rows of C get zeros up to a multiple of 8
  E* keep;  // what the backward needs of the activation; NULL: not kept
  int64_t ldk;
  int mt, nt, splits, kper;
  float* parts;  // [splits][M][ldp]: the splits' sums, instead of C
  int64_t ldp;
  const E *wholeA, *wholeB;  // as they are
  int64_t wholelda, wholeldb;
};

// act(z), and what is kept for its derivative: of the squared ReLU the value itself (before a residual;
// a rounding of it is half of one in the slope 2 sqrt(h)), else the derivative. With bf16 operands
// that is stored as its 2^14-fold in fp16: derivatives of GELU and SiLU lie in [-0.13, 1.13], so that
// none overflows and each is off by 2^-11 of itself or 2^-39, an eighth of bf16's step at the same
// bytes. (By itself, without the factor, all below 2^-25 would be 0, and the gradients of rows that
// lie there whole.)
// Where they are rounded to bf16, the hardware's exp and reciprocal do
// (2^-22 and 2^-23 of their values), and erfc(x) = exp(-x^2) erfcx(x) with erfcx as a polynomial in
// t = 1 / (1 + 0.43 x), a fit of our own for 0 <= x <= 10 (the exp is 0 from 9.4 on) that is within 1.4e-7
// of the value, 3.8e-7 as evaluated: 22 instructions instead of erfcf's 70. A coarser one would not do:
// a residual may cancel the value, and the slope passes 0.
template <typename E, int EPI>
__device__ __forceinline__ float activate(float z, float& kept) {
  constexpr bool low = sizeof(E) == 2;
  constexpr float LOG2E = 1.44269504088896341f;
  if constexpr (EPI == kRelu2) {
    const float r = z < 0.0f ? 0.0f : z;  // a NaN stays
    return kept = r * r;
  }
  if constexpr (EPI == kGelu) {
    float below, bell;  // the normal distribution function and exp(-z^2 / 2)
    if constexpr (low) {
      const float x = fabsf(z) * 0.70710678118654752f;
      const float t = __builtin_amdgcn_rcpf(fmaf(0.43f, x, 1.0f));
      float q = fmaf(0.072948128f, t, -0.307316899f);
      q = fmaf(q, t, 0.378633231f);
      q = fmaf(q, t, -0.0812397078f);
      q = fmaf(q, t, 0.244568408f);
      q = fmaf(q, t, 0.205611885f);
      q = fmaf(q, t, 0.24427399f);
      q = fmaf(q, t, 0.242520958f);
      bell = __builtin_amdgcn_exp2f(z * z * (-0.5f * LOG2E));
      const float tail = 0.5f * q * t * bell;
      below = z > 0.0f ? 1.0f - tail : tail;
    } else {
      below = 0.5f * erfcf(z * -0.70710678118654752f);
      bell = expf(-0.5f * z * z);
    }
    kept = fmaf(z * 0.39894228040143268f, bell, below);
    return z * below;
  }
  if constexpr (EPI == kSilu) {
    float s, rest;
    if constexpr (low) {
      s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * z));
      rest = 1.0f - s;
    } else {
      s = 1.0f / (1.0f + expf(-z));
      rest = 1.0f / (1.0f + expf(z));
    }
    kept = fmaf(z * s, rest, s);
    return z * s;
  }
  kept = 1.0f;
  return z;
}

// (The hardware's root is off by 2^-23 of itself, which a factor of bf16 values does not see.)
template <typename E, int EPI>
__device__ __forceinline__ float factor(float s) {
  if constexpr (EPI != kFromSquare) return s;
  return 2.0f * (sizeof(E) == 2 ? __builtin_amdgcn_sqrtf(s) : sqrtf(s));
}

// Whether a derivative is kept for GELU and SiLU or read: fp16 in bf16's place.
template <typename E, int EPI>
constexpr bool HALF = sizeof(E) == 2 && (EPI == kGelu || EPI == kSilu || EPI == kStored);
constexpr float HALF_UNIT = 0x1p14f;  // 1 as it is stored so
__device__ __forceinline__ float from_half(uint16_t h) {
  return static_cast<float>(__builtin_bit_cast(_Float16, h)) * (1.0f / HALF_UNIT);
}

// Eight columns of a row as they are stored; with H as fp16 in bf16's place.
template <typename E>
struct Eight {
  static constexpr int Q = sizeof(E) / 2;
  u32x4 q[Q];
  template <bool H = false>
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w = q[sizeof(E) == 4 ? e / 4 : 0][sizeof(E) == 4 ? e % 4 : e / 2];
    // (A bit cast of the vector's element itself would take its first.)
    if constexpr (sizeof(E) == 4) return __builtin_bit_cast(float, w);
    else if constexpr (H) return from_half(static_cast<uint16_t>(e % 2 ? w >> 16 : w));
    else return __builtin_bit_cast(float, e % 2 ? w & 0xffff0000u : w << 16);
  }
  template <bool H = false>
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e / 4][e % 4] = __builtin_bit_cast(uint32_t, v[e]);
    } else {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      typedef std::conditional_t<H, _Float16, __bf16> low __attribute__((ext_vector_type(2)));
      constexpr float unit = H ? HALF_UNIT : 1.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[0][i] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector(((f32x2){v[2 * i] * unit, v[2 * i + 1] * unit}), low));
    }
  }
};

// A tile's rows of a matrix, for accesses of eight columns at any alignment. The resource ends with the
// matrix's last row, so rows beyond it are neither read (zeros) nor written; columns beyond their
// row are sent to NOWHERE. No branch: between branches the compiler would wait for every store.
constexpr uint32_t NOWHERE = 0x80000000u;  // an offset beyond every buffer resource
template <typename E>
struct Rows {
  __amdgpu_buffer_rsrc_t rsrc;
  uint32_t at, step;  // of the lane's row in the first 16, from 16 rows to the next
  __device__ __forceinline__ void init(const E* p, int64_t ld, int m0, int n0, int rows, int cols, int row) {
    const int64_t size = p ? ((rows - 1) * ld + cols) * static_cast<int64_t>(sizeof(E)) : 0;
    rsrc = make_rsrc(p + m0 * ld + n0, static_cast<uint32_t>(size));
    at = static_cast<uint32_t>(row * ld * sizeof(E));
    step = static_cast<uint32_t>(16 * ld * sizeof(E));
  }
  __device__ __forceinline__ Eight<E> take(int block, uint32_t column) const {
    Eight<E> v;
#pragma unroll
    for (int i = 0; i < Eight<E>::Q; ++i)
      v.q[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + block * step + column + 16 * i, 0, 0);
    return v;
  }
  __device__ __forceinline__ void put(int block, uint32_t column, const Eight<E>& v) const {
#pragma unroll
    for (int i = 0; i < Eight<E>::Q; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(v.q[i], rsrc, at + block * step + column + 16 * i, 0, 0);
  }
};

template <typename E, int EPI>
__device__ __forceinline__ float beside_of(const E* p, int64_t i) {
  if constexpr (HALF<E, EPI>) return from_half(p[i]);
  else return ld(p, i);
}

// The same for one column, or for the zeros beyond the row's end.
template <typename E, int EPI>
__device__ __forceinline__ void finish_one(const Args<E>& a, int64_t m, int n, float v) {
  E* out = a.C + m * a.ldc + n;
  if (n >= a.N) {
    if (a.padC) *out = static_cast<E>(0);
    return;
  }
  float kept;
  if (a.bias) v += ld(a.bias, n);
  v = activate<E, EPI>(v, kept);
  if (a.keep) {
    if constexpr (HALF<E, EPI>) a.keep[m * a.ldk + n] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(kept * HALF_UNIT));
    else st(a.keep, m * a.ldk + n, kept);
  }
  if constexpr (EPI == kStored || EPI == kFromSquare) {
    st(out, 0, v * factor<E, EPI>(beside_of<E, EPI>(a.beside, m * a.ldr + n)));
  } else {
    st(out, 0, a.beside ? v + ld(a.beside, m * a.ldr + n) : v);
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
                 : "memory", "scc", "m0");
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
// Lane groups of 16: a's odd ones for b's even ones.
__device__ __forceinline__ void trade(float (&a)[4], float (&b)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const auto both = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a[r]),
                                                       __builtin_bit_cast(uint32_t, b[r]), false, false);
    const uint32_t first = both[0], second = both[1];
    a[r] = __builtin_bit_cast(float, first);
    b[r] = __builtin_bit_cast(float, second);
  }
}
template <bool PIN>
__device__ __forceinline__ float value(float sum) {
  if constexpr (!PIN) return sum;
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(sum));  // volatile: behind settle()
  return v;
}
template <bool PIN>
__device__ __forceinline__ void settle() {
  if constexpr (PIN) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The epilogue of a wave's TM x TN tiles of 16 x 16 sums. It goes by places of two by two tiles, whose
// operands it loads ahead of all its stores, since a load waits for the stores before it: those of
// FIRST places before the products, those of the next up to AHEAD places after them, into registers that
// held fragments.
template <typename E, int EPI, int TM, int TN, int BM, int BN, int NTH, bool PIN>
struct Epilogue {
  static constexpr int PLACES = TM * TN / 4;
  static constexpr bool WIDE = sizeof(E) == 2;
  static constexpr int AHEAD = PIN ? (WIDE ? 16 : 10) : PLACES;
  static constexpr int FIRST = std::min(PLACES, PIN ? (WIDE ? 12 : 6) : WIDE ? 2 : 1);
  static constexpr bool FACTOR = EPI == kStored || EPI == kFromSquare;
  static constexpr bool ACTS = EPI == kRelu2 || EPI == kGelu || EPI == kSilu;
  const Args<E>& a;
  const int sp, m0, n0, wm, wn, lane;  // the split, the tile's first element, the wave's in it
  const int rows, cols;                // of the tile within the matrix
  uint32_t column[TN / 2];             // in bytes from the tile's first
  Rows<E> besides;
  Eight<E> beside[AHEAD][2];
  float marked = 0.0f;  // NaN once a sum is not finite

  __device__ __forceinline__ Epilogue(const Args<E>& args, int sp_, int m0_, int n0_, int wm_, int wn_, int tid)
      : a(args), sp(sp_), m0(m0_), n0(n0_), wm(wm_), wn(wn_), lane(tid & 63),
        rows(min(BM, args.M - m0_)), cols(min(BN, args.N - n0_)) {}

  template <int P>
  __device__ __forceinline__ void fetch() {
    constexpr int R = P / (TN / 2) * 2;
    beside[P % AHEAD][0] = besides.take(R, column[P % (TN / 2)]);
    beside[P % AHEAD][1] = besides.take(R + 1, column[P % (TN / 2)]);
  }
  // Before the products; `bias_lds` [BN] is seen after the next barrier.
  __device__ __forceinline__ void begin(float* bias_lds, int tid) {
    const int li = lane & 15, group = lane >> 4;
#pragma unroll
    for (int q = 0; q < TN / 2; ++q) {
      const int c = wn + (q * 2 + group % 2) * 16 + group / 2 * 8;
      column[q] = c + 8 <= cols ? c * static_cast<uint32_t>(sizeof(E)) : NOWHERE;
    }
    if constexpr (EPI != kShare) {
      besides.init(a.beside, a.ldr, m0, n0, rows, cols, wm + li);
      for (int c = tid; c < BN; c += NTH) bias_lds[c] = a.bias && c < cols ? ld(a.bias, n0 + c) : 0.0f;
      if (a.beside)
        each_of<FIRST>([&](auto i) __attribute__((always_inline)) { fetch<decltype(i)::value>(); });
    }
  }
  // After them; no wave may still read the fragments' LDS, which `left` takes (8 floats a row).
  __device__ __forceinline__ void end(f32x4 (&acc)[TM][TN], const float* bias_lds, float* left) {
    const int li = lane & 15, group = lane >> 4;
    if constexpr (EPI != kShare)
      if (a.beside)
        each_of<AHEAD - FIRST>(
            [&](auto i) __attribute__((always_inline)) { fetch<decltype(i)::value + FIRST>(); });
    // A row's last columns, if they are fewer than eight, are left in LDS and done afterwards.
    const int rest = cols & ~7;
    const bool ragged = EPI != kShare && rest < cols;
    if (ragged) __syncthreads();
    Rows<E> out, keep;
    Rows<float> share;
    if constexpr (EPI == kShare) {
      share.init(a.parts + static_cast<int64_t>(sp) * a.M * a.ldp, a.ldp, m0, n0, rows,
                 static_cast<int>(min<int64_t>(BN, a.ldp - n0)), wm + li);
    } else {
      out.init(a.C, a.ldc, m0, n0, rows, cols, wm + li);
      if constexpr (ACTS) keep.init(a.keep, a.ldk, m0, n0, rows, cols, wm + li);
    }

    // B is the instruction's first operand: of tile (i, j) lane group g = lane / 16 holds columns 4 g
    // to 4 g + 3 of row lane % 16. Two exchanges of lane groups among two by two tiles, group 2 h + 1
    // of one register for group 2 h of the other, give each lane eight columns of a row: 64 bytes
    // (bf16) of 16 rows an access. (Through LDS instead this took 5 us more a tile of 256 x 256.)
    each_of<PLACES>([&](auto place) __attribute__((always_inline)) {
      constexpr int P = decltype(place)::value, I = P / (TN / 2) * 2, Q = P % (TN / 2), J = Q * 2;
      float x[2][2][4];  // [tile row][tile column]
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[0][j][r] = value<PIN>(acc[I][J + j][r]);
          x[1][j][r] = value<PIN>(acc[I + 1][J + j][r]);
        }
        trade(x[0][j], x[1][j]);
      }
      trade(x[0][0], x[0][1]);
      trade(x[1][0], x[1][1]);
      const int c = wn + (J + group % 2) * 16 + group / 2 * 8;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = x[e / 4][b][e % 4];
        if constexpr (!WIDE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) marked = fmaf(v[e], 0.0f, marked);
        }
        if constexpr (EPI == kShare) {
          Eight<float> all;
          all.set(v);
          share.put(I + b, c < static_cast<int>(a.ldp - n0) ? c * 4u : NOWHERE, all);
          continue;
        }
        if (ragged) {
          if (c == rest) {
            f32x4* q = reinterpret_cast<f32x4*>(left + (I * 16 + b * 16 + li) * 8);
            q[0] = (f32x4){v[0], v[1], v[2], v[3]};
            q[1] = (f32x4){v[4], v[5], v[6], v[7]};
          }
        }
        if (a.bias) {
          const f32x4 lo = *reinterpret_cast<const f32x4*>(bias_lds + c);
          const f32x4 hi = *reinterpret_cast<const f32x4*>(bias_lds + c + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] += lo[e];
            v[4 + e] += hi[e];
          }
        }
        Eight<E> done;
        if constexpr (ACTS) {
          float kept[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = activate<E, EPI>(v[e], kept[e]);
          if (a.keep) {
            done.template set<HALF<E, EPI>>(kept);
            keep.put(I + b, column[Q], done);
          }
        }
        if constexpr (FACTOR) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= factor<E, EPI>(beside[P % AHEAD][b].template get<HALF<E, EPI>>(e));
        } else if (a.beside) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += beside[P % AHEAD][b].get(e);
        }
        done.set(v);
        out.put(I + b, column[Q], done);
      }
      if constexpr (EPI != kShare && P + AHEAD < PLACES)
        if (a.beside) fetch<P + AHEAD>();
      __builtin_amdgcn_sched_barrier(0);
    });
    if (ragged && rest >= wn && rest < wn + TN * 16) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
      for (int r = lane; r < TM * 16; r += 64)
#pragma unroll 1
        for (int e = 0; e < 8; ++e)
          if (wm + r < rows) finish_one<E, EPI>(a, m0 + wm + r, n0 + rest + e, left[r * 8 + e]);
    }
  }
  // Of planes' products: an infinity meets the other operand's smaller planes too, which may be 0 or
  // of the other sign, and so leaves NaN where the product itself is infinite. Where a sum was not
  // finite, results that are NaN are formed anew from the operands as they lie, k0 to k0 + len, by
  // blocks of 64 x 64 with fp32 matrix instructions: 4096 x 2048 x 4096 with an infinite column of A,
  // which leaves no finite result, 1.33 ms, without it 0.32 (57 ms when a lane formed one result at a time).
  template <bool TA, bool TB>
  __device__ __forceinline__ void mend(int k0, int len) {
    static_assert(TM % 4 == 0 && TN % 4 == 0, "a wave has blocks of 64 x 64");
    if (!__any(marked != marked)) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const float *A = reinterpret_cast<const float*>(a.wholeA) + (TA ? k0 * a.wholelda + m0 : m0 * a.wholelda + k0);
    const float *B = reinterpret_cast<const float*>(a.wholeB) + (TB ? k0 * a.wholeldb + n0 : n0 * a.wholeldb + k0);
    const int li = lane & 15, group = lane >> 4;
    const auto place = [&](int r, int c) __attribute__((always_inline)) {
      return EPI == kShare ? a.parts + (static_cast<int64_t>(sp) * a.M + m0 + r) * a.ldp + n0 + c
                           : reinterpret_cast<float*>(a.C) + static_cast<int64_t>(m0 + r) * a.ldc + n0 + c;
    };
    const auto is_nan = [](const float* at) __attribute__((always_inline)) {
      const float old = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return old != old;
    };
#pragma unroll 1
    for (int block = 0; block < TM * TN / 16; ++block) {
      const int r0 = wm + block / (TN / 4) * 64, c0 = wn + block % (TN / 4) * 64;
      bool bad = false;
      if (c0 + lane < cols)
#pragma unroll 1
        for (int r = r0; r < min(r0 + 64, rows); ++r) bad |= is_nan(place(r, c0 + lane));
      if (!__any(bad)) continue;
      f32x4 c[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) c[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      // Four k of a row (or, where transposed, of a column), zeros beyond an edge.
      const auto take = [&](auto trans, const float* p, int64_t ld, int row, int end, int k) __attribute__((always_inline)) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (row < end) {
          if constexpr (decltype(trans)::value) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k + e < len) v[e] = p[(k + e) * ld + row];
          } else if (k + 4 <= len) {
            __builtin_memcpy(&v, p + row * ld + k, 16);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k + e < len) v[e] = p[row * ld + k + e];
          }
        }
        return v;
      };
#pragma unroll 1
      for (int k = 0; k < len; k += 16) {
        f32x4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = take(std::bool_constant<TA>{}, A, a.wholelda, r0 + i * 16 + li, rows, k + group * 4);
          y[i] = take(std::bool_constant<TB>{}, B, a.wholeldb, c0 + i * 16 + li, cols, k + group * 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              c[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[j][e], x[i][e], c[i][j], 0, 0, 0);
      }
      // The sums go where the NaN are, and from there, by the lane that left them, through the epilogue.
      uint64_t left = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = r0 + i * 16 + li, col = c0 + j * 16 + group * 4 + e;
            if (r >= rows || col >= cols || !is_nan(place(r, col))) continue;
            *place(r, col) = c[i][j][e];
            left |= 1ull << (i * 16 + j * 4 + e);
          }
      if constexpr (EPI != kShare)
#pragma unroll 1
        for (; left; left &= left - 1) {
          const int at = __builtin_ctzll(left), r = r0 + at / 16 * 16 + li, col = c0 + at / 4 % 4 * 16 + group * 4 + at % 4;
          finish_one<E, EPI>(a, m0 + r, n0 + col, *place(r, col));
        }
    }
  }
};

// Steps of 64 k through BUFS buffers in LDS, filled by loads that go there without registers, and two
// sets of fragments of 32 k each. A step's first half multiplies its first set while the second is
// read; its second half multiplies that one while the first set of the next step is read and the
// loads of step t + BUFS go out, over the buffer just read. One barrier a step, between the halves:
// before it a wave waits until its own loads of the next step have landed (they had BUFS - 1 steps'
// time) and its reads have; after it, all of the next step is in LDS and this one's buffer is free.
//
// fp32 operands come as three bf16 planes each (x = hi + mid + lo, 8 bits each, the remainders
// exact): the steps then go through six products of planes, small ones first; the three left out
// are below 2^-24 of the product. By the peaks, 2.5 PFLOP/s for bf16 against 0.16 for fp32, this is 2.6
// times the fp32 instructions' rate; at the clocks that the power allows it is 1.4 to 1.5 times.
//
// Bound by the matrix cores at the clock that the power allows. bf16: 8192^3 722 us, 1520 TFLOP/s;
// 65536 x 2048 x 8192 1660 us, its rows' gradient 1550 to 1570, its weight's 1460 to 1520. fp32:
// 8192 x 2048 x 8192 1180 to 1270 us, 215 to 233 TFLOP/s. Deep tiles are bound by their operands'
// way from L2: 256 x 2048 x 8192 13.8 us (22.7 with 128 x 128).
template <typename E, int EPI, bool TA, bool TB, int BM, int BN, int WM, int WN, int BUFS>
__global__ void __launch_bounds__(WM * WN * 64, BM * BN == 128 * 128 ? 2 : 1) product_kernel(Args<E> a, int nblk) {
  constexpr int NTH = WM * WN * 64, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int PAIRS = sizeof(E) == 4 ? 6 : 1;
  constexpr bool PIN = TM * TN == 64;
  using FA = Feed<TA, BM, NTH>;
  using FB = Feed<TB, BN, NTH>;
  __shared__ __attribute__((aligned(16))) bf16 lds[BUFS][(BM + BN) * PK];
  __shared__ __attribute__((aligned(16))) float bias_lds[BN];

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
  // All but the loads of the last LATER steps have landed, and all reads.
  auto meet = [&](auto later) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(later)::value * LOADS) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  static_assert((BUFS - 1) * LOADS < 64, "the counter of loads has six bits");
  // Multiplies set SET while the other is read from buffer BUFFER and, with TO >= 0, the next loads go to
  // buffer TO. A product takes the matrix unit 16 cycles and the wave 4, so the reads and loads
  // go between the products, one or two at a place: the reads over three quarters of them, to be back
  // at the end, the loads over all (8192^3, all three forms: 3% faster than over three quarters).
  auto half = [&](auto set, auto buffer, auto target) __attribute__((always_inline)) {
    constexpr int SET = decltype(set)::value, BUFFER = decltype(buffer)::value, TO = decltype(target)::value;
    constexpr int ALL = TM * TN, READS = TM + TN;
    constexpr int RSTEP = std::max(1, ALL * 3 / 4 / READS), LSTEP = std::max(1, ALL / LOADS);
    static_assert(READS <= ALL && LOADS <= ALL, "places for all");
    const uint32_t pa = ra.at(BUFFER * BUF, SET ^ 1), pb = rb.at(BUFFER * BUF, SET ^ 1);
    each_of<ALL>([&](auto place) __attribute__((always_inline)) {
      constexpr int P = decltype(place)::value, I = P / TN, J = P % TN;
      mma<PIN>(acc[I][J], frb[SET][J], fra[SET][I]);
      if constexpr (P % RSTEP == 0 && P / RSTEP < READS) {
        constexpr int R = P / RSTEP;
        if constexpr (R < TN) frb[SET ^ 1][R] = RB::get(pb, R);
        else fra[SET ^ 1][R - TN] = RA::get(pa, R - TN);
      }
      if constexpr (TO >= 0 && P % LSTEP == LSTEP / 2 && P / LSTEP < LOADS)
        feed(std::integral_constant<int, P / LSTEP>{}, TO);
      if constexpr (PIN) __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (!PIN) __builtin_amdgcn_sched_barrier(0);
    if constexpr (TO >= 0) fed();
  };
  using N0 = std::integral_constant<int, 0>;
  using N1 = std::integral_constant<int, 1>;
  Epilogue<E, EPI, TM, TN, BM, BN, NTH, PIN> epilogue(a, sp, m0, n0, wm, wn, tid);
  epilogue.begin(bias_lds, tid);
  each_of<BUFS>([&](auto buf) __attribute__((always_inline)) {
    each_of<LOADS>([&](auto i) __attribute__((always_inline)) { feed(i, decltype(buf)::value); });
    fed();
  });
  meet(std::integral_constant<int, BUFS - 1>{});
  {
    const uint32_t pa = ra.at(0, 0), pb = rb.at(0, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) frb[0][j] = RB::get(pb, j);
#pragma unroll
    for (int i = 0; i < TM; ++i) fra[0][i] = RA::get(pa, i);
  }
  auto step = [&](auto buffer) __attribute__((always_inline)) {
    using Next = std::integral_constant<int, (decltype(buffer)::value + 1) % BUFS>;
    half(N0{}, buffer, std::integral_constant<int, -1>{});
    meet(std::integral_constant<int, BUFS - 2>{});
    half(N1{}, Next{}, buffer);
  };
  settle<PIN>();
  int t = 0;
  for (; t + BUFS <= steps; t += BUFS) each_of<BUFS>(step);
  each_of<BUFS - 1>([&](auto buffer) __attribute__((always_inline)) {
    if (t + decltype(buffer)::value < steps) step(buffer);
  });
  // No load may land after the workgroup has gone.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  settle<PIN>();
  epilogue.end(acc, bias_lds, reinterpret_cast<float*>(lds) + wave * (BM / WM) * 8);
  if constexpr (PAIRS > 1) epilogue.template mend<TA, TB>(k0, len);
}

// fp32 operands as they lie, at any alignment, by fp32 matrix instructions: where splitting them into
// planes would take longer than it saves (few products a value, small calls). Four waves a tile; steps
// of 32 k through two buffers: step t's products while step t + 1 goes from registers to LDS and step
// t + 2 comes to registers. K-contiguous rows are 128 bytes, read as in product_kernel; transposed rows
// are read 16 columns at a time by four rows. 2048 x 256 x 1024: 14.5 us (23 with planes); 3001 x 777 x
// 1001 65 us, 72 TFLOP/s of the instruction's 154.
template <bool T, int BT>
struct Stage {
  static constexpr int COLS = T ? BT : 32, ROWS = T ? 32 : BT, CPR = COLS / 4, NV = ROWS * CPR / 256;
  static_assert(ROWS * CPR % 256 == 0, "staging must divide evenly");
  u32x4 v[NV];
  __device__ static int pos(int c, int r) { return T ? c ^ (((r >> 2) & 3) << 2) : c ^ (r & 7); }
  // The tile at row r0, column c0 of a matrix of `rows` x `cols`, zeros beyond.
  __device__ __forceinline__ void load(const float* p, int64_t ld, int r0, int c0, int rows, int cols, int tid) {
    const bool inside = r0 + ROWS <= rows && c0 + COLS <= cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = tid + i * 256, r = r0 + q / CPR, c = c0 + q % CPR * 4;
      const float* at = p + static_cast<int64_t>(r) * ld + c;
      if (inside || (r < rows && c + 4 <= cols)) {
        __builtin_memcpy(&v[i], at, 16);
      } else {
        float raw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = r < rows && c + e < cols ? at[e] : 0.0f;
        __builtin_memcpy(&v[i], raw, 16);
      }
    }
  }
  __device__ __forceinline__ void store(float* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = tid + i * 256, r = q / CPR;
      *reinterpret_cast<u32x4*>(lds + r * COLS + pos(q % CPR, r) * 4) = v[i];
    }
  }
  // Rows row0 + (lane & 15), k = ks * 16 + (lane >> 4) * 4 + 0..3: four instructions of four k each,
  // one element of every lane group at a time.
  __device__ static f32x4 get(const float* lds, int row0, int ks, int lane) {
    const int li = lane & 15, g = lane >> 4;
    if constexpr (!T) {
      return *reinterpret_cast<const f32x4*>(lds + (row0 + li) * 32 + ((ks * 4 + g) ^ (li & 7)) * 4);
    } else {
      const float* at = lds + (ks * 16 + g * 4) * BT + ((row0 >> 4) ^ g) * 16 + li;
      return (f32x4){at[0], at[BT], at[2 * BT], at[3 * BT]};
    }
  }
};

template <int EPI, bool TA, bool TB, int BT>
__global__ void __launch_bounds__(256, 2) direct_kernel(Args<float> a, int nblk) {
  constexpr int TT = BT / 32;  // tiles of 16 a wave's edge
  using SA = Stage<TA, BT>;
  using SB = Stage<TB, BT>;
  __shared__ __attribute__((aligned(16))) float ldsA[2][BT * 32], ldsB[2][BT * 32];
  __shared__ __attribute__((aligned(16))) float bias_lds[BT];
  int sp, mt, nt;
  if (!tile_of(blockIdx.x, nblk, a.splits, a.mt, a.nt, sp, mt, nt)) return;
  const int m0 = mt * BT, n0 = nt * BT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / 2 * (BT / 2), wn = wave % 2 * (BT / 2);
  const int k0 = sp * a.kper, kend = min(a.K, k0 + a.kper), steps = (kend - k0 + 31) / 32;
  const float* A = reinterpret_cast<const float*>(a.A);
  const float* B = reinterpret_cast<const float*>(a.B);
  f32x4 acc[TT][TT];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  Epilogue<float, EPI, TT, TT, BT, BT, 256, false> epilogue(a, sp, m0, n0, wm, wn, tid);
  epilogue.begin(bias_lds, tid);
  SA va;
  SB vb;
  auto load = [&](int t) __attribute__((always_inline)) {
    const int k = k0 + t * 32;
    if constexpr (TA) va.load(A, a.lda, k, m0, kend, a.M, tid);
    else va.load(A, a.lda, m0, k, a.M, kend, tid);
    if constexpr (TB) vb.load(B, a.ldb, k, n0, kend, a.N, tid);
    else vb.load(B, a.ldb, n0, k, a.N, kend, tid);
  };
  load(0);
  va.store(ldsA[0], tid);
  vb.store(ldsB[0], tid);
  if (steps > 1) load(1);
  __syncthreads();
  for (int t = 0; t < steps; ++t) {
    const int buf = t & 1;
    if (t + 1 < steps) {
      va.store(ldsA[buf ^ 1], tid);  // released by the barrier that ended step t - 1
      vb.store(ldsB[buf ^ 1], tid);
      if (t + 2 < steps) load(t + 2);
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      f32x4 fa[TT];
#pragma unroll
      for (int i = 0; i < TT; ++i) fa[i] = SA::get(ldsA[buf], wm + i * 16, ks, lane);
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        const f32x4 fb = SB::get(ldsB[buf], wn + j * 16, ks, lane);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < TT; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[e], fa[i][e], acc[i][j], 0, 0, 0);
      }
    }
    __syncthreads();
  }
  epilogue.end(acc, bias_lds, ldsA[0] + wave * (BT / 2) * 8);
}

// Up to 16 rows: bound by the way of B, which is read once, straight to registers at any alignment. A
// workgroup has WAVES waves and TN tiles of 16 columns; the waves take every WAVES-th block of BK k
// (128 bytes of each of B's rows), UNROLL blocks of loads at a time, and their sums meet in LDS in
// order. Rows of A beyond M are not read (zeros). 1 x 2048 x 8192 bf16: 6.9 us, 4.9 TB/s (8.7 by the
// tiles).
template <typename E, int EPI, int TN, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) rows_kernel(Args<E> a, const E* A, const E* B) {
  constexpr int VEC = 16 / sizeof(E), BK = 128 / sizeof(E), UNROLL = 4 / TN;
  __shared__ __attribute__((aligned(16))) float sums[WAVES][TN][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * TN;
  f32x4 acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const E* pa = A + static_cast<int64_t>(min(li, a.M - 1)) * a.lda + g * VEC;
  const E* pb[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j)
    pb[j] = B + static_cast<int64_t>(min(n0 + j * 16 + li, a.N - 1)) * a.ldb + g * VEC;
  // Chunk h of block k of a row: 16 bytes from k + h BK / 2 + g VEC on.
  auto take = [&](const E* p, int k, bool any) __attribute__((always_inline)) {
    u32x4 v = {0u, 0u, 0u, 0u};
    const int left = a.K - k - g * VEC;
    if (any && left >= VEC) {
      __builtin_memcpy(&v, p + k, 16);
    } else if (any && left > 0) {
      E raw[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) raw[e] = e < left ? p[k + e] : static_cast<E>(0);
      __builtin_memcpy(&v, raw, 16);
    }
    return v;
  };
  auto multiply = [&](f32x4& c, u32x4 b, u32x4 x) __attribute__((always_inline)) {
    if constexpr (sizeof(E) == 2) {
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
    } else {
      const f32x4 fb = __builtin_bit_cast(f32x4, b), fx = __builtin_bit_cast(f32x4, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[e], fx[e], c, 0, 0, 0);
    }
  };
  const int whole = a.K / BK * BK;  // blocks without an edge
  int k = wave * BK;
  for (; k + (UNROLL - 1) * WAVES * BK < whole; k += UNROLL * WAVES * BK) {
    u32x4 x[UNROLL][2], b[UNROLL][TN][2];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = k + u * WAVES * BK + h * (BK / 2);
#pragma unroll
        for (int j = 0; j < TN; ++j) __builtin_memcpy(&b[u][j][h], pb[j] + at, 16);
        x[u][h] = (u32x4){0u, 0u, 0u, 0u};
        if (li < a.M) __builtin_memcpy(&x[u][h], pa + at, 16);
      }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < TN; ++j) multiply(acc[j], b[u][j][h], x[u][h]);
  }
  for (; k < a.K; k += WAVES * BK)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 x = take(pa, k + h * (BK / 2), li < a.M);
#pragma unroll
      for (int j = 0; j < TN; ++j) multiply(acc[j], take(pb[j], k + h * (BK / 2), true), x);
    }
  // Row li, columns 4 g to 4 g + 3 of tile j.
#pragma unroll
  for (int j = 0; j < TN; ++j) *reinterpret_cast<f32x4*>(&sums[wave][j][li * 16 + g * 4]) = acc[j];
  __syncthreads();
  for (int i = tid; i < TN * 256; i += WAVES * 64) {
    const int j = i / 256, m = i % 256 / 16, n = n0 + j * 16 + i % 16;
    if (m >= a.M || n >= (a.padC ? (a.N + 7) & ~7 : a.N)) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += sums[w][j][i % 256];
    finish_one<E, EPI>(a, m, n, s);
  }
}

// Tiles of 256 x 256 by four waves of 128 x 128, of 128 x 128, or, where the loads are what takes
// the time (few rows), of 128 x 64 and 64 x 64 with many steps' loads under way; of 128 x 128 and 64 x
// 64 by direct_kernel; rows_kernel's.
enum Tile : int { kBig = 0, kMiddle = 1, kDeep = 2, kDeepLow = 3, kDirect = 4, kDirectLow = 5, kRows = 6 };
struct TileOf {
  int m, n;
};
inline TileOf tile_size(int tile) {
  constexpr TileOf all[] = {{256, 256}, {128, 128}, {128, 64}, {64, 64}, {128, 128}, {64, 64}};
  return all[tile];
}
template <typename E, int EPI, bool TA, bool TB>
void launch(const Args<E>& a, int tile, int nblk, hipStream_t s) {
#define DABSN_LAUNCH(BM, BN, BUFS)                                                                         \
  hipLaunchKernelGGL((product_kernel<E, EPI, TA, TB, BM, BN, 2, 2, BUFS>), dim3(nblk), dim3(256), 0, s, a, \
                     nblk)
  if (tile == kBig) DABSN_LAUNCH(256, 256, 2);
  else if (tile == kMiddle) DABSN_LAUNCH(128, 128, 2);
  if constexpr (!TB && sizeof(E) == 2) {
    if (tile == kDeep) DABSN_LAUNCH(128, 64, 6);
    else if (tile == kDeepLow) DABSN_LAUNCH(64, 64, 8);
  }
  if constexpr (sizeof(E) == 4) {
    if (tile == kDirect)
      hipLaunchKernelGGL((direct_kernel<EPI, TA, TB, 128>), dim3(nblk), dim3(256), 0, s, a, nblk);
    else if (tile == kDirectLow)
      hipLaunchKernelGGL((direct_kernel<EPI, TA, TB, 64>), dim3(nblk), dim3(256), 0, s, a, nblk);
  }
  if constexpr (!TB && EPI != kShare) {
    if (tile == kRows) {
      // Columns as they fill the units; more waves where they do not.
      const E *A = reinterpret_cast<const E*>(a.A), *B = reinterpret_cast<const E*>(a.B);
      const int tiles = (a.N + 15) / 16;
      if (tiles > 1024)
        hipLaunchKernelGGL((rows_kernel<E, EPI, 2, 4>), dim3((tiles + 1) / 2), dim3(256), 0, s, a, A, B);
      else if (tiles > 256)
        hipLaunchKernelGGL((rows_kernel<E, EPI, 1, 4>), dim3(tiles), dim3(256), 0, s, a, A, B);
      else
        hipLaunchKernelGGL((rows_kernel<E, EPI, 1, 16>), dim3(tiles), dim3(1024), 0, s, a, A, B);
    }
  }
#undef DABSN_LAUNCH
}

}  // namespace linear
}  // namespace dabsn
