// Row kernels over a vocabulary: token log probabilities and distillation.
//
// Both take rows of logits [rows, V] (or the fp32 logits of a readout before its bias) and a
// temperature T, z = x / T, and form the row's softmax in one pass, fp32, with a running reference r
// per thread, e = exp(z - r). With M the row's largest logit:
//   R = the sum of exp((x - M) / T) over all logits but M itself
//   log probabilities   logp_t = (x_t - M) / T - ln(1 + R);  H = ln(1 + R) - sum p (z - M / T);
//                       the K largest logits in order (equal ones by index)
//   distillation        sum q (ln q - logp) over a teacher's listed tokens and, with the
//                       teacher's normaliser, over the rest of the vocabulary as one event
// and a backward that reads the logits once more and writes their gradient.
//
// M stays out of the sums: of a token with nearly all the mass log p is
// -ln(1 + R) with R small, and in a sum that holds the 1 too fp32 would keep R to 2^-24 of 1, not of
// itself (log p = -1e-4 was off by 1e-3 of itself). So each thread keeps the sums of the group with
// its largest logit apart from the others', and where R turns out below 1/4 the thread that has M
// takes that group's again without it. 8192 x 32000 bf16 take 83 to 87 us with this and groups of 16, 86
// to 88 with groups of 8 or with that group taken again in every row, 82 without any of it.
//
// The pass is bound by memory where an element costs few instructions: 9.5 vector instructions here
// (counted at 8192 x 32000 bf16), against the 12 that the time of its 2 bytes allows. So the
// exponent's argument is one fma of the logit, x c - r with c = log2 e / T and r, in units of ln 2,
// near the thread's maximum; r moves only when a group exceeds it by 8. c is rounded: the sums u of
// e (x c - r), which the entropy needs anyhow, give the exact normaliser to first order. The fma
// leaves what r = x c lost in its own rounding, half an ulp of x c: below 4 up to 2^26, and 2^100 of
// a mask's -1e30, so r is kept in +-2^26. It starts at the lower end, from where the words that a
// mask rules out with any large negative number add 0 and move nothing. A row whose largest logit
// lies beyond half of the lower end or beyond the upper one takes the pass again with differences
// formed first.
#include <algorithm>

#include "../../include/dabsn_hip.h"
#include "capi.hpp"
#include "common.hpp"

namespace dabsn {
namespace vocab {

constexpr double kLn2 = 0.693147180559945309417;
constexpr float kLowest = -3.40282346638528860e38f;
constexpr int kMaxTop = 128;
// Candidates of the top selection that fit: all of a vocabulary whose vectors are fewer than
// kMaxTop (there the threshold may be below every logit), and some room for equal logits.
constexpr int kCap = 1152;
constexpr uint32_t kErrToken = 1u;

typedef u32x4 u32x4_any __attribute__((aligned(2)));

// bf16 bits, two to a word, as floats.
template <int N>
__device__ __forceinline__ void halves(const uint32_t (&u)[N / 2], float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    v[2 * k] = __builtin_bit_cast(float, u[k] << 16);
    v[2 * k + 1] = __builtin_bit_cast(float, u[k] & 0xffff0000u);
  }
}

// A row's logits, W = 8 bf16 or 4 fp32 (16 bytes) at a time, plus the readout's bias. A row of an
// odd vocabulary starts anywhere in a line of 128 bytes: its vectors begin at the first whole line,
// column `head`, and the logits before it and behind the last vector are taken one by one.
// ONCE: the loads are marked as not to be kept in the caches. 8192 x 32000 bf16 take 89 us instead
// of 98, beside a backward that writes as much 102 instead of 107, as the lines that a pass would
// leave there, and those it would push out to memory, are of no use. Whole lines at a time are
// needed for this: fp32 lanes that took two neighbouring vectors (each line fetched twice) or vectors
// across lines lost a third instead, 173 -> 205 and 231 us at 4099 x 50021.
template <typename E, bool BIAS, bool ONCE>
struct Row {
  static constexpr int W = is_bf16<E>::value ? 8 : 4;
  const E* x;
  const bf16* b;
  int V, head;
  __device__ __forceinline__ Row(const E* x_, const bf16* b_, int V_) : x(x_), b(b_), V(V_) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) & 127) / sizeof(E);
    head = min(V, static_cast<int>((128 / sizeof(E) - off) & (128 / sizeof(E) - 1)));
  }
  __device__ __forceinline__ int vectors() const { return (V - head) / W; }
  __device__ __forceinline__ int64_t column(int c) const {
    return head + static_cast<int64_t>(c) * W;
  }
  // f(column, value) for this thread's logit before the vectors and the one behind them.
  template <typename F>
  __device__ __forceinline__ void singles(F f) const {
    const int t = threadIdx.x, j = head + vectors() * W + t;
    if (t < head) f(t, at(t));
    if (j < V) f(j, at(j));
  }
  struct Raw {
    u32x4 v;
    uint32_t bias[W / 2];
  };
  __device__ __forceinline__ Raw load(int c) const {
    Raw r;
    const u32x4* p = reinterpret_cast<const u32x4*>(x + column(c));
    if constexpr (ONCE) r.v = __builtin_nontemporal_load(p);
    else r.v = *p;
    if constexpr (BIAS) __builtin_memcpy(r.bias, b + column(c), 2 * W);
    return r;
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[W]) {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = r.v[k];
    if constexpr (is_bf16<E>::value) {
      halves<W>(u, v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __builtin_bit_cast(float, u[k]);
    }
    if constexpr (BIAS) {
      float w[W];
      halves<W>(r.bias, w);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] += w[k];
    }
  }
  static __device__ __forceinline__ void keep(Raw& r) {
    asm volatile("" : "+v"(r.v));
    if constexpr (BIAS) {
#pragma unroll
      for (int k = 0; k < W / 2; ++k) asm volatile("" : "+v"(r.bias[k]));
    }
  }
  __device__ __forceinline__ float at(int64_t j) const {
    float v = ld(x, static_cast<size_t>(j));
    if constexpr (BIAS) v += bf2f(b[j]);
    return v;
  }
};

// A row's logits as its threads go through them: each(f, g) calls f(c, n, values) for groups of P =
// 8 or 16 values, the vectors c, c + NTH, ... of which the first n are the row's (-inf stands for a
// missing one's values); then g(column, value) for the logits outside the vectors. What a group
// costs beside its logits (its largest, the reference's test) is shared by P of them.
template <int NTH, int P_, typename R>
struct Group {
  static constexpr int P = P_, W = R::W, G = P / W;
  static __device__ __forceinline__ void values(const typename R::Raw (&raw)[G], int n, float (&v)[P]) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float w[W];
      R::unpack(raw[g], w);
#pragma unroll
      for (int k = 0; k < W; ++k) v[g * W + k] = g < n ? w[k] : -INFINITY;
    }
  }
  // How many of the group's vectors are among nv.
  static __device__ __forceinline__ int count(int c, int nv) {
    int n = 1;
#pragma unroll
    for (int g = 1; g < G; ++g) n += c + g * NTH < nv;
    return n;
  }
  // The group that starts at vector c.
  template <typename F>
  static __device__ __forceinline__ void last(const typename R::Raw (&raw)[G], int c, int nv, F f) {
    if (c >= nv) return;
    const int n = count(c, nv);
    float v[P];
    values(raw, n, v);
    f(c, n, v);
  }
};
// Streamed: from memory each time, 32 values' loads in flight.
template <int NTH, int P_, typename R_>
struct Streamed {
  using R = R_;
  const R& row;
  static constexpr int P = P_, W = R::W;
  template <typename F, typename H>
  __device__ __forceinline__ void each(F f, H h) const {
    using Gr = Group<NTH, P, R>;
    constexpr int G = Gr::G, U = 32 / P;
    const int nv = row.vectors(), tid = threadIdx.x;
    int b = 0;  // the block's first vector
    for (; b + U * G * NTH <= nv; b += U * G * NTH) {
      typename R::Raw raw[U][G];
#pragma unroll
      for (int k = 0; k < U * G; ++k) raw[k / G][k % G] = row.load(b + k * NTH + tid);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float v[P];
        Gr::values(raw[k], G, v);
        f(b + k * G * NTH + tid, G, v);
      }
    }
    if (b < nv) {
      typename R::Raw raw[U][G];
#pragma unroll
      for (int k = 0; k < U * G; ++k) raw[k / G][k % G] = row.load(min(b + k * NTH + tid, nv - 1));
      // Without a use out here the compiler moves each load under its condition, one at a time.
#pragma unroll
      for (int k = 0; k < U * G; ++k) R::keep(raw[k / G][k % G]);
#pragma unroll
      for (int k = 0; k < U; ++k) Gr::last(raw[k], b + k * G * NTH + tid, nv, f);
    }
    row.singles(h);
  }
};
// Held: loaded once into NV vectors of registers a thread (at most NTH NV vectors), for a row that
// is read twice and written: the second reading otherwise comes from the memory side, as the rows
// under way (2,048 of 64 KB) are far more than the L2 caches hold.
template <int NTH, int NV, typename R_>
struct Held {
  using R = R_;
  using Gr = Group<NTH, 8, R>;
  static constexpr int P = 8, W = R::W, G = Gr::G;
  const R& row;
  typename R::Raw raw[NV / G][G];
  __device__ __forceinline__ explicit Held(const R& row_) : row(row_) {
    const int nv = row.vectors();
#pragma unroll
    for (int k = 0; k < NV; ++k)
      raw[k / G][k % G] = row.load(max(0, min(k * NTH + static_cast<int>(threadIdx.x), nv - 1)));
  }
  template <typename F, typename H>
  __device__ __forceinline__ void each(F f, H h) const {
    const int nv = row.vectors();
#pragma unroll
    for (int k = 0; k < NV / G; ++k) Gr::last(raw[k], k * G * NTH + threadIdx.x, nv, f);
    row.singles(h);
  }
};
// NV = 0: streamed.
template <int NTH, int NV, int P = 8, typename R>
__device__ __forceinline__ auto source(const R& row) {
  if constexpr (NV > 0) return Held<NTH, NV, R>(row);
  else return Streamed<NTH, P, R>{row};
}

// Of a quiet NaN and a number the number; fmaxf adds an instruction an operand to quiet others.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <int P>
__device__ __forceinline__ float largest(const float (&v)[P]) {
  float m = max3(v[0], v[1], v[2]);
#pragma unroll
  for (int k = 3; k + 1 < P; k += 2) m = max3(m, v[k], v[k + 1]);
  return max3(m, v[P - 1], v[P - 1]);
}

// The sum over the block of N values a thread, to every thread; the waves' sums are added in 64
// bits (16 roundings to fp32 of a sum that grows would be most of its error). sh: N * NTH/64 floats.
template <int NTH, int N>
__device__ __forceinline__ void block_sums(float (&v)[N], double (&sum)[N], float* sh) {
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = v[i] = wave_sum(v[i]);
  if constexpr (NTH > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh[i * (NTH / 64) + (threadIdx.x >> 6)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      sum[i] = 0.0;
#pragma unroll
      for (int w = 0; w < NTH / 64; ++w) sum[i] += sh[i * (NTH / 64) + w];
    }
  }
}
template <int NTH>
__device__ __forceinline__ float block_max(float v, float* sh) {
  v = wave_max(v);
  if constexpr (NTH > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < NTH / 64; ++w) v = fmaxf(v, sh[w]);
  }
  return v;
}
// The first thread of the block for which `mine` is true.
template <int NTH>
__device__ __forceinline__ int block_first(bool mine, float* sh) {
  if constexpr (NTH == 64) return __ffsll(static_cast<unsigned long long>(__ballot(mine))) - 1;
  int* word = reinterpret_cast<int*>(sh);
  __syncthreads();
  if (threadIdx.x == 0) *word = NTH;
  __syncthreads();
  if (mine) atomicMin(word, static_cast<int>(threadIdx.x));
  __syncthreads();
  return *word;
}

// A thread's share of a row, relative to its reference r: sums of e = 2^arg and of e arg, of the
// group with its largest logit (at: its first vector, -1: a logit of its own) apart from the others.
// arg = x c - r; SAFE rows have arg = (x - r) c. Logits of -inf give e = 0; NaN makes a sum NaN.
constexpr float kFar = 67108864.0f;  // 2^26
template <bool SAFE>
struct Share {
  static constexpr float kFloor = SAFE ? kLowest : -kFar;
  float best = -INFINITY, r = kFloor;
  float s = 0.0f, u = 0.0f, sb = 0.0f, ub = 0.0f;
  int at = -1;
  float c;
  __device__ __forceinline__ explicit Share(float c_) : c(c_) {}
  static __device__ __forceinline__ float arg(float x, float r, float c) {
    return SAFE ? (x - r) * c : __builtin_fmaf(x, c, -r);
  }
  // The reference of a largest logit.
  __device__ __forceinline__ float place(float x) const { return fmaxf(SAFE ? x : x * c, kFloor); }
  // From the reference `from` to a larger one.
  __device__ __forceinline__ float shift(float from, float to) const {
    return from == to ? 0.0f : SAFE ? (from - to) * c : from - to;  // both may be inf
  }
  static __device__ __forceinline__ void scale(float d, float& s, float& u) {
    const float f = __builtin_amdgcn_exp2f(d);
    u = f == 0.0f ? 0.0f : f * (u + d * s);
    s *= f;
  }
  __device__ __forceinline__ void raise(float to) {
    const float d = shift(r, to);
    scale(d, s, u);
    scale(d, sb, ub);
    r = to;
  }
  template <int N>
  __device__ __forceinline__ void fold(const float (&v)[N], float vm, int k) {
    const float t = SAFE ? vm : vm * c;
    if (t > (SAFE ? r : r + 8.0f)) raise(t);
    float vs = 0.0f, vu = 0.0f;
    add<N>(v, -1, vs, vu);
    const bool up = vm > best;
    s += up ? sb : vs;
    u += up ? ub : vu;
    sb = up ? vs : sb;
    ub = up ? vu : ub;
    at = up ? k : at;
    best = up ? vm : best;
  }
  // Adds all but the `without`th.
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N], int without, float& vs, float& vu) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float a = arg(k == without ? -INFINITY : v[k], r, c);
      const float e = __builtin_amdgcn_exp2f(a);
      vs += e;
      vu = __builtin_fmaf(e, fmaxf(a, -1e30f), vu);  // arg = -inf has e = 0
    }
  }
  __device__ __forceinline__ void fold1(float x) {
    const float v[1] = {x};
    fold(v, x, -1);
  }
  // The block's shares as one: m, the row's largest logit, r its place, and the sums of the others.
  // group(k, v): the group whose first vector is k. sh: 2 * NTH/64 floats.
  template <int NTH, int P, typename Group>
  __device__ __forceinline__ void join(Group group, float& m, double (&sum)[2], float* sh) {
    m = block_max<NTH>(best, sh);
    raise(place(m));
    float all[2] = {s + sb, u + ub};
    block_sums<NTH, 2>(all, sum, sh);
    const float am = SAFE ? 0.0f : arg(m, r, c), em = __builtin_amdgcn_exp2f(am);  // m's own
    sum[0] -= em;
    sum[1] -= static_cast<double>(em) * am;
    if (sum[0] >= 0.25 || m == -INFINITY) return;
    if (block_first<NTH>(best == m, sh) == static_cast<int>(threadIdx.x)) {
      sb = ub = 0.0f;
      if (at >= 0) {
        float v[P];
        group(at, v);
        int k = P - 1;
#pragma unroll
        for (int i = P - 2; i >= 0; --i) k = v[i] == m ? i : k;
        add<P>(v, k, sb, ub);
      }
    }
    all[0] = s + sb;
    all[1] = u + ub;
    block_sums<NTH, 2>(all, sum, sh);
  }
};

// What a row's pass leaves. Log probabilities are differences of numbers of the size of the
// logits, so the few of a row are formed in 64 bits.
struct Norm {
  float m, r;   // the largest logit and its place
  double s, u;  // sums of the others
  bool safe;
  // f(arg) with the row's form of the exponent's argument as a function of a logit.
  template <typename F>
  __device__ __forceinline__ void with_arg(float c, F f) const {
    if (safe) f([r = r, c](float x) { return Share<true>::arg(x, r, c); });
    else f([r = r, c](float x) { return Share<false>::arg(x, r, c); });
  }
  __device__ __forceinline__ bool nan() const { return s != s || m == INFINITY; }
  __device__ __forceinline__ bool empty() const { return m == -INFINITY && s == s; }  // no finite logit
  // arg of the largest: what its place lost in its rounding, exactly.
  __device__ __forceinline__ float left(float c) const {
    return safe ? 0.0f : Share<false>::arg(m, r, c);
  }
};
// 1 / T, c and its error, from the host.
struct Scale {
  double inv_t, delta;
  float c;
};
static Scale scale_of(double t) {
  Scale k;
  k.inv_t = 1.0 / t;
  k.c = static_cast<float>(k.inv_t / kLn2);
  k.delta = k.inv_t / kLn2 / static_cast<double>(k.c) - 1.0;
  return k;
}
// 1 / x of a number at least 1: 1 ulp of fp32, doubled in bits by a step of Newton's.
__device__ __forceinline__ double reciprocal(double x) {
  const double r = __builtin_amdgcn_rcpf(static_cast<float>(x));
  return r * __builtin_fma(-x, r, 2.0);
}
// A row's sums with 1 / T at its full precision, log2 e / T = c (1 + delta): to first order each e is
// short of the factor 2^(arg delta), and all of 2^-left as M's own e is to be 1.
struct Sums {
  double at, inv_t;  // M; 1 / T
  double ln;         // ln(1 + R)
  double h;          // the entropy
  float left;
  bool empty;
  __device__ __forceinline__ Sums(const Norm& n, const Scale& k)
      : at(n.m), inv_t(k.inv_t), left(n.left(k.c)), empty(n.empty()) {
    const double f = __builtin_amdgcn_exp2f(-left);
    const double R = n.nan() ? NAN : empty ? 0.0 : f * (n.s + kLn2 * k.delta * n.u);
    // ln(1 + R) for small R too: with what the sum lost in its rounding, to first order.
    const double one = 1.0 + R;
    const double inverse = reciprocal(one);
    ln = log(one) + (R - (one - 1.0)) * inverse;
    // sum p (z - M / T) (1 + R); its own correction would need the sum of e arg^2, and what it
    // lacks, delta |arg| of itself, is an argument's rounding.
    const double w = empty ? 0.0 : kLn2 * f * (n.u - left * n.s);
    h = ln - w * inverse;
    h = h < 0.0 ? 0.0 : h;
  }
  // ln of the sum of exp((x - y) / T) over the row's logits x.
  __device__ __forceinline__ double ln_sum(double y) const {
    return empty ? -INFINITY : (at - y) * inv_t + ln;
  }
  // log p of a logit x.
  __device__ __forceinline__ double logp(float x) const {
    return empty ? -INFINITY : -ln_sum(static_cast<double>(x));
  }
  // ln of the sum of all e = 2^arg.
  __device__ __forceinline__ double ln_e() const { return ln + kLn2 * left; }
};

__device__ __forceinline__ int pad_of(int head) { return -head & 7; }

// REST: over the words whose bit in `listed` is not set.
template <int NTH, bool REST, bool SAFE, typename S, typename See, typename Last>
__device__ __forceinline__ Norm row_pass(const S& src, float c, const uint8_t* listed, float* sh,
                                         See see, Last last) {
  // Bit j + pad of `listed` is column j's: whole vectors start at a multiple of 8 (or 4) bits.
  const int pad = pad_of(src.row.head);
  const uint8_t* body = REST ? listed + (src.row.head + pad) / 8 : nullptr;
  constexpr int P = S::P;
  Share<SAFE> a(c);
  // Listed words out of a group's values; whether there is one.
  static_assert(!REST || P == 8, "a byte of marks a group");
  auto mask = [&](int k, int n, const float (&v)[P], float (&w)[P]) {
    uint32_t bits = 0;
    if constexpr (S::W == 8) {
      bits = body[k];
    } else {
      auto four = [&](int i) { return body[i >> 1] >> (4 * (i & 1)) & 15u; };
      bits = four(k) | (n == 2 ? four(k + NTH) << 4 : 0u);
    }
    if (!bits) return false;  // few vectors hold one
#pragma unroll
    for (int i = 0; i < P; ++i) w[i] = (bits >> i & 1) ? -INFINITY : v[i];
    return true;
  };
  src.each(
      [&](int k, int n, const float (&v)[P]) {
        if constexpr (REST) {
          float w[P];
          if (mask(k, n, v, w)) {
            a.fold(w, largest(w), k);
            return;
          }
        }
        const float vm = largest(v);
        a.fold(v, vm, k);
        see(k, vm);
      },
      [&](int j, float x) {
        a.fold1(REST && (listed[(j + pad) >> 3] >> ((j + pad) & 7) & 1) ? -INFINITY : x);
        last(j, x);
      });
  float m;
  double sum[2];
  a.template join<NTH, P>(
      [&](int k, float (&v)[P]) {
        using Gr = Group<NTH, P, typename S::R>;
        typename S::R::Raw raw[Gr::G];
        const int nv = src.row.vectors(), n = Gr::count(k, nv);
#pragma unroll
        for (int g = 0; g < Gr::G; ++g) raw[g] = src.row.load(min(k + g * NTH, nv - 1));
        Gr::values(raw, n, v);
        if constexpr (REST) {
          float w[P];
          if (mask(k, n, v, w)) {
#pragma unroll
            for (int i = 0; i < P; ++i) v[i] = w[i];
          }
        }
      },
      m, sum, sh);
  return Norm{m, a.r, sum[0], sum[1], SAFE};
}
// The row's norm; `see` gets each group's first vector and largest logit, `last` the logits outside.
template <int NTH, bool REST, typename S, typename See, typename Last>
__device__ __forceinline__ Norm norm_of(const S& src, float c, const uint8_t* listed, float* sh,
                                        See see, Last last) {
  const Norm n = row_pass<NTH, REST, false>(src, c, listed, sh, see, last);
  if (n.r >= -0.5f * kFar && n.r <= kFar) return n;
  __syncthreads();
  return row_pass<NTH, REST, true>(src, c, listed, sh, [](int, float) {}, [](int, float) {});
}

// ---- the K largest logits of a row ---------------------------------------------------------
// Order-preserving integers of floats; -0 counts as 0, and NaN with -inf, below every number.
constexpr uint32_t kNone = 0x007fffffu;  // key of -inf
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return kNone;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// A thread's best groups, by their largest logits: two with their places, the third's value.
struct Best {
  float v1 = -INFINITY, v2 = -INFINITY, v3 = -INFINITY;
  int c1 = -1, c2 = -1;
  __device__ __forceinline__ void see(float vm, int c) {
    const bool up1 = vm > v1, up2 = vm > v2;
    v3 = up2 ? v2 : fmaxf(v3, vm);
    v2 = up1 ? v1 : up2 ? vm : v2;
    c2 = up1 ? c1 : up2 ? c : c2;
    v1 = up1 ? vm : v1;
    c1 = up1 ? c : c1;
  }
};

template <int NTH>
struct TopShared {
  uint64_t cand[kCap];  // key << 32 | ~column: the larger, the earlier
  float best[NTH];
  uint16_t full[NTH];
  uint32_t tau;
  int count, fulls;
  int wave[NTH / 64];
};

__device__ __forceinline__ void push(uint64_t* cand, int* count, uint32_t key, int j) {
  const int at = atomicAdd(count, 1);
  if (at < kCap) cand[at] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~j);
}

// How many of the row's keys are at least `lo`.
template <int NTH, typename R>
__device__ int count_from(const R& row, uint32_t lo, TopShared<NTH>& t) {
  int n = 0;
  Streamed<NTH, 8, R>{row}.each(
      [&](int, int m, const float (&v)[8]) {
#pragma unroll
        for (int k = 0; k < 8; ++k) n += k < m * R::W && key_of(v[k]) >= lo;
      },
      [&](int, float x) { n += key_of(x) >= lo; });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) t.wave[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < NTH / 64; ++w) n += t.wave[w];
  return n;
}

// Appends the first `want` columns (in order) whose key is `key`.
template <int NTH, typename R>
__device__ void append_equal(const R& row, uint32_t key, int want, TopShared<NTH>& t) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int j0 = 0; j0 < row.V && want > 0; j0 += NTH) {
    const int j = j0 + threadIdx.x;
    const bool hit = j < row.V && key_of(row.at(j)) == key;
    const uint64_t mask = __ballot(hit);
    __syncthreads();  // the counts of the tile before have been read
    if (lane == 0) t.wave[wave] = __popcll(mask);
    __syncthreads();
    int before = __popcll(mask & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < NTH / 64; ++w) {
      before += w < wave ? t.wave[w] : 0;
      all += t.wave[w];
    }
    if (hit && before < want) push(t.cand, &t.count, key, j);
    want -= all;
  }
}

// The upper 16 bits of the K-th largest of 64 N keys, N a lane, bit by bit: a bound that K reach.
template <int N>
__device__ __forceinline__ uint32_t bound_of(const uint32_t (&k)[N], int K) {
  uint32_t tau = 0;
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t to = tau | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(k[i] >= to));
    if (n >= K) tau = to;
  }
  return tau << 16;
}
template <int N, int M>
__device__ __forceinline__ uint32_t bound_of_largest(const uint32_t (&k)[N], int K) {
  uint32_t m[M];
#pragma unroll
  for (int i = 0; i < M; ++i) m[i] = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m[i % M] = max(m[i % M], k[i]);
  return bound_of<M>(m, K);
}

// Gathers candidates that hold the K largest logits (equal ones by column). Every thread's
// largest is known from the row's pass; the K-th largest of these, or of the largest of G of their
// groups, is a bound that K logits reach, and few more do: of well mixed logits G ln(G / (G - K)), 74
// for K = 64 of 256. So only the groups that reach it are read again, gathered and ranked against
// each other (4099 x 50021 fp32: 120 us without alternatives, 125 with 1, 133 with 20, 145 with 64, 183
// with 128; bf16 69, 87, 89, 98, 115). Where more than kCap reach it (rows with many equal logits)
// the K-th largest key is found by bisection over the row. first, last: the thread's logits outside
// the vectors (-inf: none). With a workgroup a compute unit, whose time is that of one load after
// another, the threads load their best groups before the bound is known (256 x 32000 bf16 with 20
// alternatives 13.0 us instead of 13.6; one row with 5 takes 8.6, without any 5.4).
template <int NTH, typename R>
__device__ void top_k(const R& row, int K, const Best& b, float first, float last, bool nan,
                      TopShared<NTH>& t) {
  const int tid = threadIdx.x;
  constexpr int W = R::W, N = NTH / 64;
  constexpr bool AHEAD = NTH == 1024;
  const int nv = row.vectors();
  typename R::Raw ahead[8 / W];
  if constexpr (AHEAD) {
#pragma unroll
    for (int g = 0; g < 8 / W; ++g) ahead[g] = row.load(max(0, min(b.c1 + g * NTH, nv - 1)));
  }
  t.best[tid] = fmaxf(b.v1, fmaxf(first, last));
  if (tid == 0) t.count = t.fulls = 0;
  __syncthreads();
  if (tid < 64) {
    uint32_t k[N];
#pragma unroll
    for (int i = 0; i < N; ++i) k[i] = key_of(t.best[i * 64 + tid]) >> 16;
    uint32_t tau = 0;
    if (K <= 16) tau = bound_of_largest<N, 1>(k, K);
    else if (N > 4 && K <= 64) tau = bound_of_largest<N, N < 4 ? N : 4>(k, K);
    else if (K <= NTH) tau = bound_of<N>(k, K);
    if (tid == 0) t.tau = max(tau, kNone + 1);
  }
  __syncthreads();
  const uint32_t tau = t.tau;
  auto take = [&](int j, float x) {
    const uint32_t k = key_of(x);
    if (k >= tau) push(t.cand, &t.count, k, j);
  };
  auto take_raw = [&](int c, const typename R::Raw& raw) {
    float v[W];
    R::unpack(raw, v);
#pragma unroll
    for (int k = 0; k < W; ++k) take(static_cast<int>(row.column(c)) + k, v[k]);
  };
  auto take_vector = [&](int c) { take_raw(c, row.load(c)); };
  // A thread whose third best group reaches the bound too leaves all of its vectors to a wave.
  if (key_of(b.v3) >= tau) {
    t.full[atomicAdd(&t.fulls, 1)] = static_cast<uint16_t>(tid);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = i ? b.c2 : b.c1;
      if (c < 0 || key_of(i ? b.v2 : b.v1) < tau) continue;
      if (AHEAD && i == 0) {
#pragma unroll
        for (int g = 0; g < 8 / W; ++g)
          if (c + g * NTH < nv) take_raw(c + g * NTH, ahead[g]);
        continue;
      }
      take_vector(c);
      if (W == 4 && c + NTH < nv) take_vector(c + NTH);
    }
  }
  take(tid, first);
  take(row.head + nv * W + tid, last);
  __syncthreads();
  for (int i = tid >> 6; i < t.fulls; i += NTH / 64)
    for (int c = t.full[i] + (tid & 63) * NTH; c < nv; c += 64 * NTH) take_vector(c);
  __syncthreads();
  int n = t.count;
  if (n > kCap || nan) {  // a NaN may have hidden its neighbours' maximum
    uint32_t lo = nan ? 0 : tau, hi = 0xffffffffu;  // K keys are at least lo, fewer at least hi
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (count_from<NTH>(row, mid, t) >= K) lo = mid; else hi = mid;
    }
    __syncthreads();
    if (tid == 0) t.count = 0;
    __syncthreads();
    Streamed<NTH, 8, R>{row}.each(
        [&](int c, int m, const float (&v)[8]) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < m * W && key_of(v[k]) > lo)
              push(t.cand, &t.count, key_of(v[k]),
                   static_cast<int>(row.column(c + k / W * NTH)) + k % W);
        },
        [&](int j, float x) {
          if (key_of(x) > lo) push(t.cand, &t.count, key_of(x), j);
        });
    __syncthreads();
    n = t.count;
    append_equal<NTH>(row, lo, K - n, t);
    __syncthreads();
    n = t.count;
  }
  if (n < K) {  // fewer numbers than K: -inf (and NaN) fill the places
    append_equal<NTH>(row, kNone, K - n, t);
    __syncthreads();
    n = t.count;
  }
}

// What the backward needs of a row: M, and ln(1 + R) with the sign bit of a row of differences.
__device__ __forceinline__ void put_stats(float* stats, const Norm& n, const Sums& sums) {
  stats[0] = n.m;
  stats[1] = copysignf(static_cast<float>(sums.ln), n.safe ? -1.0f : 1.0f);
}
struct Stats {
  Norm n;  // without its sums
  float ln;
  __device__ __forceinline__ Stats(const float* stats, float c) {
    const bool safe = signbit(stats[1]);
    const float m = stats[0];
    n = Norm{m, fmaxf(safe ? m : m * c, kLowest), 0.0, 0.0, safe};
    ln = fabsf(stats[1]);
  }
};

// (With alternatives at most 84 registers: six waves share a SIMD, 146 us at 4099 x 50021 fp32, top 64,
// instead of 154 with five.)
template <typename E, bool BIAS, int NTH, bool TOP>
__global__ void __launch_bounds__(NTH, !TOP ? 1 : NTH == 256 ? (BIAS ? 5 : 6) : 4) logprobs_kernel(
    int V, int64_t ldl, const E* __restrict__ logits, const bf16* __restrict__ bias,
    const int64_t* __restrict__ targets, int64_t ignore, Scale k, int K,
    float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ stats,
    float* __restrict__ top_lp, int64_t* __restrict__ top_idx, uint32_t* err) {
  __shared__ float sh[2 * (NTH / 64)];
  const size_t r = blockIdx.x;
  const Row<E, BIAS, !BIAS> row(logits + r * ldl, bias, V);
  Best best;
  float first = -INFINITY, last = -INFINITY;  // this thread's logits outside the vectors
  const Norm n = norm_of<NTH, false>(
      source<NTH, 0, TOP ? 8 : 16>(row), k.c, nullptr, sh,
      [&](int c, float vm) {
        if constexpr (TOP) best.see(vm, c);
      },
      [&](int j, float x) { (j < row.head ? first : last) = x; });
  const Sums sums(n, k);
  auto lp = [&](float x) { return static_cast<float>(sums.logp(x)); };
  if (threadIdx.x == 0) {
    entropy[r] = static_cast<float>(sums.h);
    if (stats) put_stats(stats + 2 * r, n, sums);
    if (logprob) {
      const int64_t t = targets[r];
      float v = 0.0f;
      if (t != ignore) {
        if (t < 0 || t >= V) {
          atomicOr(err, kErrToken);
          v = NAN;
        } else {
          v = lp(row.at(t));
        }
      }
      logprob[r] = v;
    }
  }
  if constexpr (TOP) {
    __shared__ TopShared<NTH> t;
    top_k<NTH>(row, K, best, first, last, n.nan(), t);
    const int count = t.count;
    for (int i = threadIdx.x; i < count; i += NTH) {
      const uint64_t mine = t.cand[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < count; ++j) rank += t.cand[j] > mine;
      if (rank < K) {
        top_lp[r * K + rank] = lp(of_key(static_cast<uint32_t>(mine >> 32)));
        top_idx[r * K + rank] = static_cast<int64_t>(~static_cast<uint32_t>(mine));
      }
    }
  }
}

// ---- where a gradient goes -----------------------------------------------------------------
// A row of the logits' type; or, for the gradient products of a bf16 readout, which run as 16-bit
// matrix products with fp32 sums and round their results to bf16 (2^-9):
//   planes   two bf16 rows whose sum holds 17 bits of the fp32 value, of any size (the products'
//            error 2^-18 a term; one bf16 row would add as much as the results' rounding);
//   split    these two, for the products that sum over rows, where a word's values may all be small
//            (a third of a softmax over 32000 words lies below 1e-7), and an fp16 row, for the one
//            that sums over the row's words: times a power of two by a bound of the row's values,
//            so it holds 11 bits of values down to 2^-29 of that (an error of 2^-12 a term, an
//            eighth of the results' rounding) and costs half of the planes' products.
enum OutKind : int { kRows = 0, kPlanes = 1, kSplit = 2 };
enum Parts : int { kPartPlanes = 1, kPartHalf = 2 };  // of a split row
constexpr float kMostWeight = 256.0f;
__device__ __forceinline__ uint32_t pair(float a, float b) {
  return static_cast<uint32_t>(f2bf(a)) | static_cast<uint32_t>(f2bf(b)) << 16;
}
template <typename E>
struct RowOut {
  static constexpr int W = is_bf16<E>::value ? 8 : 4;
  E* p;
  int head;
  __device__ __forceinline__ void put(int64_t j, float v) const { st(p, j, v); }
  __device__ __forceinline__ void put(int c, const float (&v)[W]) const {
    u32x4 u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (is_bf16<E>::value) u[k] = pair(v[2 * k], v[2 * k + 1]);
      else u[k] = __builtin_bit_cast(uint32_t, v[k]);
    }
    __builtin_nontemporal_store(u, reinterpret_cast<u32x4_any*>(p + head + static_cast<size_t>(c) * W));
  }
};
struct PlanesOut {
  bf16* p;
  int64_t plane;
  int head;
  __device__ __forceinline__ static float left(float v) {
    const float r = v - bf2f(f2bf(v));
    return r == r ? r : 0.0f;  // inf and NaN are the first plane's alone
  }
  __device__ __forceinline__ void put(int64_t j, float v) const {
    p[j] = f2bf(v);
    p[plane + j] = f2bf(left(v));
  }
  __device__ __forceinline__ void put(int c, const float (&v)[4]) const {
    const uint32_t hi[2] = {pair(v[0], v[1]), pair(v[2], v[3])};
    const uint32_t lo[2] = {pair(left(v[0]), left(v[1])), pair(left(v[2]), left(v[3]))};
    bf16* q = p + head + static_cast<size_t>(c) * 4;
    __builtin_memcpy(q, hi, 8);
    __builtin_memcpy(q + plane, lo, 8);
  }
};
struct SplitOut {
  PlanesOut planes;  // the second row one stride behind the first
  _Float16* half;    // and the fp16 one behind that
  int parts;
  float scale;
  __device__ __forceinline__ void put(int64_t j, float v) const {
    if (parts & kPartPlanes) planes.put(j, v);
    if (parts & kPartHalf) half[j] = static_cast<_Float16>(v * scale);
  }
  __device__ __forceinline__ void put(int c, const float (&v)[4]) const {
    if (parts & kPartPlanes) planes.put(c, v);
    if (parts & kPartHalf) {
      _Float16 h[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) h[k] = static_cast<_Float16>(v[k] * scale);
      __builtin_memcpy(half + planes.head + static_cast<size_t>(c) * 4, h, 8);
    }
  }
};
template <typename E, int KIND>
__device__ __forceinline__ auto out_row(void* out, size_t r, int64_t ldo, int64_t plane, int head) {
  if constexpr (KIND == kPlanes) return PlanesOut{static_cast<bf16*>(out) + r * ldo, plane, head};
  else return RowOut<E>{static_cast<E*>(out) + r * ldo, head};
}

// d x_j = -(p_j / T) (g_lp + sum g_top + g_H (logp_j + H)), plus g_lp / T at the target and
// g_top / T at the alternatives. The whole row is written without these, then their places, where
// g (1 - p) comes from log p: the difference of g and g p would lose a small 1 - p.
struct LogprobGrad {
  float A, B;  // e_j (B arg_j + A) off these places
  float sum, ge, h, ln, inv_t;
  __device__ __forceinline__ LogprobGrad(const Stats& st, float c, float sum_, float ge_, float h_,
                                         float inv_t_, bool off)
      : sum(sum_), ge(ge_), h(h_), ln(st.ln), inv_t(inv_t_) {
    const float left = st.n.left(c), is = st.n.empty() ? 0.0f : expf(-ln) * __builtin_amdgcn_exp2f(-left);
    A = off ? NAN : -(sum + ge * (h - ln - static_cast<float>(kLn2) * left)) * is;
    B = -ge * static_cast<float>(kLn2) * is;
  }
  __device__ __forceinline__ float at(float e, float arg) const {
    return e * __builtin_fmaf(B, fmaxf(arg, -1e30f), A);
  }
  // At a logit x whose log probability, in these places, has the gradient g.
  __device__ __forceinline__ float point(float x, float m, float g) const {
    const float logp = fmaxf((x - m) * inv_t - ln, -1e30f);
    return -g * expm1f(logp) - expf(logp) * (sum - g + ge * (logp + h));
  }
};
template <typename E, bool BIAS, int NTH, int KIND>
__global__ void __launch_bounds__(NTH) logprobs_bwd_kernel(
    int V, int64_t ldl, const E* __restrict__ logits, const bf16* __restrict__ bias,
    const int64_t* __restrict__ targets, int64_t ignore, Scale k, int K,
    const int64_t* __restrict__ top_idx, const float* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ g_lp,
    const float* __restrict__ g_ent, const float* __restrict__ g_top, void* out, int64_t ldo,
    int64_t plane) {
  constexpr int W = RowOut<E>::W;
  __shared__ int taken;
  const size_t r = blockIdx.x;
  const Row<E, BIAS, !BIAS> row(logits + r * ldl, bias, V);
  const auto o = out_row<E, KIND>(out, r, ldo, plane, row.head);
  const float inv_t = static_cast<float>(k.inv_t), c = k.c;
  const Stats st(stats + 2 * r, c);
  int64_t t = targets && g_lp ? targets[r] : -1;
  const bool off = targets && g_lp && t != ignore && (t < 0 || t >= V);  // a NaN row
  const bool aim = targets && g_lp && t != ignore && !off;
  const float gl = aim ? g_lp[r] * inv_t : 0.0f;
  float sum = gl;
  if (g_top) {
    float part = 0.0f;
    for (int i = threadIdx.x & 63; i < K; i += 64) part += g_top[r * K + i];
    sum += wave_sum(part) * inv_t;
  }
  const float ge = g_ent ? g_ent[r] * inv_t : 0.0f;
  const LogprobGrad d(st, c, sum, ge, entropy[r], inv_t, off);
  if (threadIdx.x == 0) taken = 0;
  st.n.with_arg(c, [&](auto arg) {
    auto grad = [&](float x) {
      const float a = arg(x);
      return d.at(__builtin_amdgcn_exp2f(a), a);
    };
    source<NTH, 0>(row).each(
        [&](int c, int m, const float (&v)[8]) {
#pragma unroll
          for (int g = 0; g < 8 / W; ++g) {
            float w[W];
#pragma unroll
            for (int e = 0; e < W; ++e) w[e] = grad(v[g * W + e]);
            if (g < m) o.put(c + g * NTH, w);
          }
        },
        [&](int j, float x) { o.put(static_cast<int64_t>(j), grad(x)); });
  });
  __syncthreads();
  if (st.n.empty()) return;  // nothing depends on the row
  if (g_top) {
    for (int i = threadIdx.x; i < K; i += NTH) {
      const int64_t j = top_idx[r * K + i];
      const bool both = aim && j == t;
      if (both) taken = 1;
      const float g = d.point(row.at(j), st.n.m, g_top[r * K + i] * inv_t + (both ? gl : 0.0f));
      o.put(j, off ? NAN : g);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0 && aim && !taken) o.put(t, d.point(row.at(t), st.n.m, gl));
}

// ---- distillation --------------------------------------------------------------------------
// One row: the teacher's weights q of its listed tokens (64 bits: one less their sum is what
// the rest gets), the student's softmax, the loss
//   sum q (ln q - logp) + q_r (ln q_r - ln p_r),  p_r the student's mass off the list,
// and its gradient, with Q = sum q + q_r: p_j Q - q_j at listed words, formed here in 64 bits (a
// student near its teacher leaves a small difference), and at the others
//   p_j Q - q_r p_j / p_r = e_j a,  a = (p_r Q - q_r) / sum of e off the list.
// With the rest the pass goes over the words off the list alone, relative to the largest of these:
// p_r may be smaller than fp32 holds beside the listed words, which join in 64 bits. A student
// that has no word for the rest, by -inf or by a mass that 64 bits hold as 0, is not asked for it.
// A bit per word (with the rest; else per word modulo kBits) marks the listed tokens; one that
// was set before shows that a token may be listed twice.
constexpr int kBits = 32768;
constexpr int kMaxRestVocab = 480000;  // 60 KB of bits
constexpr float kAbsent = 3e38f;       // in the place of a listed word's gradient: not written
constexpr double kLeast = -745.0;      // ln of the smallest positive number of 64 bits

// In shared memory: in registers it would be the first wave's all through the pass, whose held rows
// leave no room for it (128 a thread for four waves a SIMD).
struct Teacher {
  double q[kMaxTop], logq[kMaxTop];
  double total;  // sum q
  int idx[kMaxTop];  // -1: absent
  float x[kMaxTop];  // the student's logits
  float g[kMaxTop];
  float a;
  float scale;  // of an fp16 row
  int twice, some, wrong;
  bool only[kMaxTop];  // a listed word's first mark, where marks are exact
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_max_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}

// Writes the row's gradient times sc; g: of the listed words, kAbsent where there is none or an
// earlier place has the word's.
template <int NTH, typename S, typename O, typename T>
__device__ __forceinline__ void distill_grad(const S& src, int K, const Norm& n, float c, float sc,
                                             float a, const T* idx, const float* g, const O& o) {
  const float asc = a * sc;
  n.with_arg(c, [&](auto arg) {
    src.each(
        [&](int c, int m, const float (&v)[8]) {
          constexpr int W = S::W;
#pragma unroll
          for (int g = 0; g < 8 / W; ++g) {
            float w[W];
#pragma unroll
            for (int e = 0; e < W; ++e) w[e] = __builtin_amdgcn_exp2f(arg(v[g * W + e])) * asc;
            if (g < m) o.put(c + g * NTH, w);
          }
        },
        [&](int j, float x) {
          o.put(static_cast<int64_t>(j), __builtin_amdgcn_exp2f(arg(x)) * asc);
        });
  });
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += NTH) {
    const float w = g[k];
    if (w != kAbsent) o.put(static_cast<int64_t>(idx[k]), w * sc);
  }
}

// GRAD: the row's gradient too while its logits are at hand, times scale[0] (T / count), which
// split rows go without.
template <typename E, bool BIAS, int NTH, int NV, bool REST, bool GRAD, int KIND>
__global__ void __launch_bounds__(NTH, NV == 8 ? 6 : NV == 16 ? 4 : 1) distill_kernel(
    int V, int64_t ldl, const E* __restrict__ logits, const bf16* __restrict__ bias, int K,
    int value_type, const void* __restrict__ values, const int64_t* __restrict__ tokens,
    int64_t ignore, Scale sc, const float* __restrict__ teacher_lse, int words,
    float* __restrict__ loss, float* __restrict__ coef, float* __restrict__ weights,
    const float* __restrict__ scale, int parts, void* out, int64_t ldo, uint32_t* err) {
  extern __shared__ uint32_t bits[];
  __shared__ float sh[2 * (NTH / 64)];
  __shared__ Teacher te;
  const size_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const Row<E, BIAS, !BIAS && (!GRAD || NV > 0)> row(logits + r * ldl, bias, V);
  const auto src = source<NTH, NV>(row);
  for (int i = tid; i < words; i += NTH) bits[i] = 0;
  if (tid == 0) te.twice = 0;
  __syncthreads();
  if (tid < 64) {
    double u[2];
    bool some = false, wrong = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = tid + 64 * h;
      u[h] = -INFINITY;
      float x = 0.0f;
      bool only = false;
      int j = -1;
      if (k < K) {
        const int64_t at = tokens[r * K + k];
        const float v = value_type == kBF16 ? ld(static_cast<const bf16*>(values), r * K + k)
                                            : ld(static_cast<const float*>(values), r * K + k);
        if (at != ignore) {
          if (at < 0 || at >= V) {
            wrong = true;
          } else if (v != -INFINITY) {
            j = static_cast<int>(at);
            u[h] = v * sc.inv_t;
            x = row.at(at);
            const uint32_t bit = static_cast<uint32_t>(j + pad_of(row.head)) %
                                 (static_cast<uint32_t>(words) * 32);
            only = !(atomicOr(&bits[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1);
            if (!only) te.twice = 1;
          }
        }
      }
      te.idx[k] = j;
      te.x[k] = x;
      te.only[k] = only;
      some = some || j >= 0;
    }
    wrong = __any(wrong);
    some = __any(some);
    double norm;
    if constexpr (REST) {
      norm = teacher_lse[r];
    } else {
      const double top = wave_max_d(fmax(u[0], u[1]));
      norm = top + log(wave_sum_d(exp(u[0] - top) + exp(u[1] - top)));
    }
    double all = 0.0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = tid + 64 * h;
      const double logq = u[h] - norm, q = te.idx[k] >= 0 ? exp(logq) : 0.0;
      te.logq[k] = logq;
      te.q[k] = q;
      all += q;
    }
    all = wave_sum_d(all);
    if (tid == 0) {
      te.total = all;
      te.some = some;
      te.wrong = wrong || all > kMostWeight;
    }
  }
  __syncthreads();
  const Norm a = norm_of<NTH, REST>(src, sc.c, reinterpret_cast<const uint8_t*>(bits), sh,
                                    [](int, float) {}, [](int, float) {});
  if (tid < 64) {
    const Sums sums(a, sc);
    bool empty = sums.empty;
    const bool some = te.some, wrong = te.wrong;
    double total = te.total;
    float x[2];
    bool only[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x[h] = te.x[tid + 64 * h];
      only[h] = te.only[tid + 64 * h];
    }
    // Of the whole row's sum: the logit it is relative to and its logarithm.
    double at = 0.0, ln_all = 0.0, ln_rest = 0.0;
    if constexpr (REST) {
      at = sums.at;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (only[h]) at = fmax(at, static_cast<double>(x[h]));
      at = wave_max_d(at);
      const double off = sums.ln_sum(at);
      double sum = 0.0;
      bool nan = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!only[h]) continue;
        sum += exp((x[h] - at) * sc.inv_t);
        nan = nan || x[h] != x[h];
      }
      sum = wave_sum_d(sum) + exp(off);
      empty = at == -INFINITY && !__any(nan);
      ln_all = log(sum);
      ln_rest = off - ln_all;
    }
    double logp[2];
    double part = 0.0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (REST) logp[h] = empty ? -INFINITY : (x[h] - at) * sc.inv_t - ln_all;
      else logp[h] = sums.logp(x[h]);
      const double q = te.q[tid + 64 * h];
      if (q != 0.0) part += q * (te.logq[tid + 64 * h] - logp[h]);
    }
    double l = wave_sum_d(part);
    // e_j a at the words off the list (without the rest: at all).
    float ca = 0.0f;
    if constexpr (REST) {
      double rest = 1.0 - total;
      rest = rest > 0.0 && !sums.empty && !(ln_rest <= kLeast) ? rest : 0.0;
      if (rest != 0.0) l += rest * (log(rest) - ln_rest);
      total += rest;
      if (!sums.empty) ca = static_cast<float>(exp(-sums.ln_e()) * (exp(ln_rest) * total - rest));
    } else {
      if (!empty) ca = static_cast<float>(exp(-sums.ln_e()) * total);
    }
    if (!some) ca = 0.0f, l = 0.0;
    if (wrong) ca = NAN, l = NAN;
    float most = 0.0f;  // of the gradient's magnitudes at listed words
    double mass = 0.0;  // the student's on them
    double sure = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = tid + 64 * h;
      if (k >= K) continue;
      const int j = te.idx[k];
      double w = te.q[k];
      bool first = j >= 0;
      if (te.twice) {
        w = 0.0;
        for (int i = 0; i < K; ++i) {
          const bool same = te.idx[i] == j;
          first = first && !(same && i < k);
          w += same ? te.q[i] : 0.0;
        }
      }
      // A row without a finite logit has no gradient.
      te.g[k] = !first  ? kAbsent
                : wrong ? NAN
                : empty ? 0.0f
                        : static_cast<float>(exp(logp[h]) * total - w);
      if (weights) weights[r * K + k] = te.g[k];
      if (KIND == kSplit && first) {
        most = fmaxf(most, fabsf(te.g[k]));
        if (!REST) {
          mass += exp(logp[h]);
          sure = fmax(sure, logp[h]);
        }
      }
    }
    if constexpr (KIND == kSplit) {
      most = wave_max(most);
      if constexpr (REST) {
        most = fmaxf(most, fabsf(ca) * __builtin_amdgcn_exp2f(sums.left));
      } else {
        // At the others p Q, p at most their mass: one less the listed words', of which the surest
        // may hold nearly all. The difference of what it leaves (fp32 sums, right to some 2^-20) and
        // the other listed words' may fall short of the mass, so 2^-10 more: no value may overflow.
        sure = wave_max_d(sure);
        const double left = -expm1(sure);
        const double others = fmax(left - (wave_sum_d(mass) - exp(sure)), 0.0) + 0x1p-10 * left;
        if (some && !empty) most = fmaxf(most, static_cast<float>(others * total));
      }
      // The largest below 2^15.
      const int up = min(15 - __builtin_amdgcn_frexp_expf(most), 126);
      if (tid == 0) {
        te.scale = ldexpf(1.0f, up);
        if (coef) coef[r] = ldexpf(1.0f, -up);
      }
    }
    if (tid == 0) {
      if (wrong) atomicOr(err, kErrToken);
      loss[2 * r] = static_cast<float>(l);
      loss[2 * r + 1] = some || wrong ? 1.0f : 0.0f;
      if (KIND != kSplit && coef) {
        coef[3 * r] = a.r;
        coef[3 * r + 1] = ca;
        coef[3 * r + 2] = a.safe ? 1.0f : 0.0f;
      }
      te.a = ca;
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    if constexpr (KIND == kSplit) {
      bf16* o = static_cast<bf16*>(out) + r * 3 * ldo;
      distill_grad<NTH>(src, K, a, sc.c, 1.0f, te.a, te.idx, te.g,
                        SplitOut{PlanesOut{o, ldo, row.head}, reinterpret_cast<_Float16*>(o + 2 * ldo),
                                 parts, te.scale});
    } else {
      distill_grad<NTH>(src, K, a, sc.c, scale[0], te.a, te.idx, te.g,
                        out_row<E, KIND>(out, r, ldo, 0, row.head));
    }
  }
}

template <typename E, int NTH>
__global__ void __launch_bounds__(NTH) distill_bwd_kernel(
    int V, int64_t ldl, const E* __restrict__ logits, int K, const int64_t* __restrict__ tokens,
    float c, const float* __restrict__ coef, const float* __restrict__ weights,
    const float* __restrict__ scale, const float* __restrict__ grad, int done, E* __restrict__ out) {
  if (done && grad[0] == 1.0f) return;  // the rows are there
  const size_t r = blockIdx.x;
  const Norm n{0.0f, coef[3 * r], 0.0, 0.0, coef[3 * r + 2] != 0.0f};
  const Row<E, false, true> row(logits + r * ldl, nullptr, V);
  distill_grad<NTH>(source<NTH, 0>(row), K, n, c, scale[0] * grad[0], coef[3 * r + 1],
                    tokens + r * K, weights + r * K, RowOut<E>{out + r * V, row.head});
}

// ---- rows of few words ---------------------------------------------------------------------
// Vocabularies of up to kNarrow words (tens of them in character and group workloads): 16 lanes
// take a row, NV values a lane in registers, 16 rows a block. What a row costs beside its logits
// (reductions of 4 lane exchanges, the teacher's exponentials, the logarithms) is shared by the
// four rows of a wave. 262144 rows of 60 fp32, a wave a row as above -> 16 lanes a row, us: log
// probabilities 202 -> 35, with alternatives 371 -> 110, backward 172 -> 35; distillation with 8
// listed tokens 347 -> 75, with the rest 421 -> 99, backward 121 -> 30. The logits are 63 MB, 12 us at
// the rate of a copy (24 for a backward): vector instructions bound the forward kernels, 311 a wave
// of four rows, 1010 with alternatives, 704 and 914 in distillation, which keep the units busy 90 to
// 100% of the time (SQ_INSTS_VALU, SQ_ACTIVE_INST_VALU).
constexpr int kNarrow = 128;

template <typename Op>
__device__ __forceinline__ float reduce16(float v, Op op) {
  v = op(v, dpp_mov<0xB1, 0xF>(v, v));   // quad_perm [1,0,3,2]
  v = op(v, dpp_mov<0x4E, 0xF>(v, v));   // quad_perm [2,3,0,1]
  v = op(v, dpp_mov<0x141, 0xF>(v, v));  // row_half_mirror
  return op(v, dpp_mov<0x140, 0xF>(v, v));  // row_mirror
}
__device__ __forceinline__ float sum16(float v) {
  return reduce16(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float max16(float v) {
  return reduce16(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int CTRL>
__device__ __forceinline__ double dpp_mov_d(double x) {
  uint64_t u = __builtin_bit_cast(uint64_t, x);
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xF, 0xF, false);
  u = static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo);
  return __builtin_bit_cast(double, u);
}
template <typename Op>
__device__ __forceinline__ double reduce16_d(double v, Op op) {
  v = op(v, dpp_mov_d<0xB1>(v));
  v = op(v, dpp_mov_d<0x4E>(v));
  v = op(v, dpp_mov_d<0x141>(v));
  return op(v, dpp_mov_d<0x140>(v));
}
__device__ __forceinline__ double sum16_d(double v) {
  return reduce16_d(v, [](double a, double b) { return a + b; });
}

// A lane's values of its row, words lane, lane + 16, ...; -inf behind the last.
template <typename E, int NV>
struct Narrow {
  int lane;
  size_t r;
  bool live;
  float x[NV];
  __device__ __forceinline__ Narrow(int64_t rows, int V, int64_t ldl, const E* logits,
                                    const bf16* bias) {
    lane = threadIdx.x & 15;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    live = row < rows;
    r = static_cast<size_t>(live ? row : rows - 1);  // all lanes take part in the exchanges
    const E* p = logits + r * ldl;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = lane + 16 * i;
      x[i] = j < V ? ld(p, j) + (bias ? bf2f(bias[j]) : 0.0f) : -INFINITY;
    }
  }
  // The sums beside the row's largest logit; off: of the words that are not listed.
  template <typename Off>
  __device__ __forceinline__ Norm norm(float c, Off off) const {
    float m = kLowest;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = off(i) ? fmaxf(m, x[i]) : m;
    m = max16(m);
    float s = 0.0f, u = 0.0f, ties = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool tie = off(i) && x[i] == m;
      const float a = Share<true>::arg(off(i) && !tie ? x[i] : -INFINITY, m, c);
      const float e = __builtin_amdgcn_exp2f(a);
      ties += tie ? 1.0f : 0.0f;
      s += e;
      u = __builtin_fmaf(e, fmaxf(a, -1e30f), u);
    }
    ties = sum16(ties);
    return Norm{ties > 0.0f ? m : -INFINITY, m,
                static_cast<double>(sum16(s)) + fmaxf(ties - 1.0f, 0.0f), sum16(u), true};
  }
  __device__ __forceinline__ Norm norm(float c) const {
    return norm(c, [](int) { return true; });
  }
};

template <typename E, int NV>
__global__ void __launch_bounds__(256) logprobs_narrow_kernel(
    int64_t rows, int V, int64_t ldl, const E* __restrict__ logits, const bf16* __restrict__ bias,
    const int64_t* __restrict__ targets, int64_t ignore, Scale k, int K,
    float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ stats,
    float* __restrict__ top_lp, int64_t* __restrict__ top_idx, uint32_t* err) {
  __shared__ __attribute__((aligned(16))) uint32_t keys[16][16 * NV];
  const Narrow<E, NV> w(rows, V, ldl, logits, bias);
  const Norm n = w.norm(k.c);
  const Sums sums(n, k);
  auto lp = [&](float x) { return static_cast<float>(sums.logp(x)); };
  if (w.live && w.lane == 0) {
    entropy[w.r] = static_cast<float>(sums.h);
    if (stats) put_stats(stats + 2 * w.r, n, sums);
  }
  if (logprob) {
    const int64_t t = targets[w.r];
    const bool inside = t >= 0 && t < V && t != ignore;
    if (w.live && w.lane == 0 && !inside) {
      if (t != ignore) atomicOr(err, kErrToken);
      logprob[w.r] = t == ignore ? 0.0f : NAN;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (w.live && inside && t == w.lane + 16 * i) logprob[w.r] = lp(w.x[i]);
  }
  if (K == 0) return;
  // A word's place is the number of words before it: of larger logits, or equal and earlier.
  uint32_t mine[NV];
  int rank[NV];
  const int g = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = w.lane + 16 * i;
    mine[i] = j < V ? key_of(w.x[i]) : 0;  // below every word's
    rank[i] = 0;
    keys[g][j] = mine[i];
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < NV; ++h) {  // words 16 h .. 16 h + 15, all before or behind the others' own
    if (16 * h >= V) break;
#pragma unroll
    for (int j0 = 0; j0 < 16; j0 += 4) {
      const u32x4 four = *reinterpret_cast<const u32x4*>(&keys[g][16 * h + j0]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t key = four[q];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (h < i) rank[i] += key >= mine[i];
          else if (h > i) rank[i] += key > mine[i];
          else rank[i] += key + (j0 + q < w.lane) > mine[i];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = w.lane + 16 * i;
    if (w.live && j < V && rank[i] < K) {
      const float x = w.x[i] > -INFINITY ? w.x[i] : -INFINITY;
      top_lp[w.r * K + rank[i]] = lp(x);
      top_idx[w.r * K + rank[i]] = j;
    }
  }
}

template <typename E, int NV, int KIND>
__global__ void __launch_bounds__(256) logprobs_narrow_bwd_kernel(
    int64_t rows, int V, int64_t ldl, const E* __restrict__ logits, const bf16* __restrict__ bias,
    const int64_t* __restrict__ targets, int64_t ignore, Scale k, int K,
    const int64_t* __restrict__ top_idx, const float* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ g_lp,
    const float* __restrict__ g_ent, const float* __restrict__ g_top, void* out, int64_t ldo,
    int64_t plane) {
  const Narrow<E, NV> w(rows, V, ldl, logits, bias);
  const float inv_t = static_cast<float>(k.inv_t);
  const Stats st(stats + 2 * w.r, k.c);
  const int64_t t = targets && g_lp ? targets[w.r] : ignore;
  const bool off = t != ignore && (t < 0 || t >= V), aim = t != ignore && !off;
  const float gl = aim ? g_lp[w.r] * inv_t : 0.0f;
  float point[NV];
  float sum = gl;
#pragma unroll
  for (int i = 0; i < NV; ++i) point[i] = aim && t == w.lane + 16 * i ? gl : 0.0f;
  if (g_top) {
    for (int q = 0; q < K; ++q) {
      const float g = g_top[w.r * K + q] * inv_t;
      const int64_t j = top_idx[w.r * K + q];
      sum += g;
#pragma unroll
      for (int i = 0; i < NV; ++i) point[i] += j == w.lane + 16 * i ? g : 0.0f;
    }
  }
  const float ge = g_ent ? g_ent[w.r] * inv_t : 0.0f;
  const LogprobGrad d(st, k.c, sum, ge, entropy[w.r], inv_t, off);
  const auto o = out_row<E, KIND>(out, w.r, ldo, plane, 0);
  float target = 0.0f;  // the gradient there, once for the four rows of a wave
  if (!g_top) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) x = point[i] != 0.0f ? w.x[i] : x;
    target = d.point(x, st.n.m, gl);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = w.lane + 16 * i;
    const float a = Share<true>::arg(w.x[i], st.n.r, k.c);
    float g = d.at(__builtin_amdgcn_exp2f(a), a);
    if (g_top) {
      if (point[i] != 0.0f) g = d.point(w.x[i], st.n.m, point[i]);
    } else {
      g = point[i] != 0.0f ? target : g;
    }
    if (off) g = NAN;
    else if (st.n.empty()) g = 0.0f;
    if (w.live && j < V) o.put(static_cast<int64_t>(j), g);
  }
}

// A lane takes up to `kEntries` of the list's entries: lane, lane + 16, ... A listed word twice is
// found by its bit; then the list is gone through for each of its places.
template <typename E, int NV, int kEntries, bool REST>
__global__ void __launch_bounds__(256) distill_narrow_kernel(
    int64_t rows, int V, int64_t ldl, const E* __restrict__ logits, const bf16* __restrict__ bias,
    int K, int value_type, const void* __restrict__ values, const int64_t* __restrict__ tokens,
    int64_t ignore, Scale sc, const float* __restrict__ teacher_lse, float* __restrict__ loss,
    float* __restrict__ coef, float* __restrict__ weights, uint32_t* err) {
  __shared__ int lists[16][16 * kEntries];  // -1: absent
  __shared__ float xs[16][16 * NV];
  __shared__ uint32_t marks[16][kNarrow / 32];
  const Narrow<E, NV> w(rows, V, ldl, logits, bias);
  const int g = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < NV; ++i) xs[g][w.lane + 16 * i] = w.x[i];
  if (w.lane < kNarrow / 32) marks[g][w.lane] = 0;
  __syncthreads();
  auto value = [&](int k) {
    return value_type == kBF16 ? ld(static_cast<const bf16*>(values), w.r * K + k)
                               : ld(static_cast<const float*>(values), w.r * K + k);
  };
  float top = -INFINITY;
  float flags = 0.0f;  // 1: an entry, 1024: one out of range
  float twice = 0.0f;
  float val[kEntries];
  int word[kEntries];
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    const int k = w.lane + 16 * i;
    word[i] = -1;
    val[i] = 0.0f;
    if (k >= K) continue;
    const int64_t at = tokens[w.r * K + k];
    val[i] = value(k);
    if (at != ignore) {
      if (at < 0 || at >= V) {
        flags += 1024.0f;
      } else if (val[i] != -INFINITY) {
        const int j = static_cast<int>(at);
        word[i] = j;
        flags += 1.0f;
        top = fmaxf(top, val[i]);
        if (atomicOr(&marks[g][j >> 5], 1u << (j & 31)) >> (j & 31) & 1) twice = 1.0f;
      }
    }
    lists[g][k] = word[i];
  }
  flags = sum16(flags);
  top = max16(top);
  twice = max16(twice);
  __syncthreads();  // the words, their marks
  const Norm n = w.norm(sc.c);
  double norm;
  if constexpr (REST) {
    norm = teacher_lse[w.r];
  } else {
    double all = 0.0;
#pragma unroll
    for (int i = 0; i < kEntries; ++i)
      if (word[i] >= 0) all += exp((static_cast<double>(val[i]) - top) * sc.inv_t);
    norm = top * sc.inv_t + log(sum16_d(all));
  }
  const Sums sums(n, sc);
  double part = 0.0, total = 0.0;
  double q[kEntries], logp[kEntries];
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    q[i] = logp[i] = 0.0;
    if (word[i] < 0) continue;
    const double logq = val[i] * sc.inv_t - norm;
    q[i] = exp(logq);
    logp[i] = sums.logp(xs[g][word[i]]);
    if (q[i] != 0.0) part += q[i] * (logq - logp[i]);
    total += q[i];
  }
  part = sum16_d(part);
  total = sum16_d(total);
  const bool wrong = flags >= 1024.0f || total > kMostWeight, some = flags > 0.0f;
  float r = n.r;
  double a = sums.empty ? 0.0 : exp(-sums.ln_e()) * total;
  if constexpr (REST) {
    uint32_t listed = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = w.lane + 16 * i;
      listed |= (marks[g][j >> 5] >> (j & 31) & 1) << i;
    }
    const Norm off = w.norm(sc.c, [&](int i) { return !(listed >> i & 1); });
    const Sums others(off, sc);
    const double ln_rest = others.ln_sum(sums.at) - sums.ln;
    double rest = 1.0 - total;
    rest = rest > 0.0 && !others.empty && !(ln_rest <= kLeast) ? rest : 0.0;
    if (rest != 0.0) part += rest * (log(rest) - ln_rest);
    total += rest;
    r = off.r;
    a = others.empty ? 0.0 : exp(-others.ln_e()) * (exp(ln_rest) * total - rest);
  }
  if (weights && w.live) {
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int k = w.lane + 16 * i;
      if (k >= K) continue;
      double sum = q[i];
      bool first = word[i] >= 0;
      if (first && twice != 0.0f) {
        sum = 0.0;
        for (int h = 0; h < K; ++h) {
          if (lists[g][h] != word[i]) continue;
          first = first && h >= k;
          sum += exp(value(h) * sc.inv_t - norm);
        }
      }
      // A row without a finite logit has no gradient.
      weights[w.r * K + k] = !first      ? kAbsent
                             : wrong     ? NAN
                             : sums.empty ? 0.0f
                                         : static_cast<float>(exp(logp[i]) * total - sum);
    }
  }
  if (!w.live || w.lane != 0) return;
  if (!some) a = 0.0, part = 0.0;
  if (wrong) {
    a = NAN, part = NAN;
    atomicOr(err, kErrToken);
  }
  loss[2 * w.r] = static_cast<float>(part);
  loss[2 * w.r + 1] = some || wrong ? 1.0f : 0.0f;
  if (coef) {
    coef[3 * w.r] = r;
    coef[3 * w.r + 1] = static_cast<float>(a);
    coef[3 * w.r + 2] = 1.0f;  // differences first
  }
}

template <typename E, int NV>
__global__ void __launch_bounds__(256) distill_narrow_bwd_kernel(
    int64_t rows, int V, int64_t ldl, const E* __restrict__ logits, int K,
    const int64_t* __restrict__ tokens, float c, const float* __restrict__ coef,
    const float* __restrict__ weights, const float* __restrict__ scale,
    const float* __restrict__ grad, E* __restrict__ out) {
  __shared__ float point[16][16 * NV];  // the listed words' gradients
  const Narrow<E, NV> w(rows, V, ldl, logits, nullptr);
  float* mine = point[threadIdx.x >> 4];
#pragma unroll
  for (int i = 0; i < NV; ++i) mine[w.lane + 16 * i] = kAbsent;
  __syncthreads();
  for (int k = w.lane; k < K; k += 16) {
    const float g = weights[w.r * K + k];
    if (g != kAbsent) mine[tokens[w.r * K + k]] = g;
  }
  __syncthreads();
  const float r = coef[3 * w.r], a = coef[3 * w.r + 1];
  const float sc = scale[0] * grad[0];
  if (!w.live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = w.lane + 16 * i;
    const float e = __builtin_amdgcn_exp2f(Share<true>::arg(w.x[i], r, c));
    const float g = mine[j];
    if (j < V) st(out, w.r * V + j, g != kAbsent ? g * sc : e * (a * sc));
  }
}

// Many rows: loss[b kMeanRows] = the sums of the rows' losses and marks from there on to the next
// one's, summed in 64 bits; the result, a mean in fp32, bears the one rounding of each. 262144 rows
// take 9 us in both kernels, 30 in the one block below alone.
constexpr int64_t kMeanRows = 4096;
__global__ void __launch_bounds__(256) distill_parts_kernel(int64_t rows, float* loss) {
  __shared__ double sh[2][4];
  float2* pairs = reinterpret_cast<float2*>(loss) + blockIdx.x * kMeanRows;
  const int n = static_cast<int>(min(kMeanRows, rows - blockIdx.x * kMeanRows));
  double l = 0.0, m = 0.0;
#pragma unroll 16
  for (int r = threadIdx.x; r < n; r += 256) {
    const float2 p = pairs[r];
    l += p.x;
    m += p.y;
  }
  l = wave_sum_d(l);
  m = wave_sum_d(m);
  if ((threadIdx.x & 63) == 0) {
    sh[0][threadIdx.x >> 6] = l;
    sh[1][threadIdx.x >> 6] = m;
  }
  __syncthreads();  // all rows have been read
  if (threadIdx.x == 0)
    pairs[0] = make_float2(static_cast<float>(sh[0][0] + sh[0][1] + sh[0][2] + sh[0][3]),
                           static_cast<float>(sh[1][0] + sh[1][1] + sh[1][2] + sh[1][3]));
}

// mean = weight T^2 * sum of loss[r][0] / max(1, sum of loss[r][1]), factor = weight T / that count,
// over the rows r = 0, step, ...; the sums in 64 bits and a fixed order, one block.
__global__ void __launch_bounds__(1024) distill_mean_kernel(int64_t rows, int64_t step,
                                                            const float* __restrict__ loss,
                                                            double t, double weight,
                                                            float* __restrict__ mean,
                                                            float* __restrict__ factor) {
  __shared__ double sh[2][16];
  double l = 0.0, n = 0.0;
  const float2* pairs = reinterpret_cast<const float2*>(loss);
#pragma unroll 16
  for (int64_t r = threadIdx.x * step; r < rows; r += 1024 * step) {
    const float2 p = pairs[r];
    l += p.x;
    n += p.y;
  }
  l = wave_sum_d(l);
  n = wave_sum_d(n);
  if ((threadIdx.x & 63) == 0) {
    sh[0][threadIdx.x >> 6] = l;
    sh[1][threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = n = 0.0;
    for (int w = 0; w < 16; ++w) {
      l += sh[0][w];
      n += sh[1][w];
    }
    n = n < 1.0 ? 1.0 : n;
    const double wt = weight * t;
    if (mean) mean[0] = static_cast<float>(wt * t * l / n);
    if (factor) factor[0] = static_cast<float>(wt / n);
  }
}

// loss[r] = (0, 1) for rows that the mean counts, (0, 0) for the others: with the kernel above
// the factor T / count before any logits are there. A wave takes a row.
__global__ void __launch_bounds__(256) distill_rows_kernel(int64_t rows, int V, int K, int value_type,
                                                           const void* __restrict__ values,
                                                           const int64_t* __restrict__ tokens,
                                                           int64_t ignore, float* __restrict__ loss) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  bool some = false;
  for (int k = threadIdx.x & 63; k < K; k += 64) {
    const int64_t at = tokens[r * K + k];
    const float v = value_type == kBF16 ? ld(static_cast<const bf16*>(values), r * K + k)
                                        : ld(static_cast<const float*>(values), r * K + k);
    some = some || (at != ignore && (v != -INFINITY || at < 0 || at >= V));
  }
  some = __any(some);
  if ((threadIdx.x & 63) == 0) {
    loss[2 * r] = 0.0f;
    loss[2 * r + 1] = some ? 1.0f : 0.0f;
  }
}

// part[b][c] = the sum over the rows b * kSumRows + 0 .. of column c of bf16 rows x (stride ld), or of
// the two planes of split rows.
constexpr int kSumRows = 64;
template <bool SPLIT>
__global__ void __launch_bounds__(256) column_sums_kernel(int64_t rows, int V, int64_t ld,
                                                          const uint16_t* __restrict__ x,
                                                          float* __restrict__ part) {
  const unsigned strips = (V + 2047) / 2048, b = blockIdx.x / strips;
  const int c = ((blockIdx.x - b * strips) * 256 + threadIdx.x) * 8;
  if (c >= V) return;
  const int64_t r0 = static_cast<int64_t>(b) * kSumRows, r1 = min(rows, r0 + kSumRows);
  float sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) sum[k] = 0.0f;
#pragma unroll 8
  for (int64_t r = r0; r < r1; ++r) {  // the stride is a multiple of 8: whole vectors
    float v[8];
    uint32_t u[4];
    const uint16_t* p = x + r * ld * (SPLIT ? 3 : 1) + c;
    __builtin_memcpy(u, __builtin_assume_aligned(p, 16), 16);
    halves<8>(u, v);
    if constexpr (SPLIT) {
      float w[8];
      __builtin_memcpy(u, __builtin_assume_aligned(p + ld, 16), 16);
      halves<8>(u, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += w[k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += c + k < V ? v[k] : 0.0f;
  }
  float* o = part + static_cast<size_t>(b) * V + c;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (c + k < V) o[k] = sum[k];
}
__global__ void __launch_bounds__(256) add_parts_kernel(int64_t parts, int V,
                                                        const float* __restrict__ part, int add,
                                                        float* __restrict__ out) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= V) return;
  float s = add ? out[c] : 0.0f;
#pragma unroll 8
  for (int64_t p = 0; p < parts; ++p) s += part[p * V + c];
  out[c] = s;
}

// bf16 values as fp16 ones times a power of two that takes the largest to [2^14, 2^15): those down
// to 2^-31 of the largest keep their 8 bits, the error of a smaller one is below 2^-39 of it. The
// first kernel (after the word is cleared) finds the largest finite magnitude, as the bits of a
// float; the second copies and leaves 1 / the power.
__global__ void clear_word_kernel(uint32_t* word) { *word = 0; }
__global__ void __launch_bounds__(256) largest_kernel(int64_t n, const bf16* __restrict__ x,
                                                      uint32_t* __restrict__ word) {
  uint32_t m = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * 8;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n; i += step) {
    bf16 u[8];
    if (i + 8 <= n) {
      __builtin_memcpy(u, __builtin_assume_aligned(x + i, 16), 16);
    } else {
      for (int k = 0; k < 8; ++k) u[k] = i + k < n ? x[i + k] : 0;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t a = u[k] & 0x7fffu;
      m = a < 0x7f80u ? max(m, a) : m;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o, 64)));
  // One atomic a block, and only of a larger value (a stale word costs one more): of every wave's
  // they took 190 us.
  __shared__ uint32_t sh[4];
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    m = max(max(sh[0], sh[1]), max(sh[2], sh[3])) << 16;
    if (m > __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(word, m);
  }
}
__global__ void __launch_bounds__(256) half_copy_kernel(int64_t n, const bf16* __restrict__ x,
                                                        const uint32_t* __restrict__ word,
                                                        _Float16* __restrict__ out,
                                                        float* __restrict__ inverse) {
  // The largest's exponent, a subnormal bf16's as that of the smallest normal one.
  const int e = max(static_cast<int>(*word >> 23), 1) - 127;
  const int shift = *word ? min(14 - e, 126) : 0;
  const float s = ldexpf(1.0f, shift);
  if (blockIdx.x == 0 && threadIdx.x == 0) *inverse = ldexpf(1.0f, -shift);
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * 8;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n; i += step) {
    if (i + 8 <= n) {
      bf16 u[8];
      _Float16 h[8];
      __builtin_memcpy(u, __builtin_assume_aligned(x + i, 16), 16);
#pragma unroll
      for (int k = 0; k < 8; ++k) h[k] = static_cast<_Float16>(bf2f(u[k]) * s);
      __builtin_memcpy(__builtin_assume_aligned(out + i, 16), h, 16);
    } else {
      for (int64_t j = i; j < n; ++j) out[j] = static_cast<_Float16>(bf2f(x[j]) * s);
    }
  }
}

// out[i] = x[i] * the product of up to three device scalars and f, in the type of out: gradients
// held in fp32 from the forward, rounded once.
struct Factors {
  const float* p[3];
  float f;
};
template <typename E>
__global__ void __launch_bounds__(256) scaled_kernel(int64_t n, const float* __restrict__ x,
                                                     Factors g, E* __restrict__ out) {
  constexpr int W = RowOut<E>::W;
  float s = g.f;
#pragma unroll
  for (int k = 0; k < 3; ++k) s *= g.p[k] ? g.p[k][0] : 1.0f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * W;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * W; i < n; i += step) {
    if (i + W <= n) {
      float v[W];
      __builtin_memcpy(v, x + i, 4 * W);
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] *= s;
      RowOut<E>{out + i, 0}.put(0, v);
    } else {
      for (int64_t j = i; j < n; ++j) st(out, j, x[j] * s);
    }
  }
}

static int checks(const char* what, int dtype, int64_t rows, int64_t V, int64_t ldl, double t) {
  DABSN_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: bad dtype %d", what, dtype);
  DABSN_REQUIRE(rows >= 0 && rows < (1ll << 31) && V > 0 && V < (1ll << 31) - 4096 && ldl >= V,
                "%s: bad shape (rows=%lld, V=%lld, ld=%lld)", what, (long long)rows, (long long)V,
                (long long)ldl);
  DABSN_REQUIRE(t >= 1e-6 && t <= 1e6, "%s: temperature %g lies outside [1e-6, 1e6]", what, t);
  return DABSN_OK;
}

// Threads a row: a wave where the row is a few vectors; the whole of a compute unit where no more
// rows than units are there; else 256, of which eight rows share a unit. With 1024 threads (of
// which a unit holds one row or two) against 256, us: 384 rows of 8200 bf16, distillation 15.8 and
// 11.4, log probabilities and their gradient 17.1 and 12.2; of 32000 20.1 and 16.7, 29.1 and 27.8,
// log probabilities with 5 alternatives 18.4 and 14.4; of 128000 36.6 and 37.4, 69 and 76. So
// plain passes (no alternatives, no list) over long rows keep 1024 up to two rows a unit.
static int threads(int64_t rows, int64_t V, bool plain) {
  const int64_t most = plain && V >= 65536 ? 511 : 256;
  return V <= 1024 ? 64 : V >= 8192 && rows <= most ? 1024 : 256;
}

// A launch holds fewer than 2^32 threads: more rows than these run as launches of that many.
constexpr int64_t kMostRows = 1 << 21;
template <typename T>
static T* past(T* p, int64_t n) {
  return p ? p + n : nullptr;
}
static const void* past(const void* p, int dtype, int64_t n) {
  return past(static_cast<const char*>(p), n * (dtype == kBF16 ? 2 : 4));
}
static void* past(void* p, int dtype, int64_t n) {
  return past(static_cast<char*>(p), n * (dtype == kBF16 ? 2 : 4));
}
// launch(first row, rows) for each of them.
template <typename F>
static int in_launches(int64_t rows, F launch) {
  int rc = DABSN_OK;
  for (int64_t s = 0; s < rows && rc == DABSN_OK; s += kMostRows)
    rc = launch(s, std::min(kMostRows, rows - s));
  return rc;
}

}  // namespace vocab
}  // namespace dabsn

using namespace dabsn;
using namespace dabsn::vocab;

#define DABSN_BY_THREADS(M)                     \
  do {                                          \
    if (nth == 64) { M(64); }                   \
    else if (nth == 256) { M(256); }            \
    else { M(1024); }                           \
  } while (0)

extern "C" {

int dabsn_hip_token_logprobs(int dtype, int64_t rows, int64_t V, const void* logits, int64_t ldl,
                             const void* bias, const int64_t* targets, int64_t ignore_index,
                             double temperature, int64_t top, float* logprob, float* entropy,
                             float* stats, float* top_logprobs, int64_t* top_indices,
                             uint32_t* err, hipStream_t stream) {
  int rc = checks("token log probabilities", dtype, rows, V, ldl, temperature);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(top >= 0 && top <= kMaxTop && top <= V,
                "token log probabilities: top %lld of %lld words (at most %d)", (long long)top,
                (long long)V, kMaxTop);
  DABSN_REQUIRE(!bias || dtype == kF32, "token log probabilities: a bias goes with fp32 logits");
  if (rows == 0) return DABSN_OK;
  DABSN_REQUIRE(logits && entropy && err && (!logprob || targets) &&
                    (top == 0 || (top_logprobs && top_indices)),
                "token log probabilities: null pointer");
  if (rows > kMostRows)
    return in_launches(rows, [&](int64_t s, int64_t n) {
      return dabsn_hip_token_logprobs(dtype, n, V, past(logits, dtype, s * ldl), ldl, bias,
                                      past(targets, s), ignore_index, temperature, top,
                                      past(logprob, s), past(entropy, s), past(stats, 2 * s),
                                      past(top_logprobs, s * top), past(top_indices, s * top), err,
                                      stream);
    });
  const int nth = threads(rows, V, top == 0);
  const dim3 grid(static_cast<unsigned>(rows));
  const Scale scale_t = scale_of(temperature);
  const bf16* b = static_cast<const bf16*>(bias);
  if (V <= kNarrow) {
#define DABSN_NARROW(E, NV)                                                                        \
  hipLaunchKernelGGL((logprobs_narrow_kernel<E, NV>), dim3(static_cast<unsigned>((rows + 15) / 16)), \
                     dim3(256), 0, stream, rows, (int)V, ldl, static_cast<const E*>(logits), b,      \
                     targets, ignore_index, scale_t, (int)top, logprob, entropy, stats,              \
                     top_logprobs, top_indices, err)
    if (dtype == kBF16) {
      if (V <= 64) DABSN_NARROW(bf16, 4); else DABSN_NARROW(bf16, 8);
    } else {
      if (V <= 64) DABSN_NARROW(float, 4); else DABSN_NARROW(float, 8);
    }
#undef DABSN_NARROW
    DABSN_HIP_CHECK(hipGetLastError());
    return DABSN_OK;
  }
#define DABSN_LAUNCH(E, BIAS, N, TOP)                                                          \
  hipLaunchKernelGGL((logprobs_kernel<E, BIAS, N, TOP>), grid, dim3(N), 0, stream, (int)V, ldl, \
                     static_cast<const E*>(logits), b, targets, ignore_index, scale_t, (int)top,  \
                     logprob, entropy, stats, top_logprobs, top_indices, err)
#define DABSN_ROWS(N)                                                                          \
  if (dtype == kBF16) {                                                                        \
    if (top) DABSN_LAUNCH(bf16, false, N, true); else DABSN_LAUNCH(bf16, false, N, false);      \
  } else if (b) {                                                                              \
    if (top) DABSN_LAUNCH(float, true, N, true); else DABSN_LAUNCH(float, true, N, false);      \
  } else {                                                                                     \
    if (top) DABSN_LAUNCH(float, false, N, true); else DABSN_LAUNCH(float, false, N, false);    \
  }
  DABSN_BY_THREADS(DABSN_ROWS);
#undef DABSN_ROWS
#undef DABSN_LAUNCH
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

int dabsn_hip_token_logprobs_bwd(int dtype, int64_t rows, int64_t V, const void* logits,
                                 int64_t ldl, const void* bias, const int64_t* targets,
                                 int64_t ignore_index, double temperature, int64_t top,
                                 const int64_t* top_indices, const float* stats,
                                 const float* entropy, const float* g_logprob,
                                 const float* g_entropy, const float* g_top, void* out,
                                 int64_t ldo, int64_t plane, hipStream_t stream) {
  int rc = checks("token log probabilities backward", dtype, rows, V, ldl, temperature);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(top >= 0 && top <= kMaxTop && top <= V && ldo >= V && plane >= 0 &&
                    (plane == 0 || (dtype == kF32 && plane >= rows * ldo)) &&
                    (!bias || dtype == kF32),
                "token log probabilities backward: bad arguments");
  if (rows == 0) return DABSN_OK;
  DABSN_REQUIRE(logits && stats && entropy && out && (!g_logprob || targets) &&
                    (!g_top || (top > 0 && top_indices)),
                "token log probabilities backward: null pointer");
  if (rows > kMostRows)
    return in_launches(rows, [&](int64_t s, int64_t n) {
      return dabsn_hip_token_logprobs_bwd(
          dtype, n, V, past(logits, dtype, s * ldl), ldl, bias, past(targets, s), ignore_index,
          temperature, top, past(top_indices, s * top), past(stats, 2 * s), past(entropy, s),
          past(g_logprob, s), past(g_entropy, s), past(g_top, s * top),
          past(out, plane ? kBF16 : dtype, s * ldo), ldo, plane, stream);
    });
  const int nth = threads(rows, V, true);
  const dim3 grid(static_cast<unsigned>(rows));
  const Scale scale_t = scale_of(temperature);
  const bf16* b = static_cast<const bf16*>(bias);
  if (V <= kNarrow) {
#define DABSN_NARROW(E, NV, KIND)                                                                  \
  hipLaunchKernelGGL((logprobs_narrow_bwd_kernel<E, NV, KIND>),                                    \
                     dim3(static_cast<unsigned>((rows + 15) / 16)), dim3(256), 0, stream, rows,    \
                     (int)V, ldl, static_cast<const E*>(logits), b, targets, ignore_index, scale_t, \
                     (int)top, top_indices, stats, entropy, g_logprob, g_entropy, g_top, out, ldo,  \
                     plane)
    if (dtype == kBF16) {
      if (V <= 64) DABSN_NARROW(bf16, 4, kRows); else DABSN_NARROW(bf16, 8, kRows);
    } else if (plane) {
      if (V <= 64) DABSN_NARROW(float, 4, kPlanes); else DABSN_NARROW(float, 8, kPlanes);
    } else {
      if (V <= 64) DABSN_NARROW(float, 4, kRows); else DABSN_NARROW(float, 8, kRows);
    }
#undef DABSN_NARROW
    DABSN_HIP_CHECK(hipGetLastError());
    return DABSN_OK;
  }
#define DABSN_LAUNCH(E, BIAS, N, KIND)                                                           \
  hipLaunchKernelGGL((logprobs_bwd_kernel<E, BIAS, N, KIND>), grid, dim3(N), 0, stream, (int)V, \
                     ldl, static_cast<const E*>(logits), b, targets, ignore_index, scale_t,         \
                     (int)top, top_indices, stats, entropy, g_logprob, g_entropy, g_top, out,     \
                     ldo, plane)
#define DABSN_ROWS(N)                                                                             \
  if (dtype == kBF16) {                                                                           \
    DABSN_LAUNCH(bf16, false, N, kRows);                                                          \
  } else if (b) {                                                                                 \
    if (plane) DABSN_LAUNCH(float, true, N, kPlanes); else DABSN_LAUNCH(float, true, N, kRows);    \
  } else {                                                                                        \
    if (plane) DABSN_LAUNCH(float, false, N, kPlanes); else DABSN_LAUNCH(float, false, N, kRows);  \
  }
  DABSN_BY_THREADS(DABSN_ROWS);
#undef DABSN_ROWS
#undef DABSN_LAUNCH
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

static int distill_checks(const char* what, int dtype, int64_t rows, int64_t V, int64_t ldl,
                          int64_t top, double temperature) {
  int rc = checks(what, dtype, rows, V, ldl, temperature);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(top > 0 && top <= kMaxTop, "%s: %lld listed tokens a row (1 to %d)", what,
                (long long)top, kMaxTop);
  return DABSN_OK;
}

int dabsn_hip_distill_rows(int64_t rows, int64_t V, int64_t top, int value_dtype,
                           const void* values, const int64_t* tokens, int64_t ignore_index,
                           float* loss, hipStream_t stream) {
  int rc = distill_checks("distillation rows", kF32, rows, V, V, top, 1.0);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(value_dtype == kF32 || value_dtype == kBF16, "distillation rows: bad dtype %d",
                value_dtype);
  if (rows == 0) return DABSN_OK;
  DABSN_REQUIRE(values && tokens && loss, "distillation rows: null pointer");
  if (rows > kMostRows)
    return in_launches(rows, [&](int64_t s, int64_t n) {
      return dabsn_hip_distill_rows(n, V, top, value_dtype, past(values, value_dtype, s * top),
                                    past(tokens, s * top), ignore_index, past(loss, 2 * s), stream);
    });
  hipLaunchKernelGGL(distill_rows_kernel, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0,
                     stream, rows, (int)V, (int)top, value_dtype, values, tokens, ignore_index,
                     loss);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

int dabsn_hip_distill_mean(int64_t rows, float* loss, double temperature, double weight, float* mean,
                           float* factor, hipStream_t stream) {
  DABSN_REQUIRE(rows >= 0 && rows < (1ll << 31) && (rows == 0 || loss) && (mean || factor),
                "distillation mean: bad arguments");
  const bool parts = rows > 4 * kMeanRows;
  if (parts)
    hipLaunchKernelGGL(distill_parts_kernel,
                       dim3(static_cast<unsigned>((rows + kMeanRows - 1) / kMeanRows)), dim3(256), 0,
                       stream, rows, loss);
  hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(1024), 0, stream, rows,
                     parts ? kMeanRows : 1, loss, temperature, weight, mean, factor);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

int dabsn_hip_distill(int dtype, int64_t rows, int64_t V, const void* logits, int64_t ldl,
                      const void* bias, int64_t top, int value_dtype, const void* values,
                      const int64_t* tokens, int64_t ignore_index, double temperature,
                      const float* teacher_lse, float* loss, float* coef, float* weights,
                      const float* scale, int split, void* out, int64_t ldo, uint32_t* err,
                      hipStream_t stream) {
  int rc = distill_checks("distillation", dtype, rows, V, ldl, top, temperature);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(value_dtype == kF32 || value_dtype == kBF16, "distillation: bad value dtype %d",
                value_dtype);
  DABSN_REQUIRE(!teacher_lse || V <= kMaxRestVocab,
                "distillation: the rest of more than %d words is not supported (V=%lld)",
                kMaxRestVocab, (long long)V);
  DABSN_REQUIRE(!bias || dtype == kF32, "distillation: a bias goes with fp32 logits");
  DABSN_REQUIRE(!out || (ldo >= V && split >= 0 && split <= 3 &&
                         (split ? dtype == kF32 && (coef || !(split & kPartHalf)) : scale && !bias)),
                "distillation: bad gradient rows");
  if (rows == 0) return DABSN_OK;
  DABSN_REQUIRE(logits && values && tokens && loss && err, "distillation: null pointer");
  if (rows > kMostRows)
    return in_launches(rows, [&](int64_t s, int64_t n) {
      return dabsn_hip_distill(dtype, n, V, past(logits, dtype, s * ldl), ldl, bias, top, value_dtype,
                               past(values, value_dtype, s * top), past(tokens, s * top),
                               ignore_index, temperature, past(teacher_lse, s), past(loss, 2 * s),
                               past(coef, split ? s : 3 * s), past(weights, s * top), scale, split,
                               split ? past(out, kBF16, 3 * s * ldo) : past(out, dtype, s * ldo), ldo,
                               err, stream);
    });
  const int nth = threads(rows, V, false);
  const dim3 grid(static_cast<unsigned>(rows));
  const Scale scale_t = scale_of(temperature);
  const bf16* b = static_cast<const bf16*>(bias);
  const int words = static_cast<int>(((teacher_lse ? V : std::min<int64_t>(V, kBits)) + 7 + 31) / 32);
  if (V <= kNarrow && !out) {
#define DABSN_NARROW(E, NV, NE, REST)                                                              \
  hipLaunchKernelGGL((distill_narrow_kernel<E, NV, NE, REST>),                                     \
                     dim3(static_cast<unsigned>((rows + 15) / 16)), dim3(256), 0, stream, rows,    \
                     (int)V, ldl, static_cast<const E*>(logits), b, (int)top, value_dtype, values,  \
                     tokens, ignore_index, scale_t, teacher_lse, loss, coef, weights, err)
#define DABSN_NE(E, NV, REST) \
  if (top <= 16) DABSN_NARROW(E, NV, 1, REST); else DABSN_NARROW(E, NV, kMaxTop / 16, REST)
#define DABSN_NV(E, REST) \
  if (V <= 64) { DABSN_NE(E, 4, REST); } else { DABSN_NE(E, 8, REST); }
    if (dtype == kBF16) {
      if (teacher_lse) { DABSN_NV(bf16, true); } else { DABSN_NV(bf16, false); }
    } else {
      if (teacher_lse) { DABSN_NV(float, true); } else { DABSN_NV(float, false); }
    }
#undef DABSN_NV
#undef DABSN_NE
#undef DABSN_NARROW
    DABSN_HIP_CHECK(hipGetLastError());
    return DABSN_OK;
  }
#define DABSN_LAUNCH(E, BIAS, N, NV, REST, GRAD, KIND)                                            \
  hipLaunchKernelGGL((distill_kernel<E, BIAS, N, NV, REST, GRAD, KIND>), grid, dim3(N), 4 * words,  \
                     stream, (int)V, ldl, static_cast<const E*>(logits), b, (int)top, value_dtype,  \
                     values, tokens, ignore_index, scale_t, teacher_lse, words, loss, coef, weights, \
                     scale, split, out, ldo, err)
#define DABSN_REST(E, BIAS, N, NV, GRAD, KIND)                    \
  if (teacher_lse) DABSN_LAUNCH(E, BIAS, N, NV, true, GRAD, KIND); \
  else DABSN_LAUNCH(E, BIAS, N, NV, false, GRAD, KIND)
#define DABSN_ROWS(N)                                                                        \
  if (dtype == kBF16) {                                                                      \
    if (out) { DABSN_REST(bf16, false, N, 0, true, kRows); }                                 \
    else { DABSN_REST(bf16, false, N, 0, false, kRows); }                                    \
  } else if (!out) {                                                                         \
    if (b) { DABSN_REST(float, true, N, 0, false, kRows); }                                  \
    else { DABSN_REST(float, false, N, 0, false, kRows); }                                   \
  } else if (split) {                                                                        \
    if (b) { DABSN_REST(float, true, N, 0, true, kSplit); }                                  \
    else { DABSN_REST(float, false, N, 0, true, kSplit); }                                   \
  } else {                                                                                   \
    DABSN_REST(float, false, N, 0, true, kRows);                                             \
  }
  // Held rows: 64 registers a thread, so that four waves share a SIMD.
  const bool hold = out && !split && V > 1024;
  const int64_t nv = V / (dtype == kBF16 ? 8 : 4);
  if (hold && dtype == kBF16 && nv <= 512 * 16) {
    if (nv <= 256 * 8) { DABSN_REST(bf16, false, 256, 8, true, kRows); }
    else if (nv <= 256 * 16) { DABSN_REST(bf16, false, 256, 16, true, kRows); }
    else { DABSN_REST(bf16, false, 512, 16, true, kRows); }
  } else if (hold && dtype == kF32 && nv <= 1024 * 16) {
    if (nv <= 256 * 8) { DABSN_REST(float, false, 256, 8, true, kRows); }
    else if (nv <= 256 * 16) { DABSN_REST(float, false, 256, 16, true, kRows); }
    else if (nv <= 512 * 16) { DABSN_REST(float, false, 512, 16, true, kRows); }
    else { DABSN_REST(float, false, 1024, 16, true, kRows); }
  } else {
    DABSN_BY_THREADS(DABSN_ROWS);
  }
#undef DABSN_ROWS
#undef DABSN_REST
#undef DABSN_LAUNCH
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

int dabsn_hip_distill_bwd(int dtype, int64_t rows, int64_t V, const void* logits, int64_t ldl,
                          int64_t top, const int64_t* tokens, double temperature, const float* coef,
                          const float* weights, const float* scale, const float* grad, int done,
                          void* dlogits, hipStream_t stream) {
  int rc = distill_checks("distillation backward", dtype, rows, V, ldl, top, temperature);
  if (rc != DABSN_OK) return rc;
  if (rows == 0) return DABSN_OK;
  DABSN_REQUIRE(logits && tokens && coef && weights && scale && grad && dlogits,
                "distillation backward: null pointer");
  if (rows > kMostRows)
    return in_launches(rows, [&](int64_t s, int64_t n) {
      return dabsn_hip_distill_bwd(dtype, n, V, past(logits, dtype, s * ldl), ldl, top,
                                   past(tokens, s * top), temperature, past(coef, 3 * s),
                                   past(weights, s * top), scale, grad, done,
                                   past(dlogits, dtype, s * V), stream);
    });
  const int nth = threads(rows, V, false);
  const dim3 grid(static_cast<unsigned>(rows));
  const Scale scale_t = scale_of(temperature);
  if (V <= kNarrow) {
#define DABSN_NARROW(E, NV)                                                                        \
  hipLaunchKernelGGL((distill_narrow_bwd_kernel<E, NV>),                                           \
                     dim3(static_cast<unsigned>((rows + 15) / 16)), dim3(256), 0, stream, rows,    \
                     (int)V, ldl, static_cast<const E*>(logits), (int)top, tokens, scale_t.c, coef, \
                     weights, scale, grad, static_cast<E*>(dlogits))
    if (dtype == kBF16) {
      if (V <= 64) DABSN_NARROW(bf16, 4); else DABSN_NARROW(bf16, 8);
    } else {
      if (V <= 64) DABSN_NARROW(float, 4); else DABSN_NARROW(float, 8);
    }
#undef DABSN_NARROW
    DABSN_HIP_CHECK(hipGetLastError());
    return DABSN_OK;
  }
#define DABSN_LAUNCH(E, N)                                                                       \
  hipLaunchKernelGGL((distill_bwd_kernel<E, N>), grid, dim3(N), 0, stream, (int)V, ldl,           \
                     static_cast<const E*>(logits), (int)top, tokens, scale_t.c, coef, weights, scale, \
                     grad, done, static_cast<E*>(dlogits))
#define DABSN_ROWS(N) \
  if (dtype == kBF16) { DABSN_LAUNCH(bf16, N); } else { DABSN_LAUNCH(float, N); }
  DABSN_BY_THREADS(DABSN_ROWS);
#undef DABSN_ROWS
#undef DABSN_LAUNCH
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

size_t dabsn_hip_column_sums_partials(int64_t rows, int64_t V) {
  return rows <= 0 || V <= 0 ? 0 : static_cast<size_t>((rows + kSumRows - 1) / kSumRows) * V;
}

int dabsn_hip_column_sums(int split, int64_t rows, int64_t V, int64_t ld, const void* x, int add,
                          float* partials, float* out, hipStream_t stream) {
  const int64_t parts = (rows + kSumRows - 1) / kSumRows, strips = (V + 2047) / 2048;
  DABSN_REQUIRE(rows >= 0 && V > 0 && V < (1ll << 31) - 4096 && parts * strips < (1ll << 31) &&
                    ld >= V && ld % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && out &&
                    (rows == 0 || (x && partials)),
                "column sums: bad arguments (rows=%lld, V=%lld, ld=%lld)", (long long)rows,
                (long long)V, (long long)ld);
  const dim3 grid(static_cast<unsigned>(strips * parts));
  if (rows > 0 && split)
    hipLaunchKernelGGL((column_sums_kernel<true>), grid, dim3(256), 0, stream, rows, (int)V, ld,
                       static_cast<const uint16_t*>(x), partials);
  else if (rows > 0)
    hipLaunchKernelGGL((column_sums_kernel<false>), grid, dim3(256), 0, stream, rows, (int)V, ld,
                       static_cast<const uint16_t*>(x), partials);
  hipLaunchKernelGGL(add_parts_kernel, dim3(static_cast<unsigned>((V + 255) / 256)), dim3(256), 0,
                     stream, parts, (int)V, partials, add, out);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

int dabsn_hip_half_copy(int64_t n, const void* x, uint32_t* word, void* out, float* inverse,
                        hipStream_t stream) {
  DABSN_REQUIRE(n >= 0 && word && inverse && (n == 0 || (x && out)) &&
                    reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(out) % 16 == 0,
                "half copy: bad arguments");
  const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((n + 2047) / 2048, 2048))));
  hipLaunchKernelGGL(clear_word_kernel, dim3(1), dim3(1), 0, stream, word);
  hipLaunchKernelGGL(largest_kernel, grid, dim3(256), 0, stream, n, static_cast<const bf16*>(x), word);
  hipLaunchKernelGGL(half_copy_kernel, grid, dim3(256), 0, stream, n, static_cast<const bf16*>(x),
                     word, static_cast<_Float16*>(out), inverse);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

int dabsn_hip_scaled(int dtype, int64_t n, const float* x, const float* s0, const float* s1,
                     const float* s2, float factor, void* out, hipStream_t stream) {
  DABSN_REQUIRE((dtype == kF32 || dtype == kBF16) && n >= 0 && (n == 0 || (x && out)),
                "scaled copy: bad arguments");
  if (n == 0) return DABSN_OK;
  const Factors g{{s0, s1, s2}, factor};
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((n + 2047) / 2048, 1 << 16)));
  if (dtype == kBF16)
    hipLaunchKernelGGL((scaled_kernel<bf16>), grid, dim3(256), 0, stream, n, x, g,
                       static_cast<bf16*>(out));
  else
    hipLaunchKernelGGL((scaled_kernel<float>), grid, dim3(256), 0, stream, n, x, g,
                       static_cast<float*>(out));
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

}  // extern "C"
