// Scaled token embedding and the gradient of its table.
//
// Forward: out[i] = scale * weight[id_i], a copy of rows bound by memory.
// Backward: dweight[v] = scale * (the sum of the rows grad[i] with id_i = v, in token order),
// fp32 sums, one rounding; a row of zeros where no token is v. The order is fixed, so the same
// inputs give the same bits: no float atomics. The tokens are sorted by word (stable, so each
// word's tokens stay in order), the sorted list is cut into pieces of about equal length whatever the
// words' frequencies, a wave sums a piece's rows word by word, and the words of many pieces are
// joined from partial sums, piece after piece.
#include <algorithm>

#include "../../include/dabsn_hip.h"
#include "capi.hpp"
#include "common.hpp"

namespace dabsn {
namespace embed {

constexpr uint32_t kErrToken = 1u;
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// The W = 8 bf16 or 4 fp32 (16 bytes) of a row that a lane takes at a time, at any element alignment:
// raw, as loaded, and as floats. ONCE: the access is marked as not to be kept in the caches, which
// then hold what is read again (the table's rows) and are not written out for what is not: each
// called in a loop of its own, 65536 rows of 4096 bf16 are looked up in 94 us instead of 132 and
// their gradients summed in 107 instead of 140 (called in turn with each other: 131 and 128). Lanes
// take neighbouring 16 bytes, so that such accesses are whole lines.
template <typename E>
struct Vec {
  static constexpr int W = 16 / sizeof(E);
  u32x4 u;
  // The columns c .. c + W - 1 of a row of H: fewer at its end (zeros are read there).
  template <bool ONCE>
  __device__ __forceinline__ void load(const E* row, int c, int H) {
    if (c + W <= H) {
      const u32x4_any* q = reinterpret_cast<const u32x4_any*>(row + c);
      if constexpr (ONCE) u = __builtin_nontemporal_load(q);
      else u = *q;
    } else {
      float v[W];
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = c + k < H ? to_f(row[c + k]) : 0.0f;
      set(v);
    }
  }
  template <bool ONCE>
  __device__ __forceinline__ void store(E* row, int c, int H) const {
    if (c + W <= H) {
      u32x4_any* q = reinterpret_cast<u32x4_any*>(row + c);
      if constexpr (ONCE) __builtin_nontemporal_store(u, q);
      else *q = u;
    } else {
      float v[W];
      get(v);
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (c + k < H) row[c + k] = from_f<E>(v[k]);
    }
  }
  __device__ __forceinline__ void get(float (&v)[W]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t x = u[k];  // a cast of the element itself reads element 0
      if constexpr (W == 8) {
        v[2 * k] = __builtin_bit_cast(float, x << 16);
        v[2 * k + 1] = __builtin_bit_cast(float, x & 0xffff0000u);
      } else {
        v[k] = __builtin_bit_cast(float, x);
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[W]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (W == 8)
        u[k] = static_cast<uint32_t>(f2bf(v[2 * k])) | static_cast<uint32_t>(f2bf(v[2 * k + 1])) << 16;
      else
        u[k] = __builtin_bit_cast(uint32_t, v[k]);
    }
  }
};
template <typename E, bool ONCE, int W>
__device__ __forceinline__ void put(E* row, int c, int H, const float (&v)[W]) {
  static_assert(W == Vec<E>::W, "a lane's values");
  Vec<E> x;
  x.set(v);
  x.template store<ONCE>(row, c, H);
}
// Partial sums: a lane's W fp32 of a row, in two accesses for W = 8.
template <int W>
__device__ __forceinline__ void get_sums(const float* row, int c, int H, float (&v)[W]) {
#pragma unroll
  for (int h = 0; h < W; h += 4) {
    Vec<float> x;
    float w[4];
    x.load<false>(row, c + h, H);
    x.get(w);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[h + k] = w[k];
  }
}
template <int W>
__device__ __forceinline__ void put_sums(float* row, int c, int H, const float (&v)[W]) {
#pragma unroll
  for (int h = 0; h < W; h += 4) {
    const float w[4] = {v[h], v[h + 1], v[h + 2], v[h + 3]};
    put<float, false>(row, c + h, H, w);
  }
}

// A wave takes 64 / lanes rows at a time, `lanes` (a power of two) lanes a row.
template <typename E>
__global__ void __launch_bounds__(256) lookup_kernel(int64_t n, int64_t V, int H, int lanes_log2,
                                                     const int64_t* __restrict__ ids,
                                                     const E* __restrict__ weight, int64_t ldw,
                                                     float scale, E* __restrict__ out,
                                                     uint32_t* err) {
  const int lanes = 1 << lanes_log2;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  constexpr int W = Vec<E>::W;
  if (i >= n) return;
  const int64_t id = ids[i];
  const bool ok = id >= 0 && id < V;
  if (!ok && lane == 0) atomicOr(err, kErrToken);
  const E* w = weight + (ok ? id : 0) * ldw;
  const float s = ok ? scale : NAN;
  E* o = out + i * H;
#pragma unroll 4
  for (int c = lane * W; c < H; c += lanes * W) {
    Vec<E> x;
    float v[W];
    x.template load<false>(w, c, H);
    x.get(v);
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] *= s;
    put<E, true>(o, c, H, v);
  }
}

// ---- stable sort of the tokens by word -----------------------------------------------------
// Tokens that give no gradient (out of range, the padding word) get the key V and come last.
__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t V, int64_t padding) {
  return id < 0 || id >= V || id == padding ? static_cast<uint32_t>(V) : static_cast<uint32_t>(id);
}

// Few tokens: a token's place is the number of tokens before it in the order (key, index),
// counted against all of them in shared memory; four threads share a token's count.
constexpr int kRankTokens = 4096;
__global__ void __launch_bounds__(256) rank_kernel(int n, int64_t V, int64_t padding,
                                                   const int64_t* __restrict__ ids,
                                                   uint32_t* __restrict__ keys,
                                                   uint32_t* __restrict__ pos) {
  __shared__ uint32_t all[kRankTokens];
  for (int j = threadIdx.x; j < n; j += 256) all[j] = key_of(ids[j], V, padding);
  __syncthreads();
  const int i = blockIdx.x * 64 + (threadIdx.x >> 2), part = threadIdx.x & 3;
  const uint32_t mine = i < n ? all[i] : 0;
  int rank = 0;
  for (int j = part; j < n; j += 4) rank += all[j] < mine + (j < i);  // equal and earlier, or less
  rank += __shfl_xor(rank, 1, 64);
  rank += __shfl_xor(rank, 2, 64);
  if (part == 0 && i < n) {
    keys[rank] = mine;
    pos[rank] = static_cast<uint32_t>(i);
  }
}

// Many tokens: passes over digits of `bits` bits, the lowest first. A block counts its tile's
// digits; then each block finds where its tile's digits start (all smaller digits, and the same
// digit in earlier tiles) and places its tokens, 64 at a time a wave, by their rank among equal
// digits: bits ballots.
constexpr int kMaxBits = 10;
template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(int64_t i, int64_t V, int64_t padding,
                                             const int64_t* ids, const uint32_t* keys) {
  if constexpr (FIRST) return key_of(ids[i], V, padding);
  return keys[i];
}
template <bool FIRST>
__global__ void __launch_bounds__(256) digits_kernel(int64_t n, int64_t V, int64_t padding, int tile,
                                                     int shift, int bits,
                                                     const int64_t* __restrict__ ids,
                                                     const uint32_t* __restrict__ keys,
                                                     uint32_t* __restrict__ counts) {
  __shared__ uint32_t h[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += 256) h[b] = 0;
  __syncthreads();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * tile, i1 = min(n, i0 + tile);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += 256)
    atomicAdd(&h[sort_key<FIRST>(i, V, padding, ids, keys) >> shift & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 256)
    counts[static_cast<size_t>(blockIdx.x) * bins + b] = h[b];
}
template <bool FIRST>
__global__ void __launch_bounds__(256) place_kernel(int64_t n, int64_t V, int64_t padding, int tile,
                                                    int shift, int bits, int tiles,
                                                    const int64_t* __restrict__ ids,
                                                    const uint32_t* __restrict__ keys,
                                                    const uint32_t* __restrict__ pos,
                                                    const uint32_t* __restrict__ counts,
                                                    uint32_t* __restrict__ keys_out,
                                                    uint32_t* __restrict__ pos_out,
                                                    uint32_t* __restrict__ starts) {
  __shared__ uint32_t at[4][1 << kMaxBits];
  __shared__ uint32_t total[1 << kMaxBits];
  __shared__ uint32_t waves[4];
  const int bins = 1 << bits, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int b = tid; b < bins; b += 256) {
    uint32_t before = 0, all = 0;
#pragma unroll 32
    for (int t = 0; t < tiles; ++t) {
      const uint32_t x = counts[static_cast<size_t>(t) * bins + b];
      before += t < static_cast<int>(blockIdx.x) ? x : 0;
      all += x;
    }
    at[0][b] = before;
    at[1][b] = at[2][b] = at[3][b] = 0;
    total[b] = all;
  }
  __syncthreads();
  // Exclusive sums of the digits' totals: a thread's run of bins, then over lanes and waves.
  const int run = (bins + 255) / 256, b0 = tid * run;
  uint32_t mine = 0;
  for (int b = b0; b < min(b0 + run, bins); ++b) mine += total[b];
  uint32_t up = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = __shfl_up(up, o, 64);
    up += lane >= o ? x : 0;
  }
  if (lane == 63) waves[wave] = up;
  __syncthreads();
  uint32_t start = up - mine;
  for (int w = 0; w < wave; ++w) start += waves[w];
  for (int b = b0; b < min(b0 + run, bins); ++b) {
    at[0][b] += start;
    if (starts && blockIdx.x == 0 && b <= V) starts[b] = start;  // the only pass: digits are words
    start += total[b];
  }
  // The waves' quarters of the tile: counts of the quarters before a wave's own.
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * tile, i1 = min(n, i0 + tile);
  const int quarter = tile / 4;
  const int64_t q0 = i0 + static_cast<int64_t>(wave) * quarter, q1 = min(i1, q0 + quarter);
  if (wave < 3) {
    for (int64_t i = q0 + lane; i < q1; i += 64)
      atomicAdd(&at[wave + 1][sort_key<FIRST>(i, V, padding, ids, keys) >> shift & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = tid; b < bins; b += 256) {
    uint32_t s = at[0][b];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      s += at[w][b];
      at[w][b] = s;
    }
  }
  __syncthreads();
  for (int64_t i = q0; i < q1; i += 64) {
    const bool live = i + lane < q1;
    const uint32_t key = live ? sort_key<FIRST>(i + lane, V, padding, ids, keys) : 0;
    const uint32_t d = key >> shift & (bins - 1);
    uint64_t same = __ballot(live);
    for (int b = 0; b < bits; ++b) {
      const bool one = d >> b & 1;
      const uint64_t with = __ballot(one);
      same &= one ? with : ~with;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const uint32_t from = live ? at[wave][d] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // all lanes have read
    if (live && rank == 0) at[wave][d] = from + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    if (live) {
      keys_out[from + rank] = key;
      pos_out[from + rank] = FIRST ? static_cast<uint32_t>(i + lane) : pos[i + lane];
    }
  }
}

// starts[v] = the first sorted token of a word >= v, v = 0 .. V.
__global__ void __launch_bounds__(256) starts_kernel(uint32_t n, uint32_t V,
                                                     const uint32_t* __restrict__ keys,
                                                     uint32_t* __restrict__ starts) {
  const uint32_t v = blockIdx.x * 256 + threadIdx.x;
  if (v > V) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  starts[v] = lo;
}

// ---- sums ----------------------------------------------------------------------------------
// The sum of the rows `at(i)`, i = i0 .. i1 - 1 in order, over this lane's W columns; U rows' loads
// in flight.
template <int U, typename E, int W, typename At>
__device__ __forceinline__ void add_rows(const E* grad, int H, int c, int i0, int i1, At at,
                                         float (&sum)[W]) {
  for (int i = i0; i < i1; i += U) {
    Vec<E> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c < H) x[u].template load<true>(grad + static_cast<size_t>(at(min(i + u, i1 - 1))) * H, c, H);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < i1) {
        float v[W];
        x[u].get(v);
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] += v[k];
      }
    }
  }
}

// Few tokens and words: a wave takes a word and 64 W columns, finds the word's tokens among all
// and sums their rows, zeros included: one launch instead of four.
constexpr int kDirectTokens = 512;
constexpr int64_t kDirectWork = 1 << 23;  // tokens * words
template <typename E>
__global__ void __launch_bounds__(256) direct_kernel(int n, int64_t V, int64_t padding, int H,
                                                     int strips, int64_t tasks,
                                                     const int64_t* __restrict__ ids,
                                                     const E* __restrict__ grad, float scale,
                                                     E* __restrict__ dweight) {
  constexpr int W = Vec<E>::W;
  __shared__ uint16_t lists[4][kDirectTokens];
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  uint16_t* list = lists[threadIdx.x >> 6];
  const int64_t word = task / strips;  // no word at all behind the last task
  const int c = (static_cast<int>(task - word * strips) * 64 + lane) * W;
  int count = 0;
  for (int i = 0; i < n; i += 64) {
    const bool mine = i + lane < n && ids[i + lane] == word && word != padding && word < V;
    const uint64_t mask = __ballot(mine);
    if (mine) list[count + __popcll(mask & ((1ull << lane) - 1))] = static_cast<uint16_t>(i + lane);
    count += __popcll(mask);
  }
  __syncthreads();
  if (task >= tasks || c >= H) return;
  float sum[W];
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] = 0.0f;
  add_rows<8>(grad, H, c, 0, count, [&](int i) { return list[i]; }, sum);
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] *= scale;
  put<E, true>(dweight + word * H, c, H, sum);
}

// The sorted tokens in pieces of kPiece. A word of at most kPiece tokens belongs to the piece in
// which it begins (so a piece sums fewer than 2 kPiece tokens, and short words, whose sums would
// cost as much to pass on as their rows, cross no piece). A longer word is cut where pieces end:
// it leaves the partial sum of its first piece in slot 2 piece + 1 and those of the next ones in
// slot 2 piece. A wave sums a piece over 64 W columns.
constexpr int kPiece = 32;
template <typename E>
__global__ void __launch_bounds__(256) pieces_kernel(int H, int strips, int64_t tasks, uint32_t V,
                                                     const uint32_t* __restrict__ starts,
                                                     const uint32_t* __restrict__ keys,
                                                     const uint32_t* __restrict__ pos,
                                                     const E* __restrict__ grad, float scale,
                                                     E* __restrict__ dweight,
                                                     float* __restrict__ partial) {
  constexpr int W = Vec<E>::W;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (task >= tasks) return;
  const int lane = threadIdx.x & 63;
  const uint32_t piece = static_cast<uint32_t>(task / strips);
  const int c = (static_cast<int>(task - static_cast<int64_t>(piece) * strips) * 64 + lane) * W;
  const uint32_t n = starts[V];  // tokens that give a gradient
  const uint32_t lo = piece * kPiece, hi = min(n, lo + kPiece);
  if (lo >= n) return;
  // A lane a token, the first ones of the next piece too: its word and where that begins and ends.
  const uint32_t at = lo + lane;
  const uint32_t key = keys[min(at, n - 1)], row = pos[min(at, n - 1)];
  const uint32_t from = starts[key], to = starts[key + 1];
  const bool cut = to - from > kPiece;
  const uint64_t ends = __ballot(at < n && to == at + 1), cuts = __ballot(cut);
  const uint64_t begun = __ballot(from >= lo);
  const int tail = static_cast<int>(hi - lo) - 1;
  const uint32_t first_to = __builtin_amdgcn_readlane(to, 0);
  const uint32_t last_to = __builtin_amdgcn_readlane(to, tail);
  // From behind a short word of the piece before, to the end of the last short word.
  int i = (begun & 1) || (cuts & 1) ? 0 : static_cast<int>(first_to - lo);
  const int end = (cuts >> tail & 1) ? tail + 1 : static_cast<int>(last_to - lo);
  float sum[W];
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] = 0.0f;
  constexpr int U = 8;  // rows' loads in flight, whatever words they belong to
  for (; i < end; i += U) {
    Vec<E> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t r = __builtin_amdgcn_readlane(row, min(i + u, end - 1));
      if (c < H) x[u].template load<true>(grad + r * H, c, H);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = i + u;
      if (j >= end) break;
      float v[W];
      x[u].get(v);
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] += v[k];
      if ((ends >> j & 1) || j + 1 == end) {
        const uint32_t word = __builtin_amdgcn_readlane(key, j);
        if (c < H) {
          if (cuts >> j & 1) {
            const size_t slot = 2 * static_cast<size_t>(piece) + (begun >> j & 1);
            put_sums(partial + slot * H, c, H, sum);
          } else {
#pragma unroll
            for (int k = 0; k < W; ++k) sum[k] *= scale;
            put<E, true>(dweight + static_cast<size_t>(word) * H, c, H, sum);
          }
        }
#pragma unroll
        for (int k = 0; k < W; ++k) sum[k] = 0.0f;
      }
    }
  }
}

// The first `blanks` blocks write the zeros of words without tokens, 64 / lanes words a wave; then
// a block a piece and 64 W columns joins the partial sums of the cut word that begins in the piece,
// if one does (a cut word is longer than a piece, so one at most): its waves take ranges of the
// pieces, added in order.
template <typename E>
__global__ void __launch_bounds__(256) words_kernel(int H, int lanes_log2, int strips, int64_t V,
                                                    int64_t blanks, const uint32_t* __restrict__ starts,
                                                    const uint32_t* __restrict__ keys,
                                                    const float* __restrict__ partial, float scale,
                                                    E* __restrict__ dweight) {
  constexpr int W = Vec<E>::W;
  __shared__ float part[4][64 * W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (blockIdx.x < blanks) {
    const int lanes = 1 << lanes_log2;
    const int64_t v = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> lanes_log2;
    if (v >= V || starts[v] != starts[v + 1]) return;
    float zero[W];
#pragma unroll
    for (int k = 0; k < W; ++k) zero[k] = 0.0f;
    for (int c = (threadIdx.x & (lanes - 1)) * W; c < H; c += lanes * W)
      put<E, true>(dweight + v * H, c, H, zero);
    return;
  }
  const int64_t task = blockIdx.x - blanks;
  const uint32_t n = starts[V], piece = static_cast<uint32_t>(task / strips);
  const uint32_t lo = piece * kPiece;
  if (n <= kPiece || lo >= n - kPiece) return;  // no piece behind this one
  const uint32_t word = keys[lo + kPiece - 1], a = starts[word], b = starts[word + 1];
  if (a < lo || b - a <= kPiece) return;
  const uint32_t pieces = (b - 1) / kPiece - piece;  // behind the first
  const uint32_t per = (pieces + 3) / 4, p1 = min(pieces, (wave + 1) * per);
  const int c = (static_cast<int>(task - static_cast<int64_t>(piece) * strips) * 64 + lane) * W;
  float sum[W];
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] = 0.0f;
  if (c < H) {
    if (wave == 0) get_sums(partial + (2 * static_cast<size_t>(piece) + 1) * H, c, H, sum);
#pragma unroll 8
    for (uint32_t p = wave * per; p < p1; ++p) {
      float w[W];
      get_sums(partial + 2 * static_cast<size_t>(piece + 1 + p) * H, c, H, w);
#pragma unroll
      for (int k = 0; k < W; ++k) sum[k] += w[k];
    }
#pragma unroll
    for (int k = 0; k < W; ++k) part[wave][lane * W + k] = sum[k];
  }
  __syncthreads();
  if (wave != 0 || c >= H) return;
#pragma unroll
  for (int g = 1; g < 4; ++g) {
#pragma unroll
    for (int k = 0; k < W; ++k) sum[k] += part[g][lane * W + k];
  }
#pragma unroll
  for (int k = 0; k < W; ++k) sum[k] *= scale;
  put<E, true>(dweight + static_cast<size_t>(word) * H, c, H, sum);
}

// Lanes a row where a wave may share rows: W columns each, a power of two, at most the wave.
static int lanes_log2(int dtype, int64_t H) {
  int l = 0;
  while (l < 6 && ((dtype == kBF16 ? 8ll : 4ll) << l) < H) ++l;
  return l;
}
static int64_t strips_of(int dtype, int64_t H) {
  const int columns = dtype == kBF16 ? 512 : 256;
  return (H + columns - 1) / columns;
}

struct Plan {
  bool direct;
  int bits, passes, tile, tiles;
  int64_t pieces;
  size_t keys, pos, keys2, pos2, counts, starts, partial, bytes;
};
static size_t up(size_t b) { return (b + 255) / 256 * 256; }
static Plan plan_of(int64_t n, int64_t V, int64_t H) {
  Plan p{};
  // (A launch holds fewer than 2^32 threads.)
  p.direct = n <= kDirectTokens && n * V <= kDirectWork && V * strips_of(kF32, H) < (1ll << 25);
  if (p.direct) return p;
  int need = 1;
  while ((1ll << need) <= V) ++need;  // keys 0 .. V
  const bool rank = n <= kRankTokens;
  p.passes = rank ? 0 : (need + kMaxBits - 1) / kMaxBits;
  p.bits = rank ? 0 : (need + p.passes - 1) / p.passes;
  // At most 128 tiles, whose counts every block adds up; a multiple of 256, the waves' rounds.
  p.tile = static_cast<int>(std::max<int64_t>(1024, (n + 127) / 128));
  p.tile = (p.tile + 255) / 256 * 256;
  p.tiles = static_cast<int>((n + p.tile - 1) / p.tile);
  p.pieces = (n + kPiece - 1) / kPiece;
  size_t at = 0;
  auto take = [&](size_t b) { const size_t o = at; at += up(b); return o; };
  p.keys = take(4 * n);
  p.pos = take(4 * n);
  p.keys2 = p.passes > 1 ? take(4 * n) : p.keys;
  p.pos2 = p.passes > 1 ? take(4 * n) : p.pos;
  p.counts = take(p.passes ? 4ull * p.tiles << p.bits : 0);
  p.starts = take(4 * (V + 1));
  p.partial = take(8ull * p.pieces * H);
  p.bytes = at;
  return p;
}

static int checks(const char* what, int dtype, int64_t n, int64_t V, int64_t H) {
  DABSN_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: bad dtype %d", what, dtype);
  DABSN_REQUIRE(n >= 0 && n < (1ll << 31) && V > 0 && V < (1ll << 31) - 256 && H > 0 && H < (1 << 24),
                "%s: bad shape (tokens=%lld, V=%lld, H=%lld)", what, (long long)n, (long long)V,
                (long long)H);
  return DABSN_OK;
}

template <typename E>
static void launch_bwd(const Plan& p, int64_t n, int64_t V, int H, const int64_t* ids, int64_t padding,
                       const E* grad, float scale, E* dweight, char* ws, hipStream_t stream) {
  constexpr int dtype = is_bf16<E>::value ? kBF16 : kF32;
  const int strips = static_cast<int>(strips_of(dtype, H));
  if (p.direct) {
    const int64_t tasks = V * strips;
    hipLaunchKernelGGL((direct_kernel<E>), dim3(static_cast<unsigned>((tasks + 3) / 4)), dim3(256), 0,
                       stream, static_cast<int>(n), V, padding, H, strips, tasks, ids, grad, scale,
                       dweight);
    return;
  }
  auto* keys = reinterpret_cast<uint32_t*>(ws + p.keys);
  auto* pos = reinterpret_cast<uint32_t*>(ws + p.pos);
  auto* counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  auto* starts = reinterpret_cast<uint32_t*>(ws + p.starts);
  auto* partial = reinterpret_cast<float*>(ws + p.partial);
  if (p.passes == 0 && n > 0) {
    hipLaunchKernelGGL(rank_kernel, dim3(static_cast<unsigned>((n + 63) / 64)), dim3(256), 0, stream,
                       static_cast<int>(n), V, padding, ids, keys, pos);
  }
  // Passes alternate between two buffers and end in the first.
  uint32_t *ka = keys, *pa = pos;
  uint32_t *kb = reinterpret_cast<uint32_t*>(ws + p.keys2), *pb = reinterpret_cast<uint32_t*>(ws + p.pos2);
  if (p.passes % 2 == 0) {
    std::swap(ka, kb);
    std::swap(pa, pb);
  }
  for (int s = 0; s < p.passes; ++s) {
    const dim3 grid(static_cast<unsigned>(p.tiles));
    const int shift = s * p.bits;
    if (s == 0) {
      hipLaunchKernelGGL((digits_kernel<true>), grid, dim3(256), 0, stream, n, V, padding, p.tile,
                         shift, p.bits, ids, nullptr, counts);
      hipLaunchKernelGGL((place_kernel<true>), grid, dim3(256), 0, stream, n, V, padding, p.tile,
                         shift, p.bits, p.tiles, ids, nullptr, nullptr, counts, ka, pa,
                         p.passes == 1 ? starts : nullptr);
    } else {
      hipLaunchKernelGGL((digits_kernel<false>), grid, dim3(256), 0, stream, n, V, padding, p.tile,
                         shift, p.bits, ids, kb, counts);
      hipLaunchKernelGGL((place_kernel<false>), grid, dim3(256), 0, stream, n, V, padding, p.tile,
                         shift, p.bits, p.tiles, ids, kb, pb, counts, ka, pa, nullptr);
    }
    std::swap(ka, kb);
    std::swap(pa, pb);
  }
  if (p.passes != 1)
    hipLaunchKernelGGL(starts_kernel, dim3(static_cast<unsigned>(V / 256 + 1)), dim3(256), 0, stream,
                       static_cast<uint32_t>(n), static_cast<uint32_t>(V), keys, starts);
  const int64_t tasks = p.pieces * strips;
  if (tasks > 0)
    hipLaunchKernelGGL((pieces_kernel<E>), dim3(static_cast<unsigned>((tasks + 3) / 4)), dim3(256), 0,
                       stream, H, strips, tasks, static_cast<uint32_t>(V), starts, keys, pos, grad,
                       scale, dweight, partial);
  const int log2 = lanes_log2(dtype, H);
  const int64_t blanks = ((V << log2) + 255) / 256;
  hipLaunchKernelGGL((words_kernel<E>), dim3(static_cast<unsigned>(blanks + tasks)), dim3(256), 0,
                     stream, H, log2, strips, V, blanks, starts, keys, partial, scale, dweight);
}

}  // namespace embed
}  // namespace dabsn

using namespace dabsn;
using namespace dabsn::embed;

extern "C" {

int dabsn_hip_embedding_fwd(int dtype, int64_t n, int64_t V, int64_t H, const int64_t* ids,
                            const void* weight, int64_t ldw, float scale, void* out, uint32_t* err,
                            hipStream_t stream) {
  int rc = checks("embedding", dtype, n, V, H);
  if (rc != DABSN_OK) return rc;
  DABSN_REQUIRE(ldw >= H, "embedding: row stride %lld of %lld values", (long long)ldw, (long long)H);
  if (n == 0) return DABSN_OK;
  DABSN_REQUIRE(ids && weight && out && err, "embedding: null pointer");
  const int log2 = lanes_log2(dtype, H);
  const int64_t blocks = ((n << log2) + 255) / 256;
  DABSN_REQUIRE(blocks < (1ll << 24), "embedding: %lld tokens in one call", (long long)n);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (dtype == kBF16)
    hipLaunchKernelGGL((lookup_kernel<bf16>), grid, dim3(256), 0, stream, n, V, (int)H, log2, ids,
                       static_cast<const bf16*>(weight), ldw, scale, static_cast<bf16*>(out), err);
  else
    hipLaunchKernelGGL((lookup_kernel<float>), grid, dim3(256), 0, stream, n, V, (int)H, log2, ids,
                       static_cast<const float*>(weight), ldw, scale, static_cast<float*>(out), err);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

size_t dabsn_hip_embedding_workspace_bytes(int64_t n, int64_t V, int64_t H) {
  if (n < 0 || n >= (1ll << 31) || V <= 0 || V >= (1ll << 31) - 256 || H <= 0 || H >= (1 << 24)) return 0;
  return plan_of(n, V, H).bytes;
}

int dabsn_hip_embedding_bwd(int dtype, int64_t n, int64_t V, int64_t H, const int64_t* ids,
                            int64_t padding_idx, const void* grad, float scale, void* dweight,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int rc = checks("embedding backward", dtype, n, V, H);
  if (rc != DABSN_OK) return rc;
  const Plan p = plan_of(n, V, H);
  DABSN_REQUIRE(((ids && grad) || n == 0) && dweight && (workspace || p.bytes == 0),
                "embedding backward: null pointer");
  DABSN_REQUIRE(workspace_bytes >= p.bytes, "embedding backward: workspace of %zu bytes, %zu needed",
                workspace_bytes, p.bytes);
  const int64_t strips = strips_of(dtype, H);
  DABSN_REQUIRE(p.pieces * strips + ((V << lanes_log2(dtype, H)) + 255) / 256 < (1ll << 24),
                "embedding backward: %lld x %lld values in one call", (long long)n, (long long)H);
  if (dtype == kBF16)
    launch_bwd<bf16>(p, n, V, (int)H, ids, padding_idx, static_cast<const bf16*>(grad), scale,
                     static_cast<bf16*>(dweight), static_cast<char*>(workspace), stream);
  else
    launch_bwd<float>(p, n, V, (int)H, ids, padding_idx, static_cast<const float*>(grad), scale,
                      static_cast<float*>(dweight), static_cast<char*>(workspace), stream);
  DABSN_HIP_CHECK(hipGetLastError());
  return DABSN_OK;
}

}  // extern "C"
