// logprob.cuh — log probabilities of given tokens, the entropy and the most
// likely tokens of each row of logits, and the gradient of the logits.
//
// With z = scale x over the V columns of a row (fp32 throughout):
//   lse = log sum e^z      logprob = z[target] - lse      H = lse - sum p z
//   gradient, for upstream g (logprob), h (entropy) and l (lse):
//   dx_j = scale (g ([j = target] - p_j) - h p_j (log p_j + H) + l p_j),  p_j = e^(z_j - lse)
// A row of only -inf has no distribution: lse and every log probability are
// -inf, its entropy and its gradient 0. A NaN or +inf makes the row NaN.
//
// The gradient takes z - lse from the row's norm, its maximum m and log2 of s
// (below), as (x - m) scale log2 e - log2 s: off by 2^-24 of |z - m| and of log s.
// From lse, one rounded number, it would be off by 2^-24 |lse|, which is 4e-3 at a
// common offset of 1e5, and everything for a row of the type's lowest value.
//
// Forward reads the logits once: every thread keeps a running maximum m of x,
// s = sum 2^y and t = sum y 2^y with y = (x - m) scale log2 e, and rescales them
// when its maximum grows, so H = ln 2 (log2 s - t / s) needs no second pass.
// (One fused multiply-add per y would be off by the rounding of m scale log2 e:
// a certain token would not get log probability 0.) Bound by memory for 32-bit
// logits; for 16-bit ones the one exponential per value takes about 3/4 of the
// special-function rate that goes with the full read rate.
//
// The top k of a row need hardly any work in that pass: a thread notes the
// largest value of each of up to 8 stretches of its pieces. Of the row's w warps (8,
// 4 or 1), each finds the ceil(k / w)-th largest of its threads' maxima; the least of
// these is reached by k values at least, so it bounds the k-th largest from below,
// and only stretches whose maximum reaches it (about 2 k of 2048, by 8 warps) can hold
// a value of the top k. Their pieces are read once more (from L2), one or two by each
// thread, and what reaches the bound goes into a list in shared memory. Values
// are ordered by (value, lower index), which makes every key different; pieces
// that overflow the list (rows with many equal values) raise the bound to the
// k-th best key of the list and are listed again.
//
// A row goes to a CTA, or to a single warp where it has at most 512 pieces of 16
// bytes and rows are many. Few long rows are split over a cluster of up to 8 CTAs, which join their
// partial results through distributed shared memory in the order of their ranks.
//
// Measured on a B200: 2048x131072 bf16 86 us (6.2 TB/s, 95 % of measured copy
// bandwidth), with 20 alternatives 108 us, its gradient 183 us (5.9 TB/s);
// 512x131072 fp32 41 us, with 8 alternatives 47 us; one row of 32768 fp32 3.1 us,
// with 5 alternatives 6.7 us; 2048x1000 bf16 3.8 us.
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "elem.cuh"

namespace kt {
namespace logprob {

constexpr int kBlock = 256;     // threads of a row; kSmall where rows are many and not the longest
constexpr int kSmall = 128;
constexpr int kBwdBlock = 128;
constexpr int kPieces = 4;     // 16-byte pieces of a thread per tile
constexpr int kStretches = 8;  // of a thread's pieces in a row
constexpr int kMaxTop = 32;
// Rows of at most so many pieces go to single warps where there are more than two
// per SM: 2048 rows of 4000 bf16 columns take 7 us by warps and 15 by CTAs (8
// alternatives: 13 and 31), 64 rows 4.3 and 3.4 (7.8 and 7.2).
constexpr int kWarpPieces = 512;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct FwdArgs {
  const void* x;
  int64_t ld;
  const int64_t* targets;  // may be null: no log probabilities
  int64_t rows;
  int64_t vocab;
  int64_t ignore;
  float scale;
  int top;
  float* logprob;
  float* entropy;
  float* lse;
  float2* norm;  // may be null
  float* top_logprob;
  int64_t* top_index;
};

struct BwdArgs {
  const void* x;
  int64_t ld;
  const int64_t* targets;
  const float2* norm;  // or, where null,
  const float* lse;
  const float* entropy;
  const float* g;  // may be null: 0
  const float* h;  // may be null: 0
  const float* l;  // may be null: 0
  int64_t rows;
  int64_t vocab;
  int64_t ignore;
  float scale;
  void* dx;
  int64_t ld_dx;
  int64_t chunks;  // CTAs per row
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

using elem::add2;
using elem::fma2;
using elem::halves;
using elem::mul2;
using elem::pair;

// Largest of a 16-byte piece; NaNs are passed over.
__device__ __forceinline__ float piece_max(const uint4& r, float) {
  return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
__device__ __forceinline__ float piece_max(const uint4& r, __nv_bfloat16) {
  const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&r);
  const float2 m = __bfloat1622float2(__hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
  return fmaxf(m.x, m.y);
}
__device__ __forceinline__ float piece_max(const uint4& r, __half) {
  const __half2* v = reinterpret_cast<const __half2*>(&r);
  const float2 m = __half22float2(__hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
  return fmaxf(m.x, m.y);
}

// Order-preserving key of a value and its index: greater values first, NaN
// above all, -0 equal to +0, lower indices first among equals.
__device__ __forceinline__ uint32_t order_bits(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  if (v != v) return 0xFFFFFFFFu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t make_key(float v, uint32_t index) {
  return ((uint64_t)order_bits(v) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

// Running statistics of a set of values: m = max x, s = sum 2^y, t = sum y 2^y
// with y = (x - m) c. Empty: m = -inf, s = t = 0.
struct Stats {
  float m, s, t;
};
// `a` as seen from the maximum `to` >= a.m.
__device__ __forceinline__ Stats moved(const Stats& a, float to, float c) {
  if (a.m == -INFINITY) return Stats{to, a.s, a.t};  // s = t = 0, or NaN
  // 2^-256 is 0; less would be -inf for a value like the type's lowest, and make t NaN
  const float d = fmaxf((a.m - to) * c, -256.f), f = ex2(d);
  return Stats{to, a.s * f, fmaf(a.s, d, a.t) * f};
}

// `raw` with the columns outside [0, vocab) as -inf.
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& raw, int e0, int vocab) {
  constexpr uint32_t none = std::is_same<T, float>::value ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00u
                                                                                                         : 0xFF80u;
  uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      if (e0 + k < 0 || e0 + k >= vocab) w[k] = none;
    } else {
      if (e0 + 2 * k < 0 || e0 + 2 * k >= vocab) w[k] = (w[k] & 0xFFFF0000u) | none;
      if (e0 + 2 * k + 1 < 0 || e0 + 2 * k + 1 >= vocab) w[k] = (w[k] & 0x0000FFFFu) | none << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Columns [e0, e0 + V) of the row, on a 16-byte boundary; those outside
// [0, vocab) are -inf. A piece that a row's end cuts also holds its neighbour's
// columns; only at the two ends [begin, end) of the logits may those not be there.
template <typename T>
__device__ __forceinline__ uint4 load_logits(const T* row, int e0, int vocab, const T* begin, const T* end) {
  constexpr int V = elem::kVec<T>;
  if (e0 >= 0 && e0 + V <= vocab) return elem::ld_once16(row + e0);
  const int e = elem::opaque(e0);
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (e < vocab) {
    if (row + e >= begin && row + e + V <= end) {
      raw = elem::ld_once16(row + e);
    } else {
      uint64_t lo = 0, hi = 0;
#pragma unroll 1
      for (int j = 0; j < V; ++j) {
        if (e + j < 0 || e + j >= vocab) continue;
        uint64_t bits;
        if constexpr (sizeof(T) == 4) bits = reinterpret_cast<const uint32_t*>(row)[e + j];
        else bits = reinterpret_cast<const uint16_t*>(row)[e + j];
        bits <<= (j % (V / 2)) * 8 * (int)sizeof(T);
        if (j < V / 2) lo |= bits;
        else hi |= bits;
      }
      raw = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    }
  }
  return masked<T>(raw, e, vocab);
}

// What the G threads of a row (or of a CTA's share of it) need to find its top k.
template <int G>
struct Top {
  static constexpr int kList = 512;
  uint64_t list[kList];
  uint64_t best[kMaxTop];  // sorted
  uint64_t threshold;      // keys up to this one are not listed
  uint32_t maxima[kStretches][G];
  uint32_t bounds[G / 32];
  uint16_t places[kStretches * G];
  int place_count, count, best_count;
};

template <int G>
__device__ __forceinline__ void sync() {
  if constexpr (G == 32) __syncwarp();
  else __syncthreads();
}
template <int G>
__device__ __forceinline__ bool any(bool v) {
  if constexpr (G == 32) {
    __syncwarp();  // a vote orders no memory
    return __any_sync(0xffffffffu, v);
  } else {
    return __syncthreads_or(v);
  }
}

// Sorted top k of the first n listed keys, by the threads t of G.
template <int G, int H>
__device__ __forceinline__ void best_of_list(Top<H>& top, int n, int k, int t) {
#pragma unroll 1
  for (int i = t; i < n; i += G) {
    const uint64_t key = top.list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += top.list[j] > key;
    if (key != 0 && rank < k) top.best[rank] = key;
  }
  if (t == 0) top.best_count = n < k ? n : k;
  sync<G>();
}

// One row's geometry for this CTA (or warp): pieces [first, last) of 16 bytes,
// thread t of G holding first + t, first + t + G, ...
template <typename T>
struct Row {
  const T* x;
  int shift, first, last;
  // a stretch: so many pieces of a thread, as whole tiles
  template <int G>
  __device__ __forceinline__ int stretch() const {
    const int tiles = (last - first + G * kPieces - 1) / (G * kPieces);
    return (tiles + kStretches - 1) / kStretches * kPieces;
  }
  __device__ __forceinline__ Row(const FwdArgs& p, int64_t row, int split, int part) {
    x = static_cast<const T*>(p.x) + row * p.ld;
    shift = elem::misalign<T>(x);
    const int pieces = ((int)p.vocab + shift + elem::kVec<T> - 1) / elem::kVec<T>;
    const int share = (pieces + split - 1) / split;
    first = part * share;
    last = first + share < pieces ? first + share : pieces;
  }
};
template <typename T>
__device__ __forceinline__ uint4 load_logits(const FwdArgs& p, const Row<T>& r, int pc) {
  const T* begin = static_cast<const T*>(p.x);
  const int vocab = (int)p.vocab;
  return load_logits<T>(r.x, pc < r.last ? pc * elem::kVec<T> - r.shift : vocab, vocab, begin,
                        begin + (p.rows - 1) * p.ld + vocab);
}

// The top k of the pieces of a row that G threads (number t) have streamed:
// top.maxima[stretch][t] holds their maximum_bits. Left in top.best.
template <typename T, int G>
__device__ __forceinline__ void find_top(Top<G>& top, const FwdArgs& p, const Row<T>& r, int t) {
  constexpr int V = elem::kVec<T>;
  constexpr int W = G / 32;
  constexpr int B = G == 32 ? 4 : 2;  // pieces of a thread at a time
  constexpr int kList = Top<G>::kList;
  const int lane = t & 31, k = p.top;
  const int stretch = r.template stretch<G>();
  const int per_thread = (r.last - r.first + G - 1) / G;  // pieces, at most
  const int stretches = (per_thread + stretch - 1) / stretch;
  // the ceil(k / W)-th largest of this warp's maxima; its low 12 bits are dropped,
  // which only lowers it (and drops bit 0 of maximum_bits)
  {
    uint32_t mine = 0, bound = 0;
    for (int s = 0; s < stretches; ++s) mine = max(mine, top.maxima[s][t] & 0xFFFFF000u);
    for (int left = (k + W - 1) / W; left > 0;) {
      bound = __reduce_max_sync(0xffffffffu, mine);
      left -= __popc(__ballot_sync(0xffffffffu, mine == bound));
      if (mine == bound) mine = 0;
    }
    if (lane == 0) top.bounds[t / 32] = bound;
    if (t == 0) top.place_count = top.count = 0;
  }
  sync<G>();
  uint32_t bound = top.bounds[0];
#pragma unroll
  for (int i = 1; i < W; ++i) bound = min(bound, top.bounds[i]);
  for (int s = 0; s < stretches; ++s) {
    const uint32_t v = top.maxima[s][t];
    if (v >= bound || (v & 1u)) top.places[atomicAdd(&top.place_count, 1)] = (uint16_t)(s * G + t);
  }
  if (t == 0) top.threshold = (uint64_t)bound << 32;
  sync<G>();

  const int total = top.place_count * stretch;
#pragma unroll 1
  for (int at0 = 0; at0 < total; at0 += G * B) {
    uint4 raw[B];
    int e0[B];  // first column; past the last where there is no piece
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int at = at0 + i * G + t;
      int pc = r.last;
      if (at < total) {
        const int which = at / stretch, place = top.places[which];
        pc = r.first + (place / G * stretch + at - which * stretch) * G + place % G;
      }
      e0[i] = pc < r.last ? pc * V - r.shift : (int)p.vocab;
      raw[i] = load_logits<T>(p, r, pc);
    }
#pragma unroll 1
    for (int i = 0; i < B; ++i) {
      const uint4 now = B == 2 ? (i == 0 ? raw[0] : raw[1])
                               : (i == 0 ? raw[0] : i == 1 ? raw[1] : i == 2 ? raw[B - 2] : raw[B - 1]);
      const int from = B == 2 ? (i == 0 ? e0[0] : e0[1])
                              : (i == 0 ? e0[0] : i == 1 ? e0[1] : i == 2 ? e0[B - 2] : e0[B - 1]);
      int before = top.count;  // at most kList, as the last step ended
      sync<G>();
      for (;;) {
        const uint64_t threshold = top.threshold;
        const float least = key_value(threshold | 0xFFFFFFFFu);
        bool over = false;
        float f[V];
        elem::unpack_vec<T>(now, f);
        uint32_t reach = 0;  // which of them reach the bound (a NaN does): few, so what follows is no unrolled code
#pragma unroll
        for (int j = 0; j < V; ++j) reach |= (f[j] < least ? 0u : 1u) << j;
#pragma unroll 1
        for (; reach; reach &= reach - 1) {
          const int j = __ffs(reach) - 1;
          float v = f[0];
#pragma unroll
          for (int i = 1; i < V; ++i) v = i == j ? f[i] : v;
          const uint64_t key = make_key(v, (uint32_t)(from + j));
          if (from + j >= 0 && from + j < (int)p.vocab && key > threshold) {
            const int to = atomicAdd(&top.count, 1);
            if (to < kList) top.list[to] = key;
            else over = true;
          }
        }
        if (!any<G>(over)) break;
        // too many: raise the threshold to the k-th best of the list (it and better
        // ones pass), keep what was listed before this step and still passes (at
        // most k keys), and list the step again; each time drops kList - 2 k keys
        for (int q = t; q < kList; q += G) {
          const uint64_t key = top.list[q];
          int rank = 0;
          for (int j = 0; j < kList; ++j) rank += top.list[j] > key;
          if (rank == k - 1) top.threshold = key - 1;
        }
        uint64_t old[kList / G];
#pragma unroll
        for (int q = 0; q < kList / G; ++q) old[q] = t + q * G < before ? top.list[t + q * G] : 0;
        sync<G>();
        if (t == 0) top.count = 0;
        sync<G>();
#pragma unroll
        for (int q = 0; q < kList / G; ++q)
          if (old[q] > top.threshold) top.list[atomicAdd(&top.count, 1)] = old[q];
        sync<G>();
        before = top.count;
        sync<G>();
      }
    }
  }
  sync<G>();
  best_of_list<G>(top, top.count, k, t);
}

// A row's target and its logit, loaded before the row is streamed.
struct Target {
  int64_t at;
  float x;
  bool is_column;
};
template <typename T>
__device__ __forceinline__ Target load_target(const FwdArgs& p, int64_t row) {
  Target t{p.ignore, 0.f, false};
  if (p.targets) t.at = p.targets[row];
  t.is_column = t.at != p.ignore && t.at >= 0 && t.at < p.vocab;
  if (t.is_column) t.x = elem::to_f(static_cast<const T*>(p.x)[row * p.ld + t.at]);
  return t;
}

// The outputs of a row, by one warp, from its statistics and sorted top k.
template <bool TOP>
__device__ __forceinline__ void write_row(const FwdArgs& p, int64_t row, const Stats& a, const Target& target,
                                          const uint64_t* best) {
  const int lane = threadIdx.x & 31, k = p.top;
  const float log2s = log2f(a.s);
  const bool none = a.m == -INFINITY && a.s == 0.f;
  auto log_p = [&](float x) { return none ? -INFINITY : fmaf(-log2s, kLn2, (x - a.m) * p.scale); };
  if (lane == 0) {
    p.lse[row] = none ? -INFINITY : fmaf(log2s, kLn2, a.m * p.scale);
    if (p.norm) p.norm[row] = make_float2(a.m, log2s);
    if (p.entropy) p.entropy[row] = none ? 0.f : (log2s - a.t / a.s) * kLn2;
    if (p.targets) {
      float v = target.is_column ? log_p(target.x) : 0.f;
      if (!target.is_column && target.at != p.ignore) {
        v = __uint_as_float(0x7FC00000u);
        raise_device_error(DEV_BAD_SHAPE);
      }
      p.logprob[row] = v;
    }
  }
  if (TOP && lane < k) {
    const uint64_t key = best[lane];
    p.top_logprob[row * k + lane] = log_p(key_value(key));
    p.top_index[row * k + lane] = (int64_t)key_index(key);
  }
}

// What find_top takes of a stretch: its largest value but for NaNs, a lower bound
// of its largest, and in bit 0 whether a NaN (or an infinity) is among its values.
__device__ __forceinline__ uint32_t maximum_bits(float largest, float s) {
  return (order_bits(largest) & ~1u) | (s != s ? 1u : 0u);
}

// Statistics of the values that one of G threads (number t) streams, and, with
// TOP, its stretches' maximum_bits in maxima[stretch][t].
template <typename T, int G, bool TOP>
__device__ __forceinline__ Stats stream(const FwdArgs& p, const Row<T>& r, int t, float c, uint32_t (*maxima)[G]) {
  constexpr int V = elem::kVec<T>;
  constexpr int kTile = G * kPieces;
  float largest = -INFINITY, recent = -INFINITY;  // of all, and of this stretch
  uint64_t s2 = 0, t2 = 0;                        // even and odd values' s and t
  const int stretch = TOP ? r.template stretch<G>() / kPieces : 0;
  int left = stretch, at = 0;
  uint4 next[kPieces];
  const int whole = ((int)p.vocab + r.shift) / V;  // pieces before this one end inside the row
  auto fetch = [&](int tile0) {
    if (tile0 * V >= r.shift && tile0 + kTile <= min(r.last, whole)) {  // no row's end in this tile
      const uint4* at = reinterpret_cast<const uint4*>(r.x - r.shift) + tile0 + t;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) next[i] = elem::ld_once16(at + i * G);
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) next[i] = load_logits<T>(p, r, tile0 + i * G + t);
    }
  };
  fetch(r.first);
  for (int tile0 = r.first; tile0 < r.last; tile0 += kTile) {
    uint4 cur[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) cur[i] = next[i];
    if (tile0 + kTile < r.last) fetch(tile0 + kTile);
    float top = piece_max(cur[0], T());
#pragma unroll
    for (int i = 1; i < kPieces; ++i) top = fmaxf(top, piece_max(cur[i], T()));
    if (top > largest) {
      const Stats even = moved(Stats{largest, halves(s2).x, halves(t2).x}, top, c);
      const Stats odd = moved(Stats{largest, halves(s2).y, halves(t2).y}, top, c);
      s2 = pair(even.s, odd.s);
      t2 = pair(even.t, odd.t);
      largest = top;
    }
    const float m = largest == -INFINITY ? 0.f : largest;
    const uint64_t minus = pair(-m, -m), by = pair(c, c);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      float f[V];
      elem::unpack_vec<T>(cur[i], f);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const float2 y = halves(mul2(add2(pair(f[j], f[j + 1]), minus), by));
        const uint64_t e = pair(ex2(y.x), ex2(y.y));
        s2 = add2(s2, e);
        t2 = fma2(pair(fmaxf(y.x, -256.f), fmaxf(y.y, -256.f)), e, t2);  // 2^-256 is 0: -inf adds 0, not NaN
      }
    }
    if constexpr (TOP) {
      recent = fmaxf(recent, top);
      if (--left == 0 || tile0 + kTile >= r.last) {
        maxima[at++][t] = maximum_bits(recent, halves(s2).x + halves(s2).y);
        left = stretch;
        recent = -INFINITY;
      }
    }
  }
  return Stats{largest, halves(s2).x + halves(s2).y, halves(t2).x + halves(t2).y};
}

// The statistics of the lanes' values together.
__device__ __forceinline__ Stats warp_stats(const Stats& a, float c) {
  Stats w = moved(a, warp_max(a.m), c);
  w.s = warp_sum(w.s);
  w.t = warp_sum(w.t);
  return w;
}

template <int G, bool TOP>
struct Shared {
  Top<TOP ? G : 32> top;
  Stats warp[G / 32];
  Stats all;
};

template <typename T, bool TOP, int G>
__global__ void __launch_bounds__(G, (TOP ? 5 : 4) * kBlock / G) fwd_kernel(const FwdArgs p) {
  namespace cg = cooperative_groups;
  __shared__ Shared<G, TOP> sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float c = p.scale * kLog2e;
  const int64_t row = blockIdx.x / split;
  const Row<T> r(p, row, split, part);
  Target target{};
  if (part == 0 && threadIdx.x == 0) target = load_target<T>(p, row);
  uint32_t(*maxima)[G] = nullptr;
  if constexpr (TOP) maxima = sh.top.maxima;
  Stats a = warp_stats(stream<T, G, TOP>(p, r, threadIdx.x, c, maxima), c);
  if (lane == 0) sh.warp[warp] = a;
  __syncthreads();
  if (warp == 0) {
    a = warp_stats(lane < G / 32 ? sh.warp[lane] : Stats{-INFINITY, 0.f, 0.f}, c);
    if (lane == 0) sh.all = a;
  }
  if constexpr (TOP) find_top<T, G>(sh.top, p, r, threadIdx.x);
  static_assert(!TOP || kBlock >= kMaxCluster * kMaxTop, "a thread per key of the joined lists");
  if (G == kBlock && split > 1) {  // the first CTA joins the others' results
    cluster.sync();
    if (part == 0) {
      if (warp == 0) {
        a = Stats{-INFINITY, 0.f, 0.f};
        if (lane < split) a = cluster.map_shared_rank(&sh, lane)->all;
        a = warp_stats(a, c);
      }
      if constexpr (TOP) {
        const int n = split * p.top, i = threadIdx.x;  // up to 8 x 32
        if (i < n) {
          const auto& o = cluster.map_shared_rank(&sh, i / p.top)->top;
          sh.top.list[i] = i % p.top < o.best_count ? o.best[i % p.top] : 0;  // 0 is below every key
        }
        __syncthreads();
        best_of_list<G>(sh.top, n, p.top, i);
      }
    }
  }
  if (part == 0 && warp == 0) write_row<TOP>(p, row, a, target, sh.top.best);
  if (G == kBlock && split > 1) cluster.sync();  // the other CTAs' shared memory is read above
}

// Short rows by single warps.
template <typename T, bool TOP>
__global__ void __launch_bounds__(TOP ? 128 : kBlock) fwd_warp_kernel(const FwdArgs p) {
  __shared__ Top<32> tops[TOP ? 4 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float c = p.scale * kLog2e;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / 32) + warp;
  if (row >= p.rows) return;
  const Row<T> r(p, row, 1, 0);
  Target target{};
  if (lane == 0) target = load_target<T>(p, row);
  Top<32>& top = tops[TOP ? warp : 0];
  const Stats a = warp_stats(stream<T, 32, TOP>(p, r, lane, c, top.maxima), c);
  if constexpr (TOP) {
    __syncwarp();
    find_top<T, 32>(top, p, r, lane);
  }
  write_row<TOP>(p, row, a, target, top.best);
}

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kBwdBlock) bwd_kernel(const BwdArgs p) {
  constexpr int V = VECTOR ? elem::kVec<T> : 1;
  const int64_t row = blockIdx.x / p.chunks;
  const int64_t at = blockIdx.x - row * p.chunks;
  const T* xr = static_cast<const T*>(p.x) + row * p.ld;
  T* dr = static_cast<T*>(p.dx) + row * p.ld_dx;
  const int shift = VECTOR ? elem::misalign<T>(xr) : 0;
  const int64_t target = p.targets ? p.targets[row] : p.ignore;
  // log2 of a probability is fma(fma(x, a, b), c, d); its natural logarithm, from
  // lse, is the inner one
  float a = 1.f, b, c = p.scale * kLog2e, d;
  bool none;  // the row has no distribution
  if (p.norm) {
    const float2 n = p.norm[row];
    b = -n.x;
    d = -n.y;
    none = n.x == -INFINITY && n.y == -INFINITY;  // (of NaNs and -inf the maximum is -inf too, the sum NaN)
  } else {
    a = p.scale;
    b = -p.lse[row];
    c = kLog2e;
    d = 0.f;
    none = b == INFINITY;
  }
  const bool scored = target != p.ignore && target >= 0 && target < p.vocab;
  float g = p.g && target != p.ignore ? p.g[row] * p.scale : 0.f;
  if (!scored && g != 0.f) g = __uint_as_float(0x7FC00000u);  // of a target that is no column: NaN, as its value
  const float h = p.h ? p.h[row] * p.scale : 0.f;
  const float l = p.l ? p.l[row] * p.scale : 0.f;
  // nothing comes from above, or the row has no distribution: the gradient is 0
  const bool zero = (g == 0.f && h == 0.f && l == 0.f) || none;
  const float each = p.h ? fmaf(h, p.entropy[row], g - l) : g - l, by = h * kLn2;
  auto grad = [&](float x, int64_t e) {
    const float y = fmaf(fmaf(x, a, b), c, d);
    const float v = -ex2(y) * fmaf(by, fmaxf(y, -1e4f), each);  // p = 0: 0, not NaN
    return e == target ? v + g : v;
  };
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int64_t e0 = ((at * kPieces + i) * kBwdBlock + threadIdx.x) * V - shift;
    if (e0 >= p.vocab) continue;
    if (V > 1 && e0 >= 0 && e0 + V <= p.vocab) {
      float f[elem::kVec<T>];
      if (zero) {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = 0.f;
      } else {
        elem::unpack_vec<T>(*reinterpret_cast<const uint4*>(xr + e0), f);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = grad(f[j], e0 + j);
      }
      *reinterpret_cast<uint4*>(dr + e0) = elem::pack_vec<T>(f);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int64_t e = e0 + j;
        if (e >= 0 && e < p.vocab) dr[e] = elem::from_f<T>(zero ? 0.f : grad(elem::to_f(xr[e]), e));
      }
    }
  }
}

// ---------------------------------------------------------------- host
inline int check_common(const char* what, int64_t rows, int64_t vocab, int64_t ld, float scale, int dtype) {
  if (rows < 0 || vocab < 0 || ld < 0)
    return fail(KT_ERR_ARG, "%s: negative shape rows=%lld vocab=%lld ld=%lld", what, (long long)rows,
                (long long)vocab, (long long)ld);
  if (elem::size_of(dtype) == 0) return fail(KT_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (!(scale > 0.f) || isinf(scale * kLog2e))  // (the kernels use scale log2 e)
    return fail(KT_ERR_ARG, "%s: scale must be positive and at most 2^127", what);
  if (rows > 0 && vocab == 0) return fail(KT_ERR_ARG, "%s: rows without columns", what);
  if (vocab > (int64_t)1 << 30) return fail(KT_ERR_UNSUPPORTED, "%s: vocab > 2^30", what);
  return KT_OK;
}

template <typename T, bool TOP>
inline int fwd_typed(const FwdArgs& a, cudaStream_t st) {
  constexpr int64_t kTile = (int64_t)kBlock * kPieces * elem::kVec<T>;
  if (a.vocab <= (int64_t)kWarpPieces * elem::kVec<T> && a.rows > 2 * sm_count()) {
    const int block = TOP ? 128 : kBlock;
    const int64_t grid = (a.rows + block / 32 - 1) / (block / 32);
    if (grid > INT32_MAX) return fail(KT_ERR_UNSUPPORTED, "token_logprobs: too many rows");
    fwd_warp_kernel<T, TOP><<<(unsigned)grid, block, 0, st>>>(a);
    return check_launch("token_logprobs warps");
  }
  // CTAs of 128 threads where more rows than four per SM have at most 8192 pieces:
  // more of them end and begin at a time, and the last wave is shorter. 2048 rows of
  // 50001 bf16 columns take 42 us by 128 threads each and 48 by 256 (8 alternatives:
  // 55 and 63); of 131072 columns 89 and 88 (20: 114 and 106).
  if (a.rows > 4 * sm_count() && a.vocab <= (int64_t)8192 * elem::kVec<T>) {
    if (a.rows > INT32_MAX) return fail(KT_ERR_UNSUPPORTED, "token_logprobs: too many rows");
    fwd_kernel<T, TOP, kSmall><<<(unsigned)a.rows, kSmall, 0, st>>>(a);
    return check_launch("token_logprobs small CTAs");
  }
  // a cluster per row while all CTAs fit on the device at once and each has a tile:
  // one row of 131072 bf16 columns takes 4 us by 8 CTAs and 10 by one
  int split = 1;
  while (split < kMaxCluster && a.rows * split * 2 <= 2 * sm_count() && a.vocab > kTile * split) split *= 2;
  if (a.rows * split > INT32_MAX) return fail(KT_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * split));
  cfg.blockDim = dim3(kBlock);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, fwd_kernel<T, TOP, kBlock>, a), "token_logprobs launch");
}

inline int forward(const FwdArgs& a, int dtype, cudaStream_t st) {
  const int rc = check_common("token_logprobs", a.rows, a.vocab, a.ld, a.scale, dtype);
  if (rc != KT_OK) return rc;
  if (a.top < 0 || a.top > kMaxTop) return fail(KT_ERR_ARG, "token_logprobs: top_k must be in [0, %d]", kMaxTop);
  if (a.top > a.vocab && a.rows > 0) return fail(KT_ERR_ARG, "token_logprobs: top_k > vocab");
  if (a.rows == 0) return KT_OK;
  if (!a.x || !a.lse || (a.targets && !a.logprob) || (a.top > 0 && (!a.top_logprob || !a.top_index)))
    return fail(KT_ERR_ARG, "token_logprobs: null pointer");
  if (!elem::aligned_to(a.x, elem::size_of(dtype)) || !elem::aligned_to(a.targets, 8) ||
      !elem::aligned_to(a.top_index, 8) || !elem::aligned_to(a.norm, 8))
    return fail(KT_ERR_ARG, "token_logprobs: a pointer is not aligned to its elements");
  const bool top = a.top > 0;
  if (dtype == KT_F32) return top ? fwd_typed<float, true>(a, st) : fwd_typed<float, false>(a, st);
  if (dtype == KT_BF16) return top ? fwd_typed<__nv_bfloat16, true>(a, st) : fwd_typed<__nv_bfloat16, false>(a, st);
  return top ? fwd_typed<__half, true>(a, st) : fwd_typed<__half, false>(a, st);
}

template <typename T>
inline int bwd_typed(BwdArgs a, cudaStream_t st) {
  constexpr int V = elem::kVec<T>;
  // pieces are aligned in both tensors, for every row
  const bool vec = elem::misalign<T>(a.x) == elem::misalign<T>(a.dx) && (a.rows == 1 || (a.ld - a.ld_dx) % V == 0);
  const int64_t per = (int64_t)kBwdBlock * kPieces * (vec ? V : 1);
  a.chunks = (a.vocab + (vec ? V - 1 : 0) + per - 1) / per;
  if (a.rows * a.chunks > (int64_t)INT32_MAX) return fail(KT_ERR_UNSUPPORTED, "token_logprobs_bwd: too many values");
  const unsigned grid = (unsigned)(a.rows * a.chunks);
  if (vec) bwd_kernel<T, true><<<grid, kBwdBlock, 0, st>>>(a);
  else bwd_kernel<T, false><<<grid, kBwdBlock, 0, st>>>(a);
  return check_launch("token_logprobs_bwd");
}

inline int backward(const BwdArgs& a, int dtype, cudaStream_t st) {
  const int rc = check_common("token_logprobs_bwd", a.rows, a.vocab, a.ld, a.scale, dtype);
  if (rc != KT_OK) return rc;
  if (a.rows == 0) return KT_OK;
  if (a.ld_dx < a.vocab) return fail(KT_ERR_ARG, "token_logprobs_bwd: rows of the gradient overlap");
  if (!a.x || (!a.norm && !a.lse) || !a.dx || (a.g && !a.targets) || (a.h && !a.entropy))
    return fail(KT_ERR_ARG, "token_logprobs_bwd: null pointer");
  const int sz = elem::size_of(dtype);
  if (!elem::aligned_to(a.x, sz) || !elem::aligned_to(a.dx, sz) || !elem::aligned_to(a.targets, 8) ||
      !elem::aligned_to(a.norm, 8))
    return fail(KT_ERR_ARG, "token_logprobs_bwd: a pointer is not aligned to its elements");
  if (dtype == KT_F32) return bwd_typed<float>(a, st);
  if (dtype == KT_BF16) return bwd_typed<__nv_bfloat16>(a, st);
  return bwd_typed<__half>(a, st);
}

}  // namespace logprob
}  // namespace kt
