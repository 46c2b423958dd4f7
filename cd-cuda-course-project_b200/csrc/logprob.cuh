// logprob.cuh — log probabilities of given tokens, the entropy and the most
// likely tokens of each row of logits, and the gradient of the logits.
//
// With z = scale x over the V columns of a row (fp32 throughout):
//   lse = log sum e^z      logprob = z[target] - lse      H = lse - sum p z
//   gradient, for upstream g (logprob) and h (entropy):
//   dx_j = scale (g ([j = target] - p_j) - h p_j (log p_j + H)),  p_j = e^(z_j - lse)
// A row of only -inf has no distribution: lse and every log probability are
// -inf, its entropy and its gradient 0. A NaN or +inf makes the row NaN.
//
// Forward reads the logits once: every thread keeps a running maximum m of x,
// s = sum 2^y and t = sum y 2^y with y = (x - m) scale log2 e, and rescales them
// when its maximum grows, so H = ln 2 (log2 s - t / s) needs no second pass.
// (One fused multiply-add per y would be off by the rounding of m scale log2 e:
// a certain token would not get log probability 0.) Bound by memory for 32-bit logits; for 16-bit ones the one
// exponential per value takes about 3/4 of the special-function rate that goes
// with the full read rate.
//
// The top k of a row need no work in that pass: each thread's maximum is one of
// its values, so the k-th largest of the 256 maxima is a lower bound of the k-th
// largest value, and only threads whose maximum reaches it (about k of 256) can
// hold a value of the top k. Their pieces are read once more (from L2), by all
// threads, and what reaches the bound goes into a list in shared memory. Values
// are ordered by (value, lower index), which makes every key different; pieces
// that overflow the list (rows with many equal values) raise the bound to the
// k-th best key of the list and are listed again.
//
// Few rows are split over a cluster of up to 8 CTAs, which join their partial
// results through distributed shared memory in the order of their ranks.
#pragma once
#include <cooperative_groups.h>

#include "elem.cuh"

namespace kt {
namespace logprob {

constexpr int kBlock = 256;
constexpr int kPieces = 4;     // 16-byte pieces of a thread per tile
constexpr int kMaxTop = 32;
constexpr int kList = 1024;    // entries of the list of candidates
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
  float* top_logprob;
  int64_t* top_index;
};

struct BwdArgs {
  const void* x;
  int64_t ld;
  const int64_t* targets;
  const float* lse;
  const float* entropy;
  const float* g;  // may be null: 0
  const float* h;  // may be null: 0
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

// Two fp32 operations by one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

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

template <typename T>
__device__ __forceinline__ uint4 load_logits(const T* row, int64_t e0, int64_t lo, int64_t hi) {
  // columns [e0, e0 + V) of the row; those outside [lo, hi) are -inf
  constexpr int V = elem::kVec<T>;
  if (e0 >= lo && e0 + V <= hi) return elem::ld_once16(row + e0);
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = (e0 + j >= lo && e0 + j < hi) ? elem::to_f(row[e0 + j]) : -INFINITY;
  return elem::pack_vec<T>(f);
}

struct Shared {
  uint64_t list[kList];
  uint64_t best[kMaxTop];  // this CTA's top k, sorted
  uint64_t threshold;      // keys up to this one are not listed
  uint32_t maxima[kBlock]; // order_bits of the threads' maxima
  int threads[kBlock];     // those that may hold a value of the top k
  int thread_count;
  int count;               // listed so far (may exceed kList)
  int best_count;
  Stats warp[kBlock / 32];
  Stats all;
};

// The k-th best key of the first n of the list is left in sh.threshold.
__device__ __forceinline__ void raise_to_kth(Shared& sh, int n, int k) {
  for (int i = threadIdx.x; i < n; i += kBlock) {
    const uint64_t key = sh.list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.list[j] > key;
    if (rank == k - 1) sh.threshold = key - 1;  // the k-th itself still passes
  }
}

// Lists the values of this CTA's pieces [first, last) that may be in its top k:
// leaves sh.count of them in sh.list.
template <typename T>
__device__ __forceinline__ void list_candidates(Shared& sh, const T* xr, int64_t first, int64_t last, int shift,
                                                int64_t vocab, int k) {
  constexpr int V = elem::kVec<T>;
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid < 32) {
    // the largest b, of the top 20 bits, that k maxima reach, by its bits from above
    uint32_t m[kBlock / 32], bound = 0;
#pragma unroll
    for (int i = 0; i < kBlock / 32; ++i) m[i] = sh.maxima[lane + 32 * i];
    for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < kBlock / 32; ++i) n += m[i] >= (bound | bit);
      if (__reduce_add_sync(0xffffffffu, n) >= k) bound |= bit;
    }
    if (lane == 0) {
      sh.threshold = (uint64_t)bound << 32;
      sh.thread_count = 0;
      sh.count = 0;
    }
  }
  __syncthreads();
  if (sh.maxima[tid] >= (uint32_t)(sh.threshold >> 32)) sh.threads[atomicAdd(&sh.thread_count, 1)] = tid;
  __syncthreads();
  const int each = (int)((last - first + kBlock - 1) / kBlock);  // pieces of a thread, at most
  const int64_t total = (int64_t)sh.thread_count * each;
  for (int64_t at0 = 0; at0 < total; at0 += kBlock) {
    const int64_t at = at0 + tid;
    int64_t pc = last;
    if (at < total) {
      const int turn = (int)(at / each);
      pc = first + (at - (int64_t)turn * each) * kBlock + sh.threads[turn];
    }
    const int64_t e0 = pc * V - shift;
    float f[V];
    elem::unpack_vec<T>(load_logits<T>(xr, e0, 0, pc < last ? vocab : 0), f);
    int before = sh.count;  // at most kList, as the last turn ended
    __syncthreads();
    for (;;) {
      const uint64_t threshold = sh.threshold;
      const uint32_t least = (uint32_t)(threshold >> 32);
      bool over = false;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (pc < last && order_bits(f[j]) >= least && e0 + j >= 0 && e0 + j < vocab) {
          const uint64_t key = make_key(f[j], (uint32_t)(e0 + j));
          if (key > threshold) {
            const int to = atomicAdd(&sh.count, 1);
            if (to < kList) sh.list[to] = key;
            else over = true;
          }
        }
      }
      if (!__syncthreads_or(over)) break;
      raise_to_kth(sh, kList, k);
      // keep what earlier turns listed and still passes (at most k keys)
      uint64_t old[kList / kBlock];
#pragma unroll
      for (int i = 0; i < kList / kBlock; ++i) old[i] = tid + i * kBlock < before ? sh.list[tid + i * kBlock] : 0;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kList / kBlock; ++i)
        if (old[i] > sh.threshold) sh.list[atomicAdd(&sh.count, 1)] = old[i];
      __syncthreads();
      before = sh.count;
      __syncthreads();
    }
  }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kBlock, 4) fwd_kernel(const FwdArgs p) {
  namespace cg = cooperative_groups;
  constexpr int V = elem::kVec<T>;
  constexpr int64_t kTile = (int64_t)kBlock * kPieces;
  __shared__ Shared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / split;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* xr = static_cast<const T*>(p.x) + row * p.ld;
  const int shift = elem::misalign<T>(xr);
  const int64_t pieces = (p.vocab + shift + V - 1) / V;
  const int64_t share = (pieces + split - 1) / split;
  const int64_t first = part * share, last = first + share < pieces ? first + share : pieces;
  const float c = p.scale * kLog2e;
  const int k = p.top;

  Stats st{-INFINITY, 0.f, 0.f};
  uint64_t s2 = 0, t2 = 0;  // even and odd values' s and t
  uint4 next[kPieces];
  auto fetch = [&](int64_t tile0) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int64_t pc = tile0 + (int64_t)i * kBlock + tid;
      next[i] = load_logits<T>(xr, pc * V - shift, 0, pc < last ? p.vocab : 0);
    }
  };
  fetch(first);
  for (int64_t tile0 = first; tile0 < last; tile0 += kTile) {
    uint4 cur[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) cur[i] = next[i];
    if (tile0 + kTile < last) fetch(tile0 + kTile);
    float top = piece_max(cur[0], T());
#pragma unroll
    for (int i = 1; i < kPieces; ++i) top = fmaxf(top, piece_max(cur[i], T()));
    if (top > st.m) {
      const Stats even = moved(Stats{st.m, halves(s2).x, halves(t2).x}, top, c);
      const Stats odd = moved(Stats{st.m, halves(s2).y, halves(t2).y}, top, c);
      s2 = pair(even.s, odd.s);
      t2 = pair(even.t, odd.t);
      st.m = top;
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
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
  }
  st.s = halves(s2).x + halves(s2).y;
  st.t = halves(t2).x + halves(t2).y;
  if constexpr (TOP) sh.maxima[tid] = st.s != st.s ? 0xFFFFFFFFu : order_bits(st.m);  // a NaN may be among them

  // the CTA's statistics
  {
    const float m = warp_max(st.m);
    st = moved(st, m, c);
    st.s = warp_sum(st.s);
    st.t = warp_sum(st.t);
    if (lane == 0) sh.warp[warp] = st;
    __syncthreads();
    if (warp == 0) {
      Stats w = lane < kBlock / 32 ? sh.warp[lane] : Stats{-INFINITY, 0.f, 0.f};
      w = moved(w, warp_max(w.m), c);
      w.s = warp_sum(w.s);
      w.t = warp_sum(w.t);
      if (lane == 0) sh.all = w;
    }
  }
  if constexpr (TOP) {
    list_candidates<T>(sh, xr, first, last, shift, p.vocab, k);
    const int n = sh.count;  // at most kList: every turn ended without an overflow
    if (tid == 0) sh.best_count = n < k ? n : k;
    for (int i = tid; i < n; i += kBlock) {
      const uint64_t key = sh.list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sh.list[j] > key;
      if (rank < k) sh.best[rank] = key;
    }
  }
  __syncthreads();

  // the row's, joined by the first CTA of the cluster
  if (split > 1) {
    cluster.sync();
    if (part == 0) {
      Stats w{-INFINITY, 0.f, 0.f};
      if (warp == 0) {
        if (lane < split) w = cluster.map_shared_rank(&sh, lane)->all;
        w = moved(w, warp_max(w.m), c);
        w.s = warp_sum(w.s);
        w.t = warp_sum(w.t);
        __syncwarp();
        if (lane == 0) sh.all = w;
      }
      if constexpr (TOP) {
        const int from = tid / kMaxTop, at = tid % kMaxTop;  // 8 lists of up to 32
        uint64_t key = 0;
        if (from < split) {
          const Shared* o = cluster.map_shared_rank(&sh, from);
          if (at < o->best_count) key = o->best[at];
        }
        sh.list[tid] = key;  // 0 is below every key
        __syncthreads();
        int rank = 0;
        for (int j = 0; j < kBlock; ++j) rank += sh.list[j] > key;
        if (key != 0 && rank < k) sh.best[rank] = key;
      }
      __syncthreads();
    }
  }
  if (part == 0) {
    const Stats a = sh.all;
    const float log2s = log2f(a.s);
    const bool none = a.m == -INFINITY && a.s == 0.f;
    const float lse = none ? -INFINITY : fmaf(log2s, kLn2, a.m * p.scale);
    auto log_p = [&](float x) { return none ? -INFINITY : fmaf(-log2s, kLn2, (x - a.m) * p.scale); };
    if (tid == 0) {
      p.lse[row] = lse;
      if (p.entropy) p.entropy[row] = none ? 0.f : (log2s - a.t / a.s) * kLn2;
      if (p.targets) {
        const int64_t target = p.targets[row];
        float v = 0.f;
        if (target != p.ignore) {
          if (target >= 0 && target < p.vocab) {
            v = log_p(elem::to_f(xr[target]));
          } else {
            v = __uint_as_float(0x7FC00000u);
            raise_device_error(DEV_BAD_SHAPE);
          }
        }
        p.logprob[row] = v;
      }
    }
    if (TOP && tid >= 32 && tid < 32 + k) {
      const uint64_t key = sh.best[tid - 32];
      p.top_logprob[row * k + tid - 32] = log_p(key_value(key));
      p.top_index[row * k + tid - 32] = (int64_t)key_index(key);
    }
  }
  if (split > 1) cluster.sync();  // the other CTAs' shared memory is read above
}

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kBlock) bwd_kernel(const BwdArgs p) {
  constexpr int V = VECTOR ? elem::kVec<T> : 1;
  const int64_t row = blockIdx.x / p.chunks;
  const int64_t at = blockIdx.x - row * p.chunks;
  const T* xr = static_cast<const T*>(p.x) + row * p.ld;
  T* dr = static_cast<T*>(p.dx) + row * p.ld_dx;
  const int shift = VECTOR ? elem::misalign<T>(xr) : 0;
  const int64_t target = p.targets ? p.targets[row] : p.ignore;
  const float lse = p.lse[row];
  const bool scored = target != p.ignore && target >= 0 && target < p.vocab;
  const float g = scored && p.g ? p.g[row] * p.scale : 0.f;
  const float h = p.h ? p.h[row] * p.scale : 0.f;
  const float entropy = p.h ? p.entropy[row] : 0.f;
  // nothing comes from above, or the row has no distribution: the gradient is 0
  const bool zero = (g == 0.f && h == 0.f) || lse == -INFINITY;
  auto grad = [&](float x, int64_t e) {
    const float logp = fmaf(x, p.scale, -lse);
    const float prob = ex2(logp * kLog2e);
    const float d = -prob * fmaf(h, fmaxf(logp, -1e4f) + entropy, g);  // p = 0: 0, not NaN
    return e == target ? d + g : d;
  };
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int64_t e0 = ((at * kPieces + i) * kBlock + threadIdx.x) * V - shift;
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
  if (!(scale > 0.f) || isinf(scale)) return fail(KT_ERR_ARG, "%s: scale must be positive and finite", what);
  if (rows > 0 && vocab == 0) return fail(KT_ERR_ARG, "%s: rows without columns", what);
  if (vocab > (int64_t)INT32_MAX - 64) return fail(KT_ERR_UNSUPPORTED, "%s: vocab > 2^31 - 65", what);
  return KT_OK;
}

template <typename T, bool TOP>
inline int fwd_typed(const FwdArgs& a, cudaStream_t st) {
  constexpr int64_t kTile = (int64_t)kBlock * kPieces * elem::kVec<T>;
  // a cluster per row while the CTAs fit on the device once, and each has a tile
  int split = 1;
  while (split < kMaxCluster && a.rows * split * 2 <= 2 * sm_count() && a.vocab > kTile * split) split *= 2;
  if (a.rows * split > (int64_t)INT32_MAX) return fail(KT_ERR_UNSUPPORTED, "token_logprobs: too many rows");
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
  return cuda_status(cudaLaunchKernelEx(&cfg, fwd_kernel<T, TOP>, a), "token_logprobs launch");
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
      !elem::aligned_to(a.top_index, 8))
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
  const int64_t per = (int64_t)kBlock * kPieces * (vec ? V : 1);
  a.chunks = (a.vocab + (vec ? V - 1 : 0) + per - 1) / per;
  if (a.rows * a.chunks > (int64_t)INT32_MAX) return fail(KT_ERR_UNSUPPORTED, "token_logprobs_bwd: too many values");
  const unsigned grid = (unsigned)(a.rows * a.chunks);
  if (vec) bwd_kernel<T, true><<<grid, kBlock, 0, st>>>(a);
  else bwd_kernel<T, false><<<grid, kBlock, 0, st>>>(a);
  return check_launch("token_logprobs_bwd");
}

inline int backward(const BwdArgs& a, int dtype, cudaStream_t st) {
  const int rc = check_common("token_logprobs_bwd", a.rows, a.vocab, a.ld, a.scale, dtype);
  if (rc != KT_OK) return rc;
  if (a.rows == 0) return KT_OK;
  if (a.ld_dx < a.vocab) return fail(KT_ERR_ARG, "token_logprobs_bwd: rows of the gradient overlap");
  if (!a.x || !a.lse || !a.dx || (a.g && !a.targets) || (a.h && !a.entropy))
    return fail(KT_ERR_ARG, "token_logprobs_bwd: null pointer");
  const int sz = elem::size_of(dtype);
  if (!elem::aligned_to(a.x, sz) || !elem::aligned_to(a.dx, sz) || !elem::aligned_to(a.targets, 8))
    return fail(KT_ERR_ARG, "token_logprobs_bwd: a pointer is not aligned to its elements");
  if (dtype == KT_F32) return bwd_typed<float>(a, st);
  if (dtype == KT_BF16) return bwd_typed<__nv_bfloat16>(a, st);
  return bwd_typed<__half>(a, st);
}

}  // namespace logprob
}  // namespace kt
