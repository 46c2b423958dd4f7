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
// The top k of a row go through a list in shared memory that holds every value
// above a threshold: the k-th largest of 64 group maxima of what was read so
// far, a lower bound of the k-th largest value. It is raised after 1, 2, 4, ...
// tiles, so about k log2(tiles) values are listed. Values are ordered by
// (value, lower index), which makes every key different; a tile that overflows
// the list raises the threshold to the k-th best key of the list and is listed
// again.
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
constexpr int kGroups = 64;    // groups of threads whose maxima bound the k-th value
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
  int count;               // listed so far (may exceed kList)
  int best_count;
  float groups[kGroups];
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

template <typename T, bool TOP>
__global__ void __launch_bounds__(kBlock) fwd_kernel(const FwdArgs p) {
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
  const int64_t lo = 0, hi = p.vocab;
  const float c = p.scale * kLog2e;
  const int k = p.top;

  if (TOP && tid == 0) {
    sh.count = 0;
    sh.threshold = 0;
  }
  Stats st{-INFINITY, 0.f, 0.f};
  float seen = -INFINITY;  // largest value of this thread so far
  uint4 next[kPieces];
  auto fetch = [&](int64_t tile0) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int64_t pc = tile0 + (int64_t)i * kBlock + tid;
      next[i] = load_logits<T>(xr, pc * V - shift, lo, pc < last ? hi : 0);
    }
  };
  fetch(first);
  int64_t next_raise = 1, tile = 0;
  if (TOP) __syncthreads();
  for (int64_t tile0 = first; tile0 < last; tile0 += kTile) {
    uint4 cur[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) cur[i] = next[i];
    if (tile0 + kTile < last) fetch(tile0 + kTile);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      float f[V];
      elem::unpack_vec<T>(cur[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmaxf(top, f[j]);
    }
    seen = fmaxf(seen, top);
    if (top > st.m) st = moved(st, top, c);
    const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      float f[V];
      elem::unpack_vec<T>(cur[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float y = (f[j] - m) * c, e = ex2(y);
        st.s += e;
        st.t = fmaf(fmaxf(y, -256.f), e, st.t);  // 2^-256 is 0: -inf adds 0, not NaN
      }
    }
    if constexpr (TOP) {
      ++tile;
      if (tile == next_raise) {
        next_raise *= 2;
        float v = fmaxf(seen, __shfl_xor_sync(0xffffffffu, seen, 1));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        if ((lane & 3) == 0) sh.groups[tid >> 2] = v;
        __syncthreads();
        if (warp == 0) {
          const float a = sh.groups[lane], b = sh.groups[lane + 32];
          int ga = 0, gb = 0, ea = 0, eb = 0;  // groups above, and groups equal
          for (int j = 0; j < kGroups; ++j) {
            const float o = sh.groups[j];
            ga += o > a;
            gb += o > b;
            ea += o == a;
            eb += o == b;
          }
          float kth = -INFINITY;
          if (ga < k && k <= ga + ea) kth = a;
          if (gb < k && k <= gb + eb) kth = b;
          kth = warp_max(kth);
          const uint64_t bound = (uint64_t)order_bits(kth) << 32;
          if (lane == 0 && bound > sh.threshold) sh.threshold = bound;
        }
        __syncthreads();
      }
      int before = sh.count;  // at most kList, as the last tile ended
      __syncthreads();
      for (;;) {
        const uint64_t threshold = sh.threshold;
        const float least = key_value(threshold | 0xFFFFFFFFull);
        bool over = false;
        if (!(top < least) || st.s != st.s || threshold == 0) {
#pragma unroll 1
          for (int i = 0; i < kPieces; ++i) {
            float f[V];
            elem::unpack_vec<T>(i == 0 ? cur[0] : i == 1 ? cur[1] : i == 2 ? cur[2] : cur[3], f);
            const int64_t pc = tile0 + (int64_t)i * kBlock + tid;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const int64_t e = pc * V - shift + j;
              if (pc < last && e >= lo && e < hi && !(f[j] < least)) {
                const uint64_t key = make_key(f[j], (uint32_t)e);
                if (key > threshold) {
                  const int at = atomicAdd(&sh.count, 1);
                  if (at < kList) sh.list[at] = key;
                  else over = true;
                }
              }
            }
          }
        }
        if (!__syncthreads_or(over)) break;
        raise_to_kth(sh, kList, k);
        // keep what earlier tiles listed and still passes (at most k keys)
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
    const int n = sh.count;  // at most kList: every tile ended without an overflow
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
