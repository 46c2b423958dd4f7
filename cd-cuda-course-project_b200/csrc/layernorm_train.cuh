// layernorm_train.cuh — LayerNorm with its backward pass (fp32, bf16, fp16),
// optionally keeping the input for the backward pass in 8 bits.
//
// Forward, per row of C columns:
//   mu = mean(x)   r = 1/sqrt(mean((x-mu)^2) + eps)   y = gamma (x-mu) r + beta
// and mu, r (fp32) are saved. Backward, with xh = (x-mu) r and w = dy gamma:
//   dx = r (w - mean(w) - xh mean(w xh))
//   dgamma = sum over rows of dy xh      dbeta = sum over rows of dy
// All sums and statistics are fp32; y, dx, dgamma, dbeta are rounded once.
//
// 8-bit checkpoint (forward writes it, backward reads it in x's place): blocks
// of 32 columns share a power of two, E = exponent field of the block's largest
// magnitude as fp32, at least 7; q = x 2^(133-E) rounded to nearest even and
// limited to +-127, standing for q 2^(E-133). With a power of two both steps
// are exact but for the one rounding, so the numbers do not depend on who
// computes them. A block that holds an infinity or a NaN has E = 255 and stands
// for NaN. mu and r come from the unrounded x.
//
// Bound by memory: forward reads x and writes y, backward reads dy and x (or 8
// bits of it) and writes dx. TPR threads take one row as 16-byte pieces. Each
// thread copies its own pieces of the next rows into shared memory with cp.async
// (no thread waits for another's), so the reads in flight, which at one row
// ahead in registers held 16-bit rows to 2/3 of the bandwidth, cost no registers.
// The rows of a CTA are grid.x apart, which makes them equally aligned, so a
// thread always holds the same columns: gamma and beta stay in its registers, and
// dgamma and dbeta are summed there over all rows of the CTA and written once, as
// one partial row per CTA. A second kernel adds the partial rows in their order,
// so results do not change from run to run.
//
// Measured on a B200, 16384x4096, the join included: bf16 forward 46 us (5.8 TB/s,
// 89 % of measured copy bandwidth) and backward 73 us (5.5 TB/s); with checkpoints
// 62 us (5.4 TB/s) and 77 us (4.4 TB/s, issue slots 62 % busy); fp32 98 and 140 us
// (5.5 and 5.7 TB/s). 8x512 fp32: 2.3 and 3.9 us. 4096x16384 bf16: 55 and 80 us
// (79 and 136 us with gamma and beta read again from L2 in every row).
// Odd widths: 16384x2049 bf16 55 and 77 us, with checkpoints 86 and 110 us.
#pragma once
#include <type_traits>

#include "elem.cuh"

namespace kt {
namespace ln_train {

struct FwdArgs {
  const void* x;
  const void* gamma;  // may be null: 1
  const void* beta;   // may be null: 0
  void* y;
  float* mean;
  float* rstd;
  int8_t* q8;        // with 8-bit checkpoints
  uint8_t* q8_exp;   // rows x ceil(cols / 32)
  int64_t ld_q8;
  int64_t rows;
  int64_t cols;
  float eps;
  int wdtype;
};

struct BwdArgs {
  const void* dy;
  const void* x;  // null with 8-bit checkpoints
  const int8_t* q8;
  const uint8_t* q8_exp;
  int64_t ld_q8;
  const void* gamma;
  const float* mean;
  const float* rstd;
  void* dx;
  float* partial;  // [parts][2][cols]: dgamma, dbeta
  int64_t rows;
  int64_t cols;
  int wdtype;
};

// ---------------------------------------------------------------- 8-bit blocks
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Exponent code of a block from the largest bit pattern of its magnitudes
// (infinities and NaNs have the largest patterns).
__device__ __forceinline__ uint32_t block_code(uint32_t bits) {
  const uint32_t e = bits >> 23;
  return e < 7u ? 7u : e;
}
__device__ __forceinline__ float code_up(uint32_t code) {
  return code == 255u ? 0.f : __uint_as_float((260u - code) << 23);
}
__device__ __forceinline__ float code_down(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float((code - 6u) << 23);
}
__device__ __forceinline__ int quant8(float v, float up) {
  // a non-finite value meets up = 0 only; its NaN becomes 0
  return min(127, max(-127, __float2int_rn(v * up)));
}

// Four of them to a word, from two pairs. A block's values times `up` are below
// 128, so their sums with 1.5 2^23 have the integers, rounded to nearest even, in
// their low 16 bits, where +-128 becomes +-127.
__device__ __forceinline__ uint32_t quant8x4(uint64_t ab, uint64_t cd, float up, uint32_t code) {
  const uint64_t by = elem::pair(up, up), magic = elem::pair(12582912.f, 12582912.f);
  const float2 s = elem::halves(elem::fma2(ab, by, magic)), t = elem::halves(elem::fma2(cd, by, magic));
  uint32_t p = __byte_perm(__float_as_uint(s.x), __float_as_uint(s.y), 0x5410);
  uint32_t q = __byte_perm(__float_as_uint(t.x), __float_as_uint(t.y), 0x5410);
  p = __vmaxs2(__vmins2(p, 0x007F007Fu), 0xFF81FF81u);
  q = __vmaxs2(__vmins2(q, 0x007F007Fu), 0xFF81FF81u);
  const uint32_t w = __byte_perm(p, q, 0x6420);
  return code == 255u ? 0u : w;
}

// The largest magnitude of a 16-byte piece as a bit pattern of T, and as one of fp32.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const uint4& r) {
  if constexpr (sizeof(T) == 4) {
    constexpr uint32_t m = 0x7FFFFFFFu;
    return max(max(r.x & m, r.y & m), max(r.z & m, r.w & m));
  } else {
    constexpr uint32_t m = 0x7FFF7FFFu;
    const uint32_t t = __vmaxu2(__vmaxu2(r.x & m, r.y & m), __vmaxu2(r.z & m, r.w & m));
    return max(t & 0xFFFFu, t >> 16);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t as_fp32(uint32_t bits) {
  if constexpr (std::is_same<T, float>::value) return bits;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return bits << 16;
  else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)bits)));
}

// ---------------------------------------------------------------- row pieces
// `raw` with the columns outside [0, cols) as 0.
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& raw, int e0, int cols) {
  uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      if (e0 + k < 0 || e0 + k >= cols) w[k] = 0;
    } else {
      if (e0 + 2 * k < 0 || e0 + 2 * k >= cols) w[k] &= 0xFFFF0000u;
      if (e0 + 2 * k + 1 < 0 || e0 + 2 * k + 1 >= cols) w[k] &= 0x0000FFFFu;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}
// the first `bytes` of the 16; the others become 0
__device__ __forceinline__ void copy_async_part(void* to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)),
               "l"(from), "r"(bytes)
               : "memory");
}
template <int BYTES>  // 4 or 8
__device__ __forceinline__ void copy_async_small(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
               "n"(BYTES)
               : "memory");
}

// Rows whose ends lie on 16-byte boundaries have only whole pieces (EDGE false).
// Otherwise a piece that a row's end cuts also has its neighbour's columns, which
// have to count as 0: those behind the row are not copied, those before it are
// cleared by their thread when the copy has landed (testing every piece as it is
// read took up to 1.5 times as long).

// Starts the copy of columns [e0, e0+V) of row `row`, on a 16-byte boundary and
// e0 < cols, to this thread's place `to`. Only before the tensor's first row may
// the neighbour's columns not be there, and only the row's are read then.
template <typename T, bool EDGE>
__device__ __forceinline__ void copy_piece(uint4* to, const T* x, int64_t row, int e0, int cols) {
  constexpr int V = elem::kVec<T>;
  const T* at = x + row * cols + e0;
  if constexpr (!EDGE) {
    copy_async(to, at);
  } else if (e0 >= 0 || at >= x) {
    copy_async_part(to, at, min(V, cols - e0) * (int)sizeof(T));
  } else {
    const int e = elem::opaque(e0);
#pragma unroll 1
    for (int j = 0; j < V; ++j) reinterpret_cast<T*>(to)[j] = e + j >= 0 && e + j < cols ? at[j] : T(0.f);
  }
}

// Stores the elements [lo, hi) of a piece of 16-bit values: the largest aligned
// parts in turn.
template <typename T>
__device__ __forceinline__ void store_part(T* at, const uint4& raw, int lo, int hi) {
  static_assert(sizeof(T) == 2, "");
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  auto one = [&](int e) {
    const uint32_t word = e < 2 ? w[0] : e < 4 ? w[1] : e < 6 ? w[2] : w[3];
    reinterpret_cast<uint16_t*>(at)[e] = (uint16_t)(e & 1 ? word >> 16 : word);
  };
  uint32_t* words = reinterpret_cast<uint32_t*>(at);
  uint2* halves = reinterpret_cast<uint2*>(at);
  if (lo > 0 && hi < 8) {
#pragma unroll 1
    for (int e = lo; e < hi; ++e) one(e);
  } else if (lo > 0) {
    if (lo & 1) one(lo++);
    if (lo & 2) {
      words[lo / 2] = lo == 2 ? w[1] : w[3];
      lo += 2;
    }
    if (lo == 4) halves[1] = make_uint2(w[2], w[3]);
  } else {
    if (hi & 4) halves[0] = make_uint2(w[0], w[1]);
    if (hi & 2) words[hi / 4 * 2] = hi & 4 ? w[2] : w[0];
    if (hi & 1) one(hi - 1);
  }
}

// PARTS: a cut piece by its parts, else by its elements, which takes fewer
// registers (16384x2049 bf16 by parts 54 and 80 us, by elements 59 and 89; where a
// thread of the backward pass has 32 columns, 4000x12345 bf16, 104 and 90 us).
template <typename T, bool EDGE, bool PARTS>
__device__ __forceinline__ void store_piece(T* row, int e0, int cols, const uint64_t (&f)[elem::kVec<T> / 2]) {
  constexpr int V = elem::kVec<T>;
  if (!EDGE || (e0 >= 0 && e0 + V <= cols)) {
    *reinterpret_cast<uint4*>(row + e0) = elem::pack_pairs<T>(f);
    return;
  }
  const int e = elem::opaque(e0);
  if constexpr (PARTS) {
    store_part<T>(row + e, elem::pack_pairs<T>(f), max(-e, 0), min(cols - e, V));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 h = elem::halves(f[j / 2]);
      if (e + j >= 0 && e + j < cols) row[e + j] = elem::from_f<T>(j % 2 ? h.y : h.x);
    }
  }
}

// The 16 bytes at byte `at` (0 to 15, a whole number of elements) of a and b.
template <typename T>
__device__ __forceinline__ uint4 bytes_at(const uint4& a, const uint4& b, int at) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const bool two = at & 8, one = at & 4;
#pragma unroll
  for (int k = 0; k < 6; ++k) w[k] = two ? w[k + 2] : w[k];
#pragma unroll
  for (int k = 0; k < 5; ++k) w[k] = one ? w[k + 1] : w[k];
  if constexpr (sizeof(T) == 2) {
    const uint32_t half = at & 2 ? 0x5432u : 0x3210u;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __byte_perm(w[k], w[k + 1], half);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// V bytes at byte `at` (1 to V) of the 2 V in raw.
template <int V>
__device__ __forceinline__ uint2 bytes8_at(const uint4& raw, int at) {
  const uint32_t by = 0x3210u + 0x1111u * (at & 3);
  if constexpr (V == 8) {
    const bool one = at >= 4, two = at >= 8;
    const uint32_t a = two ? raw.z : one ? raw.y : raw.x, b = two ? raw.w : one ? raw.z : raw.y;
    return make_uint2(__byte_perm(a, b, by), __byte_perm(b, one ? raw.w : raw.z, by));
  } else {
    return make_uint2(__byte_perm(at >= 4 ? raw.y : raw.x, raw.y, by), 0);
  }
}

// Rows of a CTA at a time, and its threads: rows of up to 64 threads share a CTA.
template <int TPR>
constexpr int kRows = TPR < 128 ? 128 / TPR : 1;
template <int TPR>
constexpr int kThreads = TPR * kRows<TPR>;

// Threads per SM that the registers are shared among: 16 columns of a thread take
// 80 (forward) and 128 (backward) with their weights and sums. A thread of wider
// rows has 32 columns and keeps gamma and beta in shared memory.
constexpr int kFwdThreads = 768, kBwdThreads = 512;
constexpr int kScalar = 16;  // columns of a thread, element by element
template <typename T, int VPT>
constexpr bool kHold = VPT * elem::kVec<T> <= 16;
template <int TPR, int PER_SM>
constexpr int kCtas = PER_SM / kThreads<TPR>;
template <typename T, int TPR, int VPT>
constexpr int kFwdPerSm = kHold<T, VPT> || TPR != 256 ? kFwdThreads : 512;
// Bytes that one weight vector takes in a CTA's shared memory.
template <typename T, int TPR, int VPT>
constexpr int kWeightBytes = kHold<T, VPT> ? 0 : VPT * elem::kVec<T> * 4 * kThreads<TPR>;
// Rows in shared memory: as many as 200 KB per SM hold (224 KB less the weights), up to 4.
template <typename T, int TPR, int VPT, int TENSORS, int PER_SM>
constexpr int kFit = ((kHold<T, VPT> ? 200 : 224) * 1024 / kCtas<TPR, PER_SM> -
                      (TENSORS == 1 ? 2 : 1) * kWeightBytes<T, TPR, VPT>) /
                     (TENSORS * VPT * 16 * kThreads<TPR>);
template <typename T, int TPR, int VPT, int TENSORS, int PER_SM>
constexpr int kDepth = kFit<T, TPR, VPT, TENSORS, PER_SM> >= 4 ? 4 : kFit<T, TPR, VPT, TENSORS, PER_SM>;
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Waits for the TPR threads of this row.
template <int TPR>
__device__ __forceinline__ void row_sync() {
  if constexpr (kRows<TPR> == 1) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / TPR), "n"(TPR) : "memory");
}

// Sum over the TPR threads of a row; every thread gets it. `scratch` holds a
// value per warp of the CTA; two calls in a row need different scratch.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  v = warp_sum(v);
  if constexpr (TPR > 32) {
    constexpr int NW = TPR / 32;
    const int lane = threadIdx.x & 31, row0 = threadIdx.x / TPR * NW;
    if (lane == 0) scratch[threadIdx.x >> 5] = v;
    row_sync<TPR>();
    v = scratch[row0 + lane % NW];
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* scratch) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (TPR > 32) {
    constexpr int NW = TPR / 32;
    const int lane = threadIdx.x & 31, row0 = threadIdx.x / TPR * NW;
    if (lane == 0) scratch[threadIdx.x >> 5] = make_float2(a, b);
    row_sync<TPR>();
    const float2 s = scratch[row0 + lane % NW];
    a = s.x;
    b = s.y;
#pragma unroll
    for (int o = NW / 2; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
  }
  return make_float2(a, b);
}

// A row's sum over its columns, rounded as by a division (per_col = 1 / cols alone
// is up to a step off, which x - mean would have in every column of a row of one
// value); infinities and NaNs as they are.
__device__ __forceinline__ float mean_of(float sum, int cols, float per_col) {
  const float m = sum * per_col, left = fmaf(-m, (float)cols, sum);
  return left == left ? fmaf(left, per_col, m) : m;
}

// Weights of columns [e0, e0 + V); `other` where there are none.
template <typename T>
__device__ __forceinline__ void load_weights(const void* w, int wdtype, int e0, int cols, float other,
                                             uint64_t (&pairs)[elem::kVec<T> / 2]) {
  constexpr int V = elem::kVec<T>;
  const int e = elem::opaque(e0);
  float f[V];
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = other;
  } else if (wdtype == KT_F32) {
    const float* at = static_cast<const float*>(w) + e;
    if (e >= 0 && e + V <= cols && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
#pragma unroll
      for (int k = 0; k < V / 4; ++k) {
        const float4 v = reinterpret_cast<const float4*>(at)[k];
        f[4 * k] = v.x; f[4 * k + 1] = v.y; f[4 * k + 2] = v.z; f[4 * k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = e + j >= 0 && e + j < cols ? at[j] : other;
    }
  } else if constexpr (sizeof(T) == 2) {  // of the input's type
    const T* at = static_cast<const T*>(w) + e;
    if (e >= 0 && e + V <= cols && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
      elem::unpack_vec<T>(*reinterpret_cast<const uint4*>(at), f);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = e + j >= 0 && e + j < cols ? elem::to_f(at[j]) : other;
    }
  }
#pragma unroll
  for (int j = 0; j < V / 2; ++j) pairs[j] = elem::pair(f[2 * j], f[2 * j + 1]);
}

// A piece's weights in this thread's places of shared memory.
template <typename T, int THREADS>
__device__ __forceinline__ void keep_weights(uint4* at, const uint64_t (&w)[elem::kVec<T> / 2]) {
#pragma unroll
  for (int j = 0; j < elem::kVec<T> / 4; ++j)
    *reinterpret_cast<ulonglong2*>(at + j * THREADS) = make_ulonglong2(w[2 * j], w[2 * j + 1]);
}
template <typename T, int THREADS>
__device__ __forceinline__ void kept_weights(const uint4* at, uint64_t (&w)[elem::kVec<T> / 2]) {
#pragma unroll
  for (int j = 0; j < elem::kVec<T> / 4; ++j) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(at + j * THREADS);
    w[2 * j] = v.x;
    w[2 * j + 1] = v.y;
  }
}

// ---------------------------------------------------------------- forward
// With EDGE a thread's pieces do not begin where blocks of the checkpoint do. Its
// eight (four) columns of a block are then part of its own piece and of the next
// thread's, which it reads too; q8 has whole words in a row and so needs no such
// care.
template <typename T, int TPR, int VPT, bool CKPT, bool EDGE>
__global__ void __launch_bounds__(kThreads<TPR>, kCtas<TPR, kFwdPerSm<T, TPR, VPT>>)
fwd_rows(const FwdArgs p) {
  using elem::add2;
  using elem::fma2;
  using elem::halves;
  using elem::mul2;
  using elem::pair;
  constexpr int V = elem::kVec<T>;
  constexpr int D = kDepth<T, TPR, VPT, 1, kFwdPerSm<T, TPR, VPT>>;
  static_assert(D >= 1, "a row fits shared memory");
  extern __shared__ uint4 ring[];  // [D][VPT][threads], then gamma and beta unless they are held
  __shared__ float red[2][32];
  const int t = threadIdx.x % TPR;
  const int cols = (int)p.cols;
  const float per_col = 1.f / (float)cols;
  const int64_t first = (int64_t)blockIdx.x * kRows<TPR> + threadIdx.x / TPR;
  const int64_t stride = (int64_t)gridDim.x * kRows<TPR>;
  const int shift = EDGE ? elem::misalign<T>(static_cast<const T*>(p.x) + first * cols) : 0;
  const int e_first = t * V - shift;  // this thread's pieces start at e_first + i TPR V
  auto place = [&](int slot, int i) { return ring + (slot * VPT + i) * kThreads<TPR> + threadIdx.x; };
  auto fetch = [&](int slot, int64_t row) {
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e0 = e_first + i * TPR * V;
        if (e0 < cols) copy_piece<T, EDGE>(place(slot, i), static_cast<const T*>(p.x), row, e0, cols);
      }
    }
    commit_copies();
  };
#pragma unroll 1
  for (int d = 0; d < D; ++d) fetch(d, first + d * stride);
  constexpr bool HOLD = kHold<T, VPT>;
  uint64_t g[HOLD ? VPT : 1][V / 2], b[HOLD ? VPT : 1][V / 2];
  auto kept = [&](int which, int i) {
    return ring + D * VPT * kThreads<TPR> + (which * VPT + i) * (V / 4) * kThreads<TPR> + threadIdx.x;
  };
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int h = HOLD ? i : 0;
    load_weights<T>(p.gamma, p.wdtype, e_first + i * TPR * V, cols, 1.f, g[h]);
    load_weights<T>(p.beta, p.wdtype, e_first + i * TPR * V, cols, 0.f, b[h]);
    if constexpr (!HOLD) {
      keep_weights<T, kThreads<TPR>>(kept(0, i), g[h]);
      keep_weights<T, kThreads<TPR>>(kept(1, i), b[h]);
    }
  }
  int slot = 0;
  for (int64_t row = first; row < p.rows; row += stride) {
    wait_copies<D - 1>();
    if (EDGE && e_first < 0) *place(slot, 0) = masked<T>(*place(slot, 0), e_first, cols);
    if constexpr (CKPT && EDGE) row_sync<TPR>();  // the other threads' copies
    // writes columns [k0, k0 + V) of the checkpoint; the lanes of a block together
    auto keep8 = [&](const uint64_t (&f)[V / 2], uint32_t top, int k0) {
      constexpr int LPB = 32 / V;  // lanes that share a block of 32 columns
#pragma unroll
      for (int o = 1; o < LPB; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (k0 < cols) {
        const uint32_t code = block_code(as_fp32<T>(top));
        const float up = code_up(code);
        uint32_t w[V / 4];
#pragma unroll
        for (int k = 0; k < V / 4; ++k) w[k] = quant8x4(f[2 * k], f[2 * k + 1], up, code);
        int8_t* qr = p.q8 + row * p.ld_q8 + k0;
        if constexpr (V == 8) *reinterpret_cast<uint2*>(qr) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(qr) = w[0];
        if (t % LPB == 0) p.q8_exp[row * ((cols + 31) / 32) + k0 / 32] = (uint8_t)code;
      }
    };
    uint64_t v[VPT][V / 2];
    uint32_t tops[VPT];
    uint64_t s2 = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (e0 < cols) raw = *place(slot, i);
      elem::unpack_pairs<T>(raw, v[i]);
      if constexpr (CKPT && !EDGE) tops[i] = top_bits<T>(raw);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) s2 = add2(s2, v[i][j]);
    }
    if constexpr (CKPT && EDGE) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e0 = e_first + i * TPR * V, k0 = e0 + shift;
        uint4 own = make_uint4(0, 0, 0, 0), next = own;
        if (e0 < cols) own = *place(slot, i);
        if (e0 + V < cols) next = t + 1 < TPR ? place(slot, i)[1] : *(place(slot, i + 1) - (TPR - 1));
        uint4 raw = bytes_at<T>(own, next, shift * (int)sizeof(T));
        uint64_t f[V / 2];
        elem::unpack_pairs<T>(raw, f);
        keep8(f, top_bits<T>(raw), k0);
      }
    } else {
      fetch(slot, row + D * stride);
    }
    const float mean = mean_of(row_sum<TPR>(halves(s2).x + halves(s2).y, red[0]), cols, per_col);
    if constexpr (CKPT && EDGE) {  // every thread has read its neighbour's piece
      if (TPR == 32) __syncwarp();
      fetch(slot, row + D * stride);
    }
    slot = slot + 1 == D ? 0 : slot + 1;
    const uint64_t minus = pair(-mean, -mean);
    if constexpr (CKPT && !EDGE) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) keep8(v[i], tops[i], e_first + i * TPR * V);
    }
    uint64_t q2 = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
      if (e0 >= cols) continue;
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[i][j] = add2(v[i][j], minus);
      if (EDGE && (e0 < 0 || e0 + V > cols)) {  // a piece that the row's end cuts
        const int e = elem::opaque(e0);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          const float2 h = halves(v[i][j]);
          v[i][j] = pair(e + 2 * j >= 0 && e + 2 * j < cols ? h.x : 0.f,
                         e + 2 * j + 1 >= 0 && e + 2 * j + 1 < cols ? h.y : 0.f);
        }
      }
#pragma unroll
      for (int j = 0; j < V / 2; ++j) q2 = fma2(v[i][j], v[i][j], q2);
    }
    const float rstd = rsqrtf(fmaf(row_sum<TPR>(halves(q2).x + halves(q2).y, red[1]), per_col, p.eps));
    if (t == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    T* yr = static_cast<T*>(p.y) + row * cols;
    const uint64_t by = pair(rstd, rstd);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
      if (e0 >= cols) continue;
      const int h = HOLD ? i : 0;
      if constexpr (!HOLD) {
        kept_weights<T, kThreads<TPR>>(kept(0, i), g[h]);
        kept_weights<T, kThreads<TPR>>(kept(1, i), b[h]);
      }
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[i][j] = fma2(mul2(v[i][j], by), g[h][j], b[h][j]);
      store_piece<T, EDGE, sizeof(T) == 2>(yr, e0, cols, v[i]);
    }
  }
}

// Wider rows, any alignment: a CTA per row, the row read once per step (from L2
// after the first). Lanes hold consecutive columns, so a warp's 32 columns are
// one block of the checkpoint.
template <typename T, bool CKPT>
__global__ void __launch_bounds__(256) fwd_any(const FwdArgs p) {
  __shared__ float red[2][32];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* xr = static_cast<const T*>(p.x) + row * p.cols;
    T* yr = static_cast<T*>(p.y) + row * p.cols;
    float s = 0.f;
    for (int64_t e = threadIdx.x; e < p.cols; e += 256) s += elem::to_f(xr[e]);
    const float mean = row_sum<256>(s, red[0]) / (float)p.cols;
    float q = 0.f;
    for (int64_t e = threadIdx.x; e < p.cols; e += 256) {
      const float d = elem::to_f(xr[e]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<256>(q, red[1]) / (float)p.cols + p.eps);
    if (threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (int64_t e0 = threadIdx.x & ~31; e0 < p.cols; e0 += 256) {
      const int64_t e = e0 + (threadIdx.x & 31);
      const float v = e < p.cols ? elem::to_f(xr[e]) : 0.f;
      if constexpr (CKPT) {
        const uint32_t code = block_code(__reduce_max_sync(0xffffffffu, abs_bits(v)));
        if (e < p.cols) p.q8[row * p.ld_q8 + e] = (int8_t)quant8(v, code_up(code));
        if ((threadIdx.x & 31) == 0) p.q8_exp[row * ((p.cols + 31) / 32) + e0 / 32] = (uint8_t)code;
      }
      if (e < p.cols) {
        const float g = p.gamma ? elem::ld_weight(p.gamma, p.wdtype, e) : 1.f;
        const float b = p.beta ? elem::ld_weight(p.beta, p.wdtype, e) : 0.f;
        yr[e] = elem::from_f<T>(fmaf((v - mean) * rstd, g, b));
      }
    }
  }
}

// ---------------------------------------------------------------- backward
// A piece of x - mean from x, or from its 8-bit checkpoint (.x, .y: eight values,
// .z: the code of the block, and 256 times that of the block before, to which the
// first `shift` columns of a piece may belong). The mean goes off before r is
// multiplied: x r - mean r would be off by the rounding of mean r where x is near
// the mean (a row of one value has xh = 0), and not finite where mean r is not.
template <typename T, bool CKPT, bool EDGE>
__device__ __forceinline__ void centred(const uint4& raw, int shift, float mean, uint64_t (&xm)[elem::kVec<T> / 2]) {
  using elem::pair;
  constexpr int V = elem::kVec<T>;
  const uint64_t minus = pair(-mean, -mean);
  if constexpr (CKPT) {
    const float down = code_down(raw.z & 255u), first = code_down(raw.z >> 8);
    const uint64_t bias = pair(-8388736.f, -8388736.f);  // 2^23 + 128
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      // q + 128 in the low bits of 2^23
      const uint32_t word = (j < 2 ? raw.x : raw.y) ^ 0x80808080u;
      const uint64_t q = (uint64_t)__byte_perm(word, 0x4B000000u, 0x7440 + (2 * (j & 1) + 1)) << 32 |
                         __byte_perm(word, 0x4B000000u, 0x7440 + 2 * (j & 1));
      const uint64_t scale = EDGE ? pair(2 * j < shift ? first : down, 2 * j + 1 < shift ? first : down)
                                  : pair(down, down);
      xm[j] = elem::fma2(elem::add2(q, bias), scale, minus);
    }
  } else {
    elem::unpack_pairs<T>(raw, xm);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) xm[j] = elem::add2(xm[j], minus);
  }
}

// Columns outside the row have dy = 0, so they add nothing to any sum.
template <typename T, int TPR, int VPT, bool CKPT, bool EDGE>
__global__ void __launch_bounds__(kThreads<TPR>, kCtas<TPR, kBwdThreads>)
bwd_rows(const BwdArgs p) {
  using elem::add2;
  using elem::fma2;
  using elem::halves;
  using elem::mul2;
  using elem::pair;
  constexpr int V = elem::kVec<T>;
  constexpr int RB = kRows<TPR>;
  constexpr int D = kDepth<T, TPR, VPT, 2, kBwdThreads>;
  static_assert(D >= 1, "a row fits shared memory");
  // [D][dy, x][VPT][threads], then gamma unless it is held; at the end, RB > 1: the rows' sums
  extern __shared__ uint4 ring[];
  __shared__ float2 red[2][32];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int cols = (int)p.cols;
  const float per_col = 1.f / (float)cols;
  const int64_t first = (int64_t)blockIdx.x * RB + sub;
  const int64_t stride = (int64_t)gridDim.x * RB;
  const int shift = EDGE ? elem::misalign<T>(static_cast<const T*>(p.dy) + first * cols) : 0;
  const int e_first = t * V - shift;
  auto place = [&](int slot, int which, int i) {
    return ring + ((slot * 2 + which) * VPT + i) * kThreads<TPR> + threadIdx.x;
  };
  auto fetch = [&](int slot, int64_t row) {
    if (row < p.rows) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e0 = e_first + i * TPR * V;
        if (e0 >= cols) continue;
        copy_piece<T, EDGE>(place(slot, 0, i), static_cast<const T*>(p.dy), row, e0, cols);
        if constexpr (CKPT) {  // with EDGE the word before as well
          const int8_t* from = p.q8 + row * p.ld_q8 + (e0 + shift);
          uint8_t* to = reinterpret_cast<uint8_t*>(place(slot, 1, i));
          if (!EDGE || e0 + shift < cols) copy_async_small<V>(to + (EDGE ? V : 0), from);
          if (EDGE && e0 + shift > 0) copy_async_small<V>(to, from - V);
        }
        if constexpr (!CKPT) copy_piece<T, EDGE>(place(slot, 1, i), static_cast<const T*>(p.x), row, e0, cols);
      }
    }
    commit_copies();
  };
  // a row's statistics and its blocks' codes, one row ahead
  float nmean = 0.f, nrstd = 0.f;
  uint32_t ncode[VPT];
  auto ahead = [&](int64_t row) {
    nmean = p.mean[row];
    nrstd = p.rstd[row];
    if constexpr (CKPT) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e0 = e_first + i * TPR * V;
        const int k0 = e0 + shift;
        const uint8_t* codes = p.q8_exp + row * ((cols + 31) / 32);
        ncode[i] = k0 < cols ? codes[k0 / 32] : 7u;
        if constexpr (EDGE) ncode[i] |= (k0 > 0 && e0 < cols ? codes[(k0 - 1) / 32] : 7u) << 8;
      }
    }
  };
#pragma unroll 1
  for (int d = 0; d < D; ++d) fetch(d, first + d * stride);
  if (first < p.rows) ahead(first);
  constexpr bool HOLD = kHold<T, VPT>;
  uint64_t g[HOLD ? VPT : 1][V / 2], dg[VPT][V / 2], db[VPT][V / 2];
  auto kept = [&](int i) {
    return ring + D * 2 * VPT * kThreads<TPR> + i * (V / 4) * kThreads<TPR> + threadIdx.x;
  };
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    load_weights<T>(p.gamma, p.wdtype, e_first + i * TPR * V, cols, 1.f, g[HOLD ? i : 0]);
    if constexpr (!HOLD) keep_weights<T, kThreads<TPR>>(kept(i), g[0]);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) dg[i][j] = db[i][j] = 0;
  }
  int turn = 0, slot = 0;
  for (int64_t row = first; row < p.rows; row += stride, turn ^= 1) {
    const float mean = nmean, rstd = nrstd;
    uint32_t code[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) code[i] = CKPT ? ncode[i] : 0;
    if (row + stride < p.rows) ahead(row + stride);
    // a piece of dy and x - mean; read for the sums and again for dx, as holding them takes twice the registers
    auto read = [&](int i, uint64_t (&d)[V / 2], uint64_t (&xm)[V / 2]) {
      elem::unpack_pairs<T>(*place(slot, 0, i), d);
      uint4 x;
      if constexpr (CKPT) {
        if constexpr (EDGE) {
          const uint2 q = bytes8_at<V>(*place(slot, 1, i), V - shift);
          x = make_uint4(q.x, q.y, code[i], 0);
        } else {
          const uint32_t* at = reinterpret_cast<const uint32_t*>(place(slot, 1, i));
          x = make_uint4(at[0], V == 8 ? at[1] : 0, code[i], 0);
        }
      } else {
        x = *place(slot, 1, i);
      }
      centred<T, CKPT, EDGE>(x, shift, mean, xm);
    };
    wait_copies<D - 1>();
    if (EDGE && e_first < 0) {
      *place(slot, 0, 0) = masked<T>(*place(slot, 0, 0), e_first, cols);
      if constexpr (!CKPT) *place(slot, 1, 0) = masked<T>(*place(slot, 1, 0), e_first, cols);
    }
    const uint64_t by = pair(rstd, rstd);
    uint64_t s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
      if (e0 >= cols) continue;
      uint64_t d[V / 2], xm[V / 2];
      read(i, d, xm);
      const int h = HOLD ? i : 0;
      if constexpr (!HOLD) kept_weights<T, kThreads<TPR>>(kept(i), g[h]);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const uint64_t xh = mul2(xm[j], by);
        dg[i][j] = fma2(d[j], xh, dg[i][j]);
        db[i][j] = add2(db[i][j], d[j]);
        const uint64_t w = mul2(d[j], g[h][j]);
        s1 = fma2(w, xh, s1);
        s2 = add2(s2, w);
      }
    }
    const float2 s = row_sum2<TPR>(halves(s1).x + halves(s1).y, halves(s2).x + halves(s2).y, red[turn]);
    const float c1 = -s.x * per_col * rstd, c2 = -mean_of(s.y, cols, per_col);
    const uint64_t m1 = pair(c1, c1), m2 = pair(c2, c2);
    T* dxr = static_cast<T*>(p.dx) + row * cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
      if (e0 >= cols) continue;
      uint64_t d[V / 2], xm[V / 2];
      read(i, d, xm);
      const int h = HOLD ? i : 0;
      if constexpr (!HOLD) kept_weights<T, kThreads<TPR>>(kept(i), g[h]);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) d[j] = mul2(by, fma2(xm[j], m1, fma2(d[j], g[h][j], m2)));
      store_piece<T, EDGE, sizeof(T) == 2 && HOLD>(dxr, e0, cols, d);
    }
    fetch(slot, row + D * stride);
    slot = slot + 1 == D ? 0 : slot + 1;
  }
  wait_copies<0>();
  if (p.partial == nullptr) return;
  float* out = p.partial + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (RB == 1) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
      if (!EDGE && e0 < cols) {  // cols is a multiple of 4
#pragma unroll
        for (int j = 0; j < V / 2; j += 2) {
          *reinterpret_cast<ulonglong2*>(out + e0 + 2 * j) = make_ulonglong2(dg[i][j], dg[i][j + 1]);
          *reinterpret_cast<ulonglong2*>(out + cols + e0 + 2 * j) = make_ulonglong2(db[i][j], db[i][j + 1]);
        }
        continue;
      }
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j >= 0 && e0 + j < cols) {
          out[e0 + j] = j % 2 ? halves(dg[i][j / 2]).y : halves(dg[i][j / 2]).x;
          out[cols + e0 + j] = j % 2 ? halves(db[i][j / 2]).y : halves(db[i][j / 2]).x;
        }
    }
  } else {
    float* part = reinterpret_cast<float*>(ring);  // [RB][2][cols]
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * TPR * V;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j >= 0 && e0 + j < cols) {
          part[sub * 2 * cols + e0 + j] = j % 2 ? halves(dg[i][j / 2]).y : halves(dg[i][j / 2]).x;
          part[(sub * 2 + 1) * cols + e0 + j] = j % 2 ? halves(db[i][j / 2]).y : halves(db[i][j / 2]).x;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * cols; e += kThreads<TPR>) {  // in the order of the rows
      float v = part[e];
#pragma unroll
      for (int w = 1; w < RB; ++w) v += part[w * 2 * cols + e];
      out[e] = v;
    }
  }
}

// ---------------------------------------------------------------- element by element
// Rows of x and y, or dy and dx, that are not equally aligned (an input that begins
// off a 16-byte boundary: 16384x4096 bf16 205 and 249 us), and checkpoints whose rows
// are no whole words: lanes hold consecutive columns (a warp's 32 are one
// block of the checkpoint), EPT per thread, as above but for the copies ahead.
template <typename T, int TPR, bool CKPT>
__global__ void __launch_bounds__(TPR) fwd_scalar(const FwdArgs p) {
  constexpr int EPT = kScalar;
  __shared__ float red[2][32];
  const int t = threadIdx.x, cols = (int)p.cols;
  const float per_col = 1.f / (float)cols;
  T next[EPT];
  auto fetch = [&](int64_t row) {
    const T* xr = static_cast<const T*>(p.x) + row * cols;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (t + i * TPR < cols) next[i] = xr[t + i * TPR];
  };
  fetch(blockIdx.x);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float v[EPT];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      v[i] = t + i * TPR < cols ? elem::to_f(next[i]) : 0.f;
      s += v[i];
    }
    if (row + gridDim.x < p.rows) fetch(row + gridDim.x);
    const float mean = mean_of(row_sum<TPR>(s, red[0]), cols, per_col);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (t + i * TPR < cols) q = fmaf(v[i] - mean, v[i] - mean, q);
    const float rstd = rsqrtf(fmaf(row_sum<TPR>(q, red[1]), per_col, p.eps));
    if (t == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    T* yr = static_cast<T*>(p.y) + row * cols;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int e = t + i * TPR;
      if constexpr (CKPT) {
        const uint32_t code = block_code(__reduce_max_sync(0xffffffffu, abs_bits(v[i])));
        if (e < cols) p.q8[row * p.ld_q8 + e] = (int8_t)quant8(v[i], code_up(code));
        if (e < cols && (t & 31) == 0) p.q8_exp[row * ((cols + 31) / 32) + e / 32] = (uint8_t)code;
      }
      if (e < cols) {
        const float g = p.gamma ? elem::ld_weight(p.gamma, p.wdtype, e) : 1.f;
        const float b = p.beta ? elem::ld_weight(p.beta, p.wdtype, e) : 0.f;
        yr[e] = elem::from_f<T>(fmaf((v[i] - mean) * rstd, g, b));
      }
    }
  }
}

template <typename T, int TPR, bool CKPT>
__global__ void __launch_bounds__(TPR) bwd_scalar(const BwdArgs p) {
  constexpr int EPT = kScalar;
  __shared__ float2 red[2][32];
  const int t = threadIdx.x, cols = (int)p.cols;
  const float per_col = 1.f / (float)cols;
  float g[EPT], dg[EPT], db[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    g[i] = t + i * TPR < cols && p.gamma ? elem::ld_weight(p.gamma, p.wdtype, t + i * TPR) : 1.f;
    dg[i] = db[i] = 0.f;
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const T* dyr = static_cast<const T*>(p.dy) + row * cols;
    T* dxr = static_cast<T*>(p.dx) + row * cols;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float d[EPT], xh[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int e = t + i * TPR;
      d[i] = e < cols ? elem::to_f(dyr[e]) : 0.f;
      if constexpr (CKPT) {
        xh[i] = e < cols ? (float)p.q8[row * p.ld_q8 + e] * code_down(p.q8_exp[row * ((cols + 31) / 32) + e / 32]) : 0.f;
      } else {
        xh[i] = e < cols ? elem::to_f(static_cast<const T*>(p.x)[row * cols + e]) : 0.f;
      }
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {  // columns outside the row have d = 0
      xh[i] = (xh[i] - mean) * rstd;
      dg[i] = fmaf(d[i], xh[i], dg[i]);
      db[i] += d[i];
      d[i] *= g[i];
      s1 = fmaf(d[i], xh[i], s1);
      s2 += d[i];
    }
    const float2 s = row_sum2<TPR>(s1, s2, red[turn]);
    const float c1 = s.x * per_col, c2 = mean_of(s.y, cols, per_col);
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (t + i * TPR < cols) dxr[t + i * TPR] = elem::from_f<T>(rstd * (d[i] - c2 - xh[i] * c1));
  }
  if (p.partial == nullptr) return;
  float* out = p.partial + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    if (t + i * TPR < cols) {
      out[t + i * TPR] = dg[i];
      out[cols + t + i * TPR] = db[i];
    }
}

// Wider rows, any alignment: dx by a CTA per row, and the partial sums by columns.
template <typename T, bool CKPT>
__device__ __forceinline__ float x_hat(const BwdArgs& p, int64_t row, int64_t e, float mean, float rstd) {
  float v;
  if constexpr (CKPT)
    v = (float)p.q8[row * p.ld_q8 + e] * code_down(p.q8_exp[row * ((p.cols + 31) / 32) + e / 32]);
  else
    v = elem::to_f(static_cast<const T*>(p.x)[row * p.cols + e]);
  return (v - mean) * rstd;
}

template <typename T, bool CKPT>
__global__ void __launch_bounds__(256) bwd_any_dx(const BwdArgs p) {
  __shared__ float2 red[2][32];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const T* dyr = static_cast<const T*>(p.dy) + row * p.cols;
    T* dxr = static_cast<T*>(p.dx) + row * p.cols;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t e = threadIdx.x; e < p.cols; e += 256) {
      const float w = elem::to_f(dyr[e]) * (p.gamma ? elem::ld_weight(p.gamma, p.wdtype, e) : 1.f);
      s1 = fmaf(w, x_hat<T, CKPT>(p, row, e, mean, rstd), s1);
      s2 += w;
    }
    const float2 s = row_sum2<256>(s1, s2, red[turn]);
    const float c1 = s.x / (float)p.cols, c2 = s.y / (float)p.cols;
    for (int64_t e = threadIdx.x; e < p.cols; e += 256) {
      const float w = elem::to_f(dyr[e]) * (p.gamma ? elem::ld_weight(p.gamma, p.wdtype, e) : 1.f);
      dxr[e] = elem::from_f<T>(rstd * (w - c2 - x_hat<T, CKPT>(p, row, e, mean, rstd) * c1));
    }
  }
}

template <typename T, bool CKPT>
__global__ void __launch_bounds__(256) bwd_any_cols(const BwdArgs p) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= p.cols) return;
  const int64_t lo = p.rows * blockIdx.y / gridDim.y, hi = p.rows * (blockIdx.y + 1) / gridDim.y;
  float dg = 0.f, db = 0.f;
  for (int64_t row = lo; row < hi; ++row) {
    const float d = elem::to_f(static_cast<const T*>(p.dy)[row * p.cols + e]);
    dg = fmaf(d, x_hat<T, CKPT>(p, row, e, p.mean[row], p.rstd[row]), dg);
    db += d;
  }
  float* out = p.partial + (int64_t)blockIdx.y * 2 * p.cols;
  out[e] = dg;
  out[p.cols + e] = db;
}

// dgamma, dbeta: the partial rows added in their order. 32 columns per CTA; each
// of 32 warps adds a slice of the rows, eight loads at a time, and the slices are
// joined in shared memory. (The loads' latency is what it takes: 8 slices took
// three times as long.)
__global__ void __launch_bounds__(1024)
bwd_join(const float* partial, int parts, int64_t cols, void* dgamma, void* dbeta, int wdtype) {
  __shared__ float slice[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t e = (int64_t)blockIdx.x * 32 + lane;  // over 2 x cols: dgamma, then dbeta
  float s = 0.f;
  cudaGridDependencySynchronize();
  if (e < 2 * cols) {
    const float* from = partial + e;
    int r = parts * w / 32;
    const int end = parts * (w + 1) / 32;
    for (; r + 8 <= end; r += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from[(int64_t)(r + i) * 2 * cols];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
#pragma unroll 4
    for (; r < end; ++r) s += from[(int64_t)r * 2 * cols];
  }
  slice[w][lane] = s;
  __syncthreads();
  s = warp_sum(slice[lane][w]);  // column w of the CTA's
  const int64_t out = (int64_t)blockIdx.x * 32 + w;
  if (lane == 0 && out < 2 * cols) {
    if (out < cols) {
      if (dgamma) elem::st_weight(dgamma, wdtype, out, s);
    } else if (dbeta) {
      elem::st_weight(dbeta, wdtype, out - cols, s);
    }
  }
}

// ---------------------------------------------------------------- host
constexpr int64_t kMaxParts = 1184;  // 8 CTAs on each of 148 SMs

// Partial rows that one call may use.
inline int64_t max_parts(int64_t rows) { return rows < kMaxParts ? rows : kMaxParts; }

inline size_t workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)max_parts(rows) * 2 * (size_t)cols * sizeof(float);
}

// CTAs for `rows`: what the device holds at once, at most one per `rb` rows and
// kMaxParts; a multiple of 8 where a CTA has several turns, so that its rows
// start at equal offsets within 16 bytes.
template <class K>
inline int row_grid(K kern, int block, int rb, size_t smem, int64_t rows, int* grid) {
  int per_sm = 0;
  const int rc = resident_ctas((const void*)kern, block, smem, &per_sm, "layernorm_train: launch shape");
  if (rc != KT_OK) return rc;
  if (per_sm < 1) return fail(KT_ERR_UNSUPPORTED, "layernorm_train: no CTA fits");
  const int64_t need = (rows + rb - 1) / rb;
  int64_t g = (int64_t)sm_count() * per_sm;
  if (g > kMaxParts) g = kMaxParts;
  g = g / 8 * 8;
  *grid = (int)(need <= g ? need : (g > 0 ? g : 8));
  return KT_OK;
}

// Calls f with the threads per row and pieces per thread for a row of `pieces`
// 16-byte pieces: 16 columns per thread (32 in the widest rows). False when a row
// is too wide. Rows of up to 64 threads share a CTA where there are more than four
// per SM (16384x512 bf16 forward: 7.5 us, and 15 by 128 threads a row); fewer rows
// are spread over the SMs (64x512 backward: 4.1 us, and 4.8 by 32 threads a row).
// Where `twice` says so, rows of 4097 to 8192 columns go to 256 threads of 32
// columns: two CTAs share an SM, and one works while the other waits for a row's
// sum (8000x8000 fp16 forward 46.5 us, and 53.1 by 512 threads; 1021x8192 11 and 10).
template <typename T, class F>
inline bool with_shape(int64_t pieces, int64_t rows, bool twice, F f) {
  constexpr int VPT = 16 / elem::kVec<T>;
  const bool many = rows > 4 * sm_count();
  using One = std::integral_constant<int, 1>;
  using All = std::integral_constant<int, VPT>;
  if (pieces <= 32 && many) return f(std::integral_constant<int, 32>{}, One{}), true;
  if (pieces <= 32 * VPT && many) return f(std::integral_constant<int, 32>{}, All{}), true;
  if (pieces <= 64 * VPT && many) return f(std::integral_constant<int, 64>{}, All{}), true;
  using Twice = std::integral_constant<int, 2 * VPT>;
  if (pieces <= 128 * VPT) return f(std::integral_constant<int, 128>{}, All{}), true;
  if (pieces <= 256 * VPT) return f(std::integral_constant<int, 256>{}, All{}), true;
  if (pieces <= 512 * VPT && twice) return f(std::integral_constant<int, 256>{}, Twice{}), true;
  if (pieces <= 512 * VPT) return f(std::integral_constant<int, 512>{}, All{}), true;
  if (pieces <= 1024 * VPT) return f(std::integral_constant<int, 512>{}, Twice{}), true;
  return false;
}

inline int check_common(const char* what, int64_t rows, int64_t cols, int dtype, int wdtype) {
  if (rows < 0 || cols < 0)
    return fail(KT_ERR_ARG, "%s: negative shape rows=%lld cols=%lld", what, (long long)rows, (long long)cols);
  if (elem::size_of(dtype) == 0) return fail(KT_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (wdtype != KT_F32 && wdtype != dtype)
    return fail(KT_ERR_ARG, "%s: weights are fp32 or of the input's type", what);
  if (cols > INT32_MAX / 2) return fail(KT_ERR_UNSUPPORTED, "%s: cols > 2^30", what);
  return KT_OK;
}

// Whether a checkpoint's rows are written and read by V bytes at a time: the last
// of them reach behind a row only where its distance is a multiple of 8.
template <int V>
inline bool whole_words(const int8_t* q8, int64_t ld, int64_t cols) {
  return elem::aligned_to(q8, V) && (ld % 8 == 0 || (ld % V == 0 && cols % V == 0));
}

// Whether two tensors of one size share memory without being one: CTAs would read
// what others have stored.
inline bool partly_one(const void* a, const void* b, size_t bytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x != y && x < y + bytes && y < x + bytes;
}

template <typename T, bool CKPT>
inline int fwd_typed(const FwdArgs& a, cudaStream_t st) {
  constexpr int V = elem::kVec<T>;
  const int shift = elem::misalign<T>(a.x);
  bool fast = elem::misalign<T>(a.y) == shift;
  if (CKPT) fast = fast && whole_words<V>(a.q8, a.ld_q8, a.cols);
  const bool edge = shift != 0 || a.cols % V != 0;
  const int64_t pieces = (a.cols + V - 1) / V + (edge ? 1 : 0);
  int rc = KT_OK;
  if (fast && with_shape<T>(pieces, a.rows, a.rows > 16 * sm_count(), [&](auto tpr, auto vpt) {
        constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
        constexpr int RB = kRows<TPR>, BLOCK = kThreads<TPR>;
        auto kern = edge ? fwd_rows<T, TPR, VPT, CKPT, true> : fwd_rows<T, TPR, VPT, CKPT, false>;
        constexpr size_t smem = (size_t)kDepth<T, TPR, VPT, 1, kFwdPerSm<T, TPR, VPT>> * VPT * BLOCK * 16 +
                                2 * kWeightBytes<T, TPR, VPT>;
        int grid = 0;
        rc = row_grid(kern, BLOCK, RB, smem, a.rows, &grid);
        if (rc != KT_OK) return;
        kern<<<grid, BLOCK, smem, st>>>(a);
        rc = check_launch("layernorm_train fwd_rows");
      }))
    return rc;
  if (a.cols <= 512 * kScalar) {
    auto kern = a.cols <= 128 * kScalar ? fwd_scalar<T, 128, CKPT> : fwd_scalar<T, 512, CKPT>;
    const int block = a.cols <= 128 * kScalar ? 128 : 512;
    int grid = 0;
    rc = row_grid(kern, block, 1, 0, a.rows, &grid);
    if (rc != KT_OK) return rc;
    kern<<<grid, block, 0, st>>>(a);
    return check_launch("layernorm_train fwd_scalar");
  }
  const int64_t g = a.rows < 4 * sm_count() ? a.rows : 4 * sm_count();
  fwd_any<T, CKPT><<<(int)g, 256, 0, st>>>(a);
  return check_launch("layernorm_train fwd_any");
}

inline int forward(const FwdArgs& a, int dtype, cudaStream_t st) {
  int rc = check_common("layernorm_train", a.rows, a.cols, dtype, a.wdtype);
  if (rc != KT_OK) return rc;
  if (!(a.eps >= 0.f)) return fail(KT_ERR_ARG, "layernorm_train: eps must be >= 0");
  if ((a.q8 == nullptr) != (a.q8_exp == nullptr))
    return fail(KT_ERR_ARG, "layernorm_train: q8 and q8_exp are given together");
  if (a.q8 && a.ld_q8 < a.cols) return fail(KT_ERR_ARG, "layernorm_train: rows of q8 overlap");
  if (a.rows == 0 || a.cols == 0) return KT_OK;
  if (!a.x || !a.y || !a.mean || !a.rstd) return fail(KT_ERR_ARG, "layernorm_train: null pointer");
  const int sz = elem::size_of(dtype), wsz = elem::size_of(a.wdtype);
  if (!elem::aligned_to(a.x, sz) || !elem::aligned_to(a.y, sz) || !elem::aligned_to(a.gamma, wsz) ||
      !elem::aligned_to(a.beta, wsz) || !elem::aligned_to(a.mean, 4) || !elem::aligned_to(a.rstd, 4))
    return fail(KT_ERR_ARG, "layernorm_train: a pointer is not aligned to its elements");
  if (partly_one(a.x, a.y, (size_t)(a.rows * a.cols) * sz))
    return fail(KT_ERR_ARG, "layernorm_train: y overlaps x without being it");
  if (dtype == KT_F32) return a.q8 ? fwd_typed<float, true>(a, st) : fwd_typed<float, false>(a, st);
  if (dtype == KT_BF16) return a.q8 ? fwd_typed<__nv_bfloat16, true>(a, st) : fwd_typed<__nv_bfloat16, false>(a, st);
  return a.q8 ? fwd_typed<__half, true>(a, st) : fwd_typed<__half, false>(a, st);
}

template <typename T, bool CKPT>
inline int bwd_typed(const BwdArgs& a, void* dgamma, void* dbeta, cudaStream_t st) {
  constexpr int V = elem::kVec<T>;
  const int shift = elem::misalign<T>(a.dy);
  bool fast = elem::misalign<T>(a.dx) == shift;
  if (CKPT) fast = fast && whole_words<V>(a.q8, a.ld_q8, a.cols);
  else fast = fast && elem::misalign<T>(a.x) == shift;
  const bool edge = shift != 0 || a.cols % V != 0;
  const int64_t pieces = (a.cols + V - 1) / V + (edge ? 1 : 0);
  int rc = KT_OK, parts = 0;
  // (8000x8000 fp16 72 us, and 77 by 512 threads; odd widths with checkpoints 140
  // and 162; whole pieces with checkpoints 88 and 81, 4096x8192 fp32 87 and 71,
  // 2400x8192 bf16 33 and 31)
  const bool twice = sizeof(T) == 2 && (!CKPT || edge) && a.rows > 32 * sm_count();
  if (!(fast && with_shape<T>(pieces, a.rows, twice, [&](auto tpr, auto vpt) {
          constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
          constexpr int RB = kRows<TPR>, BLOCK = kThreads<TPR>;
          auto kern = edge ? bwd_rows<T, TPR, VPT, CKPT, true> : bwd_rows<T, TPR, VPT, CKPT, false>;
          constexpr size_t smem = (size_t)kDepth<T, TPR, VPT, 2, kBwdThreads> * 2 * VPT * BLOCK * 16 +
                                  kWeightBytes<T, TPR, VPT>;
          static_assert(RB == 1 || smem >= RB * 2 * sizeof(float) * TPR * VPT * V, "the CTA's sums fit the ring");
          rc = row_grid(kern, BLOCK, RB, smem, a.rows, &parts);
          if (rc != KT_OK) return;
          kern<<<parts, BLOCK, smem, st>>>(a);
          rc = check_launch("layernorm_train bwd_rows");
        }))) {
    if (a.cols <= 512 * kScalar) {
      auto kern = a.cols <= 128 * kScalar ? bwd_scalar<T, 128, CKPT> : bwd_scalar<T, 512, CKPT>;
      const int block = a.cols <= 128 * kScalar ? 128 : 512;
      rc = row_grid(kern, block, 1, 0, a.rows, &parts);
      if (rc != KT_OK) return rc;
      kern<<<parts, block, 0, st>>>(a);
      rc = check_launch("layernorm_train bwd_scalar");
    } else {
      if (a.partial) {  // before dx, which may take dy's or x's place
        parts = (int)(a.rows < 64 ? a.rows : 64);
        bwd_any_cols<T, CKPT><<<dim3((unsigned)((a.cols + 255) / 256), (unsigned)parts), 256, 0, st>>>(a);
        rc = check_launch("layernorm_train bwd_any_cols");
        if (rc != KT_OK) return rc;
      }
      const int64_t g = a.rows < 4 * sm_count() ? a.rows : 4 * sm_count();
      bwd_any_dx<T, CKPT><<<(int)g, 256, 0, st>>>(a);
      rc = check_launch("layernorm_train bwd_any_dx");
    }
  }
  if (rc != KT_OK || a.partial == nullptr) return rc;
  // the join may be launched while the rows finish: it waits for them itself
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((2 * a.cols + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const float* partial = a.partial;
  return cuda_status(cudaLaunchKernelEx(&cfg, bwd_join, partial, parts, a.cols, dgamma, dbeta, a.wdtype),
                     "layernorm_train bwd_join");
}

inline int backward(BwdArgs a, int dtype, void* dgamma, void* dbeta, void* workspace, size_t ws_bytes,
                    cudaStream_t st) {
  int rc = check_common("layernorm_train bwd", a.rows, a.cols, dtype, a.wdtype);
  if (rc != KT_OK) return rc;
  if ((a.q8 == nullptr) != (a.q8_exp == nullptr))
    return fail(KT_ERR_ARG, "layernorm_train bwd: q8 and q8_exp are given together");
  if (a.q8 && a.ld_q8 < a.cols) return fail(KT_ERR_ARG, "layernorm_train bwd: rows of q8 overlap");
  if (a.cols == 0) return KT_OK;
  const int sz = elem::size_of(dtype), wsz = elem::size_of(a.wdtype);
  if (!elem::aligned_to(dgamma, wsz) || !elem::aligned_to(dbeta, wsz))
    return fail(KT_ERR_ARG, "layernorm_train bwd: a pointer is not aligned to its elements");
  if (a.rows == 0) {  // empty sums
    if (dgamma) rc = cuda_status(cudaMemsetAsync(dgamma, 0, (size_t)a.cols * wsz, st), "layernorm_train bwd: dgamma");
    if (rc == KT_OK && dbeta)
      rc = cuda_status(cudaMemsetAsync(dbeta, 0, (size_t)a.cols * wsz, st), "layernorm_train bwd: dbeta");
    return rc;
  }
  if (!a.dy || !a.dx || !a.mean || !a.rstd) return fail(KT_ERR_ARG, "layernorm_train bwd: null pointer");
  if ((a.x == nullptr) == (a.q8 == nullptr))
    return fail(KT_ERR_ARG, "layernorm_train bwd: give x or its 8-bit checkpoint, not both");
  if (!elem::aligned_to(a.dy, sz) || !elem::aligned_to(a.x, sz) || !elem::aligned_to(a.dx, sz) ||
      !elem::aligned_to(a.gamma, wsz) || !elem::aligned_to(a.mean, 4) || !elem::aligned_to(a.rstd, 4))
    return fail(KT_ERR_ARG, "layernorm_train bwd: a pointer is not aligned to its elements");
  if (partly_one(a.dx, a.dy, (size_t)(a.rows * a.cols) * sz) || partly_one(a.dx, a.x, (size_t)(a.rows * a.cols) * sz))
    return fail(KT_ERR_ARG, "layernorm_train bwd: dx overlaps dy or x without being it");
  a.partial = nullptr;
  if (dgamma || dbeta) {
    if (workspace == nullptr || ws_bytes < workspace_bytes(a.rows, a.cols) || !aligned16(workspace))
      return fail(KT_ERR_ARG, "layernorm_train bwd: workspace too small or not 16-byte aligned (%zu < %zu bytes)",
                  ws_bytes, workspace_bytes(a.rows, a.cols));
    a.partial = static_cast<float*>(workspace);
  }
  if (dtype == KT_F32) return a.q8 ? bwd_typed<float, true>(a, dgamma, dbeta, st)
                                   : bwd_typed<float, false>(a, dgamma, dbeta, st);
  if (dtype == KT_BF16) return a.q8 ? bwd_typed<__nv_bfloat16, true>(a, dgamma, dbeta, st)
                                    : bwd_typed<__nv_bfloat16, false>(a, dgamma, dbeta, st);
  return a.q8 ? bwd_typed<__half, true>(a, dgamma, dbeta, st) : bwd_typed<__half, false>(a, dgamma, dbeta, st);
}

}  // namespace ln_train
}  // namespace kt
