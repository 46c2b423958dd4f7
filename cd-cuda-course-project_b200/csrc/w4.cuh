// w4.cuh — products of a few tokens with a matrix of 4-bit weights:
//   y[m][n] = bias[n] + sum over groups G of s[n][G] sum over k in G of x[m][k] (q[n][k] - z[n][G])
// q in 0..15, two to a byte (even k in the low half), G of 32, 64 or 128
// columns, z = 8 where no zeros are given.
//
// Bound by memory: the weights are read once, N K / 2 bytes. At 6.5 TB/s that
// is 13 weights per clock and lane slot at most 2.6 instructions each, which
// fp32 multiply-adds per token would exceed from the second token on. So the
// sums run on the tensor cores (mma.sync m16n8k16: 16 weight rows by 8 tokens,
// fp32 accumulation; a tcgen05 tile of 128 rows would need the weights
// unpacked through shared memory): q - z is exact in 16 bits (or-ing q into
// the mantissa of 128 (bf16) or 1024 (fp16), then one packed subtraction), and
// so are its products with x; the scale multiplies each group's fp32 sum. fp32
// tokens are split exactly into three bf16 parts.
//
// A warp takes 16 rows and segments of 128 columns: each lane loads 16 bytes
// (32 weights) of two rows, which are four words of each row, for eight
// m16n8k16 steps. The columns a step covers can be any 16 as long as x has the
// same order, so no weight is moved between lanes for groups of 128. For
// smaller groups the four lanes of a row transpose their 4x4 words first, so
// that each word index belongs to one group. x is staged in shared memory in
// the order in which the steps read it.
//
// A CTA covers 16 rows x row-warps; its other warps, and the CTAs of a cluster,
// split the columns, and their sums are added in a fixed order through
// (distributed) shared memory.
#pragma once
#include <cooperative_groups.h>

#include "elem.cuh"

namespace kt {
namespace w4 {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSeg = 128;          // columns of a warp step
constexpr int kMaxTokens = 16;     // of one CTA; more tokens take more CTAs
constexpr int kMaxCluster = 8;
constexpr int kStageBytes = 96 * 1024;  // at most, for x

struct Args {
  const void* x;
  int64_t ldx;
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;
  const void* bias;
  void* y;
  int64_t ldy;
  int64_t M, N, K;
  int scale_dtype;
  int row_warps;   // warps of a CTA along N
  int chunk;       // columns staged at a time, a multiple of kSeg
};

// fp32 is multiplied as bf16 parts
template <typename T>
struct Mma {
  using type = T;
  static constexpr int parts = 1;
};
template <>
struct Mma<float> {
  using type = __nv_bfloat16;
  static constexpr int parts = 3;
};

template <typename H>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (base + zero) twice, where base + q has q in its low mantissa bits.
template <typename H>
__device__ __forceinline__ uint32_t zero_pair(int zero);
template <>
__device__ __forceinline__ uint32_t zero_pair<__nv_bfloat16>(int zero) { return 0x43004300u + 0x00010001u * zero; }
template <>
__device__ __forceinline__ uint32_t zero_pair<__half>(int zero) { return 0x64006400u + 0x00010001u * zero; }

// Pair i of a word: columns i and i + 4 of its eight, minus the zero.
template <typename H>
__device__ __forceinline__ uint32_t weights(uint32_t word, int i, uint32_t zero) {
  constexpr uint32_t base = std::is_same<H, __half>::value ? 0x64006400u : 0x43004300u;
  const uint32_t q = ((word >> (4 * i)) & 0x000F000Fu) | base;
  if constexpr (std::is_same<H, __half>::value) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&q), *reinterpret_cast<const __half2*>(&zero));
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&q), *reinterpret_cast<const __nv_bfloat162*>(&zero));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// 4x4 words among the four lanes of a row: lane t's word j becomes lane j's word t.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4], int t) {
  // halves of 2x2 blocks, then single words
  const bool hi = t & 2, odd = t & 1;
  uint32_t a = hi ? w[0] : w[2], b = hi ? w[1] : w[3];
  a = __shfl_xor_sync(0xffffffffu, a, 2);
  b = __shfl_xor_sync(0xffffffffu, b, 2);
  if (hi) { w[0] = a; w[1] = b; } else { w[2] = a; w[3] = b; }
  a = odd ? w[0] : w[1];
  b = odd ? w[2] : w[3];
  a = __shfl_xor_sync(0xffffffffu, a, 1);
  b = __shfl_xor_sync(0xffffffffu, b, 1);
  if (odd) { w[0] = a; w[2] = b; } else { w[1] = a; w[3] = b; }
}

// Eight columns of a token, in the order in which the steps read them.
template <typename H>
__device__ __forceinline__ uint4 order8(const float (&f)[8]) {
  return make_uint4(elem::pack2<H>(f[0], f[4]), elem::pack2<H>(f[1], f[5]), elem::pack2<H>(f[2], f[6]),
                    elem::pack2<H>(f[3], f[7]));
}

// GROUP: columns per scale. NT: blocks of 8 tokens of a CTA.
template <typename T, int GROUP, int NT>
__global__ void __launch_bounds__(kThreads) w4_kernel(const Args p) {
  namespace cg = cooperative_groups;
  using H = typename Mma<T>::type;
  constexpr int P = Mma<T>::parts;
  constexpr int GPS = kSeg / GROUP;  // groups of a segment
  extern __shared__ __align__(16) uint8_t smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rw = warp % p.row_warps, kw = warp / p.row_warps, k_warps = kWarps / p.row_warps;
  const int64_t block_row = (int64_t)blockIdx.x / split * (16 * p.row_warps);
  const int64_t m0 = (int64_t)blockIdx.y * (8 * NT);
  const int tokens = (int)(p.M - m0 < 8 * NT ? p.M - m0 : 8 * NT);
  const int64_t segs = (p.K + kSeg - 1) / kSeg;
  const int64_t seg_lo = segs * part / split, seg_hi = segs * (part + 1) / split;
  const int64_t groups = p.K / GROUP;

  // rows past the last are computed as the last and not stored
  const int64_t r0 = min(block_row + rw * 16 + g, p.N - 1), r1 = min(block_row + rw * 16 + g + 8, p.N - 1);
  const uint8_t* w0 = p.packed + r0 * (p.K / 2);
  const uint8_t* w1 = p.packed + r1 * (p.K / 2);

  const int row_bytes = p.chunk * 2 + 64;  // of a token: 8 lanes of a read cover all banks
  const int part_bytes = row_bytes * tokens;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  const int chunk_segs = p.chunk / kSeg;
  for (int64_t c_lo = seg_lo; c_lo < seg_hi; c_lo += chunk_segs) {
    const int64_t c_hi = min(c_lo + chunk_segs, seg_hi);
    // x: eight columns at a time
    const int units = (int)(c_hi - c_lo) * (kSeg / 8);
    if (c_lo != seg_lo) __syncthreads();
    for (int i = threadIdx.x; i < units * tokens; i += kThreads) {
      const int m = i / units, u = i - m * units;
      const int64_t k0 = c_lo * kSeg + u * 8;
      float f[8];
      const T* xr = static_cast<const T*>(p.x) + (m0 + m) * p.ldx + k0;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = k0 + j < p.K ? elem::to_f(xr[j]) : 0.f;
      // of a segment's 16 units, lane t reads unit 4j + t at word j (transposed
      // words), or unit 4t + j (words as loaded); both at place 4j + t
      const int in_seg = u & 15;
      const int place = (u & ~15) | (GROUP < kSeg ? in_seg : ((in_seg & 3) << 2) | (in_seg >> 2));
      uint8_t* to = smem + m * row_bytes + place * 16;
      if constexpr (P == 1) {
        *reinterpret_cast<uint4*>(to) = order8<H>(f);
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          float r[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            r[j] = __uint_as_float(__float_as_uint(f[j]) & 0xFFFF0000u);  // 8 of the 24 bits, towards zero
            f[j] = f[j] == r[j] ? 0.f : f[j] - r[j];                      // exact; an infinity leaves 0
          }
          *reinterpret_cast<uint4*>(to + q * part_bytes) = order8<H>(r);
        }
      }
    }
    __syncthreads();

    for (int64_t s = c_lo + kw; s < c_hi; s += k_warps) {
      const int64_t k0 = s * kSeg;
      uint32_t a0[4] = {0, 0, 0, 0}, a1[4] = {0, 0, 0, 0};
      if (k0 + t * 32 < p.K) {
        const uint4 v0 = elem::ld_once16(w0 + k0 / 2 + t * 16), v1 = elem::ld_once16(w1 + k0 / 2 + t * 16);
        a0[0] = v0.x; a0[1] = v0.y; a0[2] = v0.z; a0[3] = v0.w;
        a1[0] = v1.x; a1[1] = v1.y; a1[2] = v1.z; a1[3] = v1.w;
      }
      if constexpr (GROUP < kSeg) {
        transpose4(a0, t);
        transpose4(a1, t);
      }
      float s0[GPS], s1[GPS];
      uint32_t z0[GPS], z1[GPS];
#pragma unroll
      for (int q = 0; q < GPS; ++q) {
        const int64_t grp = min(s * GPS + q, groups - 1);  // past the last: x is 0
        s0[q] = elem::ld_weight(p.scales, p.scale_dtype, r0 * groups + grp);
        s1[q] = elem::ld_weight(p.scales, p.scale_dtype, r1 * groups + grp);
        z0[q] = zero_pair<H>(p.zeros ? p.zeros[r0 * groups + grp] : 8);
        z1[q] = zero_pair<H>(p.zeros ? p.zeros[r1 * groups + grp] : 8);
      }
      const uint8_t* xs = smem + (s - c_lo) * (kSeg * 2) + t * 16;
#pragma unroll
      for (int q = 0; q < GPS; ++q) {
        float sum[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[n][i] = 0.f;
#pragma unroll
        for (int jj = 0; jj < 4 / GPS; ++jj) {
          const int j = q * (4 / GPS) + jj;
          uint32_t a[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            a[h][0] = weights<H>(a0[j], 2 * h, z0[q]);
            a[h][1] = weights<H>(a1[j], 2 * h, z1[q]);
            a[h][2] = weights<H>(a0[j], 2 * h + 1, z0[q]);
            a[h][3] = weights<H>(a1[j], 2 * h + 1, z1[q]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int m = n * 8 + g < tokens ? n * 8 + g : 0;  // columns past the last are not stored
#pragma unroll
            for (int o = 0; o < P; ++o) {
              const uint4 b = *reinterpret_cast<const uint4*>(xs + o * part_bytes + m * row_bytes + j * 64);
              mma<H>(sum[n], a[0], b.x, b.y);
              mma<H>(sum[n], a[1], b.z, b.w);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(s0[q], sum[n][0], acc[n][0]);
          acc[n][1] = fmaf(s0[q], sum[n][1], acc[n][1]);
          acc[n][2] = fmaf(s1[q], sum[n][2], acc[n][2]);
          acc[n][3] = fmaf(s1[q], sum[n][3], acc[n][3]);
        }
      }
    }
  }

  // sums of the column-warps, then of the cluster, each in its order
  constexpr int C = 8 * NT;
  const int rows = 16 * p.row_warps;
  float* sums = reinterpret_cast<float*>(smem);  // [k_warps][C][rows]
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float* to = sums + ((size_t)kw * C + n * 8 + 2 * t) * rows + rw * 16 + g;
    to[0] = acc[n][0];
    to[rows] = acc[n][1];
    to[8] = acc[n][2];
    to[rows + 8] = acc[n][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * tokens; i += kThreads) {
    float v = sums[i];
    for (int w = 1; w < k_warps; ++w) v += sums[w * C * rows + i];
    sums[i] = v;
  }
  if (split > 1) cluster.sync();
  else __syncthreads();
  for (int i = threadIdx.x + part * kThreads; i < rows * tokens; i += split * kThreads) {
    const int m = i / rows, r = i - m * rows;
    float v = 0.f;
    for (int q = 0; q < split; ++q) v += split > 1 ? cluster.map_shared_rank(sums, q)[i] : sums[i];
    const int64_t n = block_row + r;
    if (n < p.N) {
      if (p.bias) v += elem::to_f(static_cast<const T*>(p.bias)[n]);
      static_cast<T*>(p.y)[(m0 + m) * p.ldy + n] = elem::from_f<T>(v);
    }
  }
  if (split > 1) cluster.sync();  // the other CTAs read this one's sums
}

// Symmetric quantisation: s = max|w| / 7 of a group, rounded to the scales'
// type, q = 8 + w / s rounded to nearest even within [0, 15] (8 where s is 0).
// A warp per group.
template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const T* __restrict__ w, int64_t total, int group, uint8_t* __restrict__ packed, void* scales,
                int scale_dtype) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * kWarps) {
    const T* from = w + i * group;
    float top = 0.f;
    bool bad = false;
    for (int k = lane; k < group; k += 32) {
      const float v = elem::to_f(from[k]);
      top = fmaxf(top, fabsf(v));
      bad |= !(fabsf(v) < INFINITY);
    }
    top = warp_max(top);
    bad = __any_sync(0xffffffffu, bad);
    float s = bad ? __uint_as_float(0x7FC00000u) : top / 7.f;
    if (scale_dtype == KT_BF16) s = __bfloat162float(__float2bfloat16_rn(s));
    if (scale_dtype == KT_F16) s = __half2float(__float2half_rn(s));
    if (lane == 0) elem::st_weight(scales, scale_dtype, i, s);
    for (int k = 2 * lane; k < group; k += 64) {
      int q[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        q[j] = s > 0.f ? min(15, max(0, __float2int_rn(elem::to_f(from[k + j]) / s) + 8)) : 8;
      packed[(i * group + k) / 2] = (uint8_t)(q[0] | (q[1] << 4));
    }
  }
}

// ---------------------------------------------------------------- host
template <typename T, int GROUP, int NT>
inline int launch_shape(Args a, cudaStream_t st) {
  auto kern = w4_kernel<T, GROUP, NT>;
  const int64_t m_tiles = (a.M + 8 * NT - 1) / (8 * NT);
  const int64_t segs = (a.K + kSeg - 1) / kSeg;
  a.row_warps = 4;
  const int64_t blocks = (a.N + 16 * a.row_warps - 1) / (16 * a.row_warps);
  // split the columns while the device is not full and each warp keeps two segments
  int split = 1;
  while (split < kMaxCluster && blocks * m_tiles * split < 2 * sm_count() &&
         segs >= 2 * split * 2 * (kWarps / a.row_warps))
    split *= 2;
  const int tokens = (int)(a.M < 8 * NT ? a.M : 8 * NT);
  const int64_t own = (segs + split - 1) / split;
  const int64_t fit = (kStageBytes / (Mma<T>::parts * tokens) - 64) / (2 * kSeg);
  a.chunk = (int)((own < fit ? own : fit) * kSeg);
  const size_t stage = (size_t)Mma<T>::parts * tokens * (a.chunk * 2 + 64);
  const size_t sums = (size_t)(kWarps / a.row_warps) * 8 * NT * 16 * a.row_warps * sizeof(float);
  const size_t bytes = stage > sums ? stage : sums;
  int rc = ensure_smem((const void*)kern, bytes, "w4_linear: shared memory");
  if (rc != KT_OK) return rc;
  if (blocks * split > INT32_MAX || m_tiles > 65535)
    return fail(KT_ERR_UNSUPPORTED, "w4_linear: N=%lld or M=%lld too large", (long long)a.N, (long long)a.M);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * split), (unsigned)m_tiles);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a), "w4_linear launch");
}

template <typename T>
inline int launch_typed(const Args& a, int group, cudaStream_t st) {
  const bool one = a.M <= 8;
  if (group == 32) return one ? launch_shape<T, 32, 1>(a, st) : launch_shape<T, 32, 2>(a, st);
  if (group == 64) return one ? launch_shape<T, 64, 1>(a, st) : launch_shape<T, 64, 2>(a, st);
  return one ? launch_shape<T, 128, 1>(a, st) : launch_shape<T, 128, 2>(a, st);
}

inline int check_matrix(const char* what, int64_t N, int64_t K, int group, int dtype, int scale_dtype) {
  if (N < 0 || K < 0) return fail(KT_ERR_ARG, "%s: negative shape N=%lld K=%lld", what, (long long)N, (long long)K);
  if (elem::size_of(dtype) == 0) return fail(KT_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (elem::size_of(scale_dtype) == 0) return fail(KT_ERR_ARG, "%s: unknown scale dtype %d", what, scale_dtype);
  if (group != 32 && group != 64 && group != 128)
    return fail(KT_ERR_UNSUPPORTED, "%s: groups of 32, 64 or 128 columns, not %d", what, group);
  if (K % group) return fail(KT_ERR_ARG, "%s: K=%lld is not a multiple of the group %d", what, (long long)K, group);
  if (K > (int64_t)1 << 30) return fail(KT_ERR_UNSUPPORTED, "%s: K > 2^30", what);
  return KT_OK;
}

inline int linear(const Args& a, int group, int dtype, cudaStream_t st) {
  const int rc = check_matrix("w4_linear", a.N, a.K, group, dtype, a.scale_dtype);
  if (rc != KT_OK) return rc;
  if (a.M < 0) return fail(KT_ERR_ARG, "w4_linear: negative M=%lld", (long long)a.M);
  if (a.M == 0 || a.N == 0) return KT_OK;
  if (a.K == 0) return fail(KT_ERR_ARG, "w4_linear: K must be positive");
  if (!a.x || !a.packed || !a.scales || !a.y) return fail(KT_ERR_ARG, "w4_linear: null pointer");
  if (a.ldx < 0 || a.ldy < a.N) return fail(KT_ERR_ARG, "w4_linear: bad row strides");
  const int sz = elem::size_of(dtype);
  if (!aligned16(a.packed)) return fail(KT_ERR_ARG, "w4_linear: packed weights must be 16-byte aligned");
  if (!elem::aligned_to(a.x, sz) || !elem::aligned_to(a.y, sz) || !elem::aligned_to(a.bias, sz) ||
      !elem::aligned_to(a.scales, elem::size_of(a.scale_dtype)))
    return fail(KT_ERR_ARG, "w4_linear: a pointer is not aligned to its elements");
  if (dtype == KT_F32) return launch_typed<float>(a, group, st);
  if (dtype == KT_BF16) return launch_typed<__nv_bfloat16>(a, group, st);
  return launch_typed<__half>(a, group, st);
}

inline int quantize(const void* w, int64_t N, int64_t K, int group, int dtype, uint8_t* packed, void* scales,
                    int scale_dtype, cudaStream_t st) {
  const int rc = check_matrix("w4_quantize", N, K, group, dtype, scale_dtype);
  if (rc != KT_OK) return rc;
  const int64_t total = N * (K / group);
  if (total == 0) return KT_OK;
  if (!w || !packed || !scales) return fail(KT_ERR_ARG, "w4_quantize: null pointer");
  if (!elem::aligned_to(w, elem::size_of(dtype)) || !elem::aligned_to(scales, elem::size_of(scale_dtype)))
    return fail(KT_ERR_ARG, "w4_quantize: a pointer is not aligned to its elements");
  const int64_t need = (total + kWarps - 1) / kWarps, most = (int64_t)sm_count() * 8;
  const unsigned grid = (unsigned)(need < most ? need : most);
  if (dtype == KT_F32)
    quantize_kernel<<<grid, kThreads, 0, st>>>(static_cast<const float*>(w), total, group, packed, scales, scale_dtype);
  else if (dtype == KT_BF16)
    quantize_kernel<<<grid, kThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(w), total, group, packed, scales,
                                               scale_dtype);
  else
    quantize_kernel<<<grid, kThreads, 0, st>>>(static_cast<const __half*>(w), total, group, packed, scales,
                                               scale_dtype);
  return check_launch("w4_quantize");
}

}  // namespace w4
}  // namespace kt
