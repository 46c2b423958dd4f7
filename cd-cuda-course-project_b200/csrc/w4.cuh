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
// A warp takes 32 rows and segments of 128 columns, 2 KB of weights, which it
// copies with cp.async into a ring of its own, kStages deep: no warp waits for
// another, and the loads in flight do not depend on registers. A step of
// m16n8k16 may take any 16 columns if x has the same order, so a lane reads the
// words of one group (the 16-byte chunks of a row are swizzled: no bank is read
// twice) and uses each as it is. x is staged once per CTA in shared memory, in
// the order of the steps; each 16 bytes of it serve two tiles of 16 rows.
//
// A CTA stays and takes blocks of 32 x row_warps rows in turn; its other warps,
// and the CTAs of a cluster, split the columns (a cluster also holds an x that
// one CTA cannot), and their sums are added in a fixed order through
// (distributed) shared memory.
#pragma once
#include <cooperative_groups.h>

#include "elem.cuh"

namespace kt {
namespace w4 {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSeg = 128;          // columns of a warp step
constexpr int kRows = 32;          // rows of a warp step
constexpr int kStages = 3;         // of a warp's ring
constexpr int kItem = kRows * kSeg / 2;  // bytes of a step
constexpr int kMaxTokens = 16;     // of one CTA; more tokens take more CTAs
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxK = 131072;  // whose share of one fp32 token a cluster's CTA can hold

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
  int tokens;      // of a CTA
  int row_warps;   // warps of a CTA along N
  int64_t blocks;  // of 32 x row_warps rows
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

__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// Eight columns of a token, in the order in which the steps read them.
template <typename H>
__device__ __forceinline__ uint4 order8(const float (&f)[8]) {
  return make_uint4(elem::pack2<H>(f[0], f[4]), elem::pack2<H>(f[1], f[5]), elem::pack2<H>(f[2], f[6]),
                    elem::pack2<H>(f[3], f[7]));
}

// Shared memory of a CTA: x [parts][tokens][share of K + 32 columns], the warps'
// rings, the sums [column warps][8 NT tokens][rows].
__host__ __device__ constexpr size_t x_row_bytes(int64_t segs) {
  return (size_t)segs * kSeg * 2 + 64;  // 64: the eight lanes of a read cover all banks
}
constexpr size_t kRingBytes = (size_t)kWarps * kStages * kItem;
constexpr size_t sums_bytes(int nt) { return (size_t)kWarps * kRows * 8 * nt * sizeof(float); }

// GROUP: columns per scale. NT: blocks of 8 tokens of a CTA.
template <typename T, int GROUP, int NT>
__global__ void __launch_bounds__(kThreads, 2) w4_kernel(const Args p) {
  namespace cg = cooperative_groups;
  using H = typename Mma<T>::type;
  constexpr int P = Mma<T>::parts;
  constexpr int GPS = kSeg / GROUP;  // groups of a segment
  extern __shared__ __align__(128) uint8_t smem[];
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int k_warps = kWarps / p.row_warps, rw = warp / k_warps, kw = warp % k_warps;
  const int rows = kRows * p.row_warps;
  const int64_t m0 = (int64_t)blockIdx.y * p.tokens;
  const int tokens = (int)(p.M - m0 < p.tokens ? p.M - m0 : p.tokens);
  const int64_t segs = (p.K + kSeg - 1) / kSeg, most = (segs + split - 1) / split;
  const int64_t seg_lo = min(part * most, segs), seg_hi = min(seg_lo + most, segs);
  const int64_t groups = p.K / GROUP;
  const int64_t step = gridDim.x / split;  // blocks between two of this cluster

  const int row_bytes = (int)x_row_bytes(most);
  const int part_bytes = row_bytes * p.tokens;
  uint8_t* ring = smem + (size_t)part_bytes * P + (size_t)warp * kStages * kItem;
  float* sums = reinterpret_cast<float*>(smem + (size_t)part_bytes * P + kRingBytes);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const int swizzle = (g >> 1) & 3;

  // this warp's steps: its segments of a block, block after block
  int64_t f_block = blockIdx.x / split, f_seg = seg_lo + kw;
  int f_slot = 0;
  auto fetch = [&]() {
    while (f_block < p.blocks && f_seg >= seg_hi) {  // (once, unless this warp has no segment)
      f_block += step;
      f_seg = seg_lo + kw;
      if (f_seg >= seg_hi) f_block = p.blocks;
    }
    if (f_block < p.blocks) {
      const int64_t k0 = f_seg * kSeg + t * 32;
      const int bytes = k0 < p.K ? 16 : 0;  // 0: zeros are written
      const int64_t at = bytes ? k0 / 2 : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // rows past the last are computed as the last and not stored
        const int64_t r = min(f_block * rows + rw * kRows + g + 8 * i, p.N - 1);
        copy16(ring_at + f_slot * kItem + (g + 8 * i) * 64 + ((t ^ swizzle) * 16), p.packed + r * (p.K / 2) + at,
               bytes);
      }
      f_seg += k_warps;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    f_slot = f_slot + 1 == kStages ? 0 : f_slot + 1;
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  // x: eight columns at a time
  {
    const int units = (int)(seg_hi - seg_lo) * (kSeg / 8);
    const bool vec = sizeof(T) == 2 && elem::misalign<T>(p.x) == 0 && p.ldx % 8 == 0;
    for (int i = threadIdx.x; i < units * tokens; i += kThreads) {
      const int m = i / units, u = i - m * units;
      const int64_t k0 = seg_lo * kSeg + u * 8;
      float f[8];
      const T* xr = static_cast<const T*>(p.x) + (m0 + m) * p.ldx + k0;
      if (sizeof(T) == 2 && vec && k0 < p.K) {  // K is a multiple of 32
        if constexpr (sizeof(T) == 2) elem::unpack_vec<T>(*reinterpret_cast<const uint4*>(xr), f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = k0 < p.K ? elem::to_f(xr[j]) : 0.f;
      }
      uint8_t* to = smem + m * row_bytes + u * 16;
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
  }
  __syncthreads();

  int slot = 0;
  for (int64_t block = blockIdx.x / split; block < p.blocks; block += step) {
    float acc[2][NT][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
    int64_t grp_row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) grp_row[i] = min(block * rows + rw * kRows + g + 8 * i, p.N - 1) * groups;

    for (int64_t s = seg_lo + kw; s < seg_hi; s += k_warps) {
      float sc[4][GPS];
      uint32_t zr[4][GPS];
#pragma unroll
      for (int q = 0; q < GPS; ++q) {
        const int64_t grp = min(s * GPS + q, groups - 1);  // past the last: x is 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[i][q] = elem::ld_weight(p.scales, p.scale_dtype, grp_row[i] + grp);
          zr[i][q] = zero_pair<H>(p.zeros ? p.zeros[grp_row[i] + grp] : 8);
        }
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();  // the copies of all lanes have landed, and the slot before was read by all
      fetch();
      const uint8_t* xs = smem + (s - seg_lo) * (kSeg * 2) + t * 16;
      const uint8_t* ws = ring + slot * kItem + g * 64 + t * 4;
      slot = slot + 1 == kStages ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < GPS; ++q) {
        float sum[2][NT][4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[r][n][i] = 0.f;
#pragma unroll
        for (int jj = 0; jj < 4 / GPS; ++jj) {
          const int j = q * (4 / GPS) + jj;
          uint32_t a[2][2][4];  // [tile][step]
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(ws + r * 1024 + ((j ^ swizzle) * 16));
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(ws + r * 1024 + 512 + ((j ^ swizzle) * 16));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              a[r][h][0] = weights<H>(w0, 2 * h, zr[2 * r][q]);
              a[r][h][1] = weights<H>(w1, 2 * h, zr[2 * r + 1][q]);
              a[r][h][2] = weights<H>(w0, 2 * h + 1, zr[2 * r][q]);
              a[r][h][3] = weights<H>(w1, 2 * h + 1, zr[2 * r + 1][q]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int m = n * 8 + g < tokens ? n * 8 + g : 0;  // columns past the last are not stored
#pragma unroll
            for (int o = 0; o < P; ++o) {
              const uint4 b = *reinterpret_cast<const uint4*>(xs + o * part_bytes + m * row_bytes + j * 64);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                mma<H>(sum[r][n], a[r][0], b.x, b.y);
                mma<H>(sum[r][n], a[r][1], b.z, b.w);
              }
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[r][n][i] = fmaf(sc[2 * r + (i >> 1)][q], sum[r][n][i], acc[r][n][i]);
      }
    }

    // sums of the column warps, then of the cluster, each in its order
    constexpr int C = 8 * NT;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* to = sums + (size_t)(kw * C + n * 8 + 2 * t) * rows + rw * kRows + r * 16 + g;
        to[0] = acc[r][n][0];
        to[rows] = acc[r][n][1];
        to[8] = acc[r][n][2];
        to[rows + 8] = acc[r][n][3];
      }
    __syncthreads();
    auto store = [&](int i, float v) {
      const int m = i / rows;
      const int64_t n = block * rows + (i - m * rows);
      if (n < p.N) {
        if (p.bias) v += elem::to_f(static_cast<const T*>(p.bias)[n]);
        static_cast<T*>(p.y)[(m0 + m) * p.ldy + n] = elem::from_f<T>(v);
      }
    };
    for (int i = threadIdx.x; i < rows * tokens; i += kThreads) {
      float v = sums[i];
      for (int w = 1; w < k_warps; ++w) v += sums[w * C * rows + i];
      if (split > 1) sums[i] = v;
      else store(i, v);
    }
    if (split > 1) {
      cluster.sync();
      for (int i = threadIdx.x + part * kThreads; i < rows * tokens; i += split * kThreads) {
        float v = 0.f;
        for (int q = 0; q < split; ++q) v += cluster.map_shared_rank(sums, q)[i];
        store(i, v);
      }
      cluster.sync();  // the other CTAs read this one's sums
    } else {
      __syncthreads();
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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
  const int64_t segs = (a.K + kSeg - 1) / kSeg;
  const int sms = sm_count();
  auto bytes_for = [&](int split) {
    return (size_t)Mma<T>::parts * a.tokens * x_row_bytes((segs + split - 1) / split) + kRingBytes + sums_bytes(NT);
  };
  // as little of a cluster as lets two CTAs share an SM, or else fits at all
  constexpr size_t kTwo = 113 * 1024, kOne = 226 * 1024;
  int split = 1;
  while (split < kMaxCluster && bytes_for(split) > kTwo) split *= 2;
  while (split > 1 && bytes_for(split) > kTwo && bytes_for(split / 2) <= kOne) split /= 2;
  if (bytes_for(split) > kOne) return fail(KT_ERR_UNSUPPORTED, "w4_linear: K=%lld is too large", (long long)a.K);
  // more of it while the device is not full and every warp keeps two segments
  auto blocks_for = [&](int row_warps) { return (a.N + kRows * row_warps - 1) / (kRows * row_warps); };
  const int64_t m_tiles = (a.M + a.tokens - 1) / a.tokens;
  while (split < kMaxCluster && blocks_for(1) * split * m_tiles < sms && segs >= 2 * split * 2 * kWarps) split *= 2;
  const size_t bytes = bytes_for(split);
  const int64_t slots = (int64_t)sms * (bytes <= kTwo ? 2 : 1) / split;
  // rows of a block: many, unless fewer share the blocks out better
  a.row_warps = 1;
  double best = 0;
  for (int r = kWarps; r >= 1; r /= 2) {
    const int64_t blocks = blocks_for(r) * m_tiles, turns = (blocks + slots - 1) / slots;
    const double used = (double)blocks / (double)(turns * slots);
    if (used > best + 0.05) {
      best = used;
      a.row_warps = r;
    }
  }
  a.blocks = blocks_for(a.row_warps);
  const int64_t per_tile = slots / m_tiles > 0 ? slots / m_tiles : 1;
  const int64_t clusters = a.blocks < per_tile ? a.blocks : per_tile;
  if (m_tiles > 65535) return fail(KT_ERR_UNSUPPORTED, "w4_linear: M=%lld is too large", (long long)a.M);
  const int rc = ensure_smem((const void*)kern, bytes, "w4_linear: shared memory");
  if (rc != KT_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * split), (unsigned)m_tiles);
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
inline int launch_typed(Args a, int group, cudaStream_t st) {
  // tokens of a CTA: fewer where a cluster cannot hold the share of more
  a.tokens = (int)(a.M < kMaxTokens ? a.M : kMaxTokens);
  const int64_t segs = (a.K + kSeg - 1) / kSeg;
  while (a.tokens > 1 && Mma<T>::parts * a.tokens * x_row_bytes((segs + kMaxCluster - 1) / kMaxCluster) > 160 * 1024)
    a.tokens /= 2;
  const bool one = a.tokens <= 8;
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
  if (K > kMaxK) return fail(KT_ERR_UNSUPPORTED, "%s: K > %lld", what, (long long)kMaxK);
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
