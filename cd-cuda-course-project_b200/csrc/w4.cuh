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
// unpacked through shared memory): q - z is exact in 16 bits, and so are its
// products with x; the scale multiplies each group's fp32 sum. fp32 tokens are
// split exactly into three bf16 parts.
//
// Unpacking takes most of the instructions, so it costs 9 for 8 weights: one
// mask for each pair of nibbles (bits 0-3 and 4-7 of both halves of a word, then
// the same of the word shifted by 8) and one packed multiply-add. In fp16 the
// nibble is or-ed into the mantissa of 1024, which makes it 1024 + q or
// 1024 + 16 q; a bf16 of nothing but a nibble in its low 8 bits is q 2^-133 or
// q 2^-129 (its subnormals and first binade are one linear range), which a power
// of two brings to (q - z) / 64; the 64 comes back when the sums are done.
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
  int tokens;      // of a CTA
  int row_warps;   // warps of a CTA along N
  int64_t blocks;  // of 32 x row_warps rows
  bool whole_groups;  // a segment's scales (and zeros) can be loaded at once
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

// d = a b (+ d)
template <typename H>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool add) {
  const float c0 = add ? d[0] : 0.f, c1 = add ? d[1] : 0.f, c2 = add ? d[2] : 0.f, c3 = add ? d[3] : 0.f;
  if constexpr (std::is_same<H, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// What a group's zero and scale become for the unpacking below.
template <typename H>
struct Unpack;
template <>
struct Unpack<__half> {
  static constexpr float scale = 1.f;
  uint32_t low, high;  // pairs of 1024 + z, and of -(64 + z)
  __device__ __forceinline__ explicit Unpack(uint32_t zero)
      : low(0x64006400u + 0x00010001u * zero), high(0xD400D400u + 0x00100010u * zero) {}
  // nibbles at bits 0-3 and 16-19 / at bits 4-7 and 20-23 of a word, minus z
  __device__ __forceinline__ uint32_t at0(uint32_t w) const {
    const uint32_t q = (w & 0x000F000Fu) | 0x64006400u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&q), *reinterpret_cast<const __half2*>(&low));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ uint32_t at4(uint32_t w) const {
    const uint32_t q = (w & 0x00F000F0u) | 0x64006400u, s = 0x2C002C00u;  // 1/16
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&q), *reinterpret_cast<const __half2*>(&s),
                              *reinterpret_cast<const __half2*>(&high));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Unpack<__nv_bfloat16> {
  static constexpr float scale = 64.f;
  uint32_t minus;  // pair of -z / 64
  __device__ __forceinline__ explicit Unpack(uint32_t zero) {
    const __nv_bfloat162 v = __float2bfloat162_rn((float)zero * -0.015625f);
    minus = *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ static uint32_t fma(uint32_t q, uint32_t power, uint32_t minus) {
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&q),
                                     *reinterpret_cast<const __nv_bfloat162*>(&power),
                                     *reinterpret_cast<const __nv_bfloat162*>(&minus));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ uint32_t at0(uint32_t w) const { return fma(w & 0x000F000Fu, 0x7F007F00u, minus); }
  __device__ __forceinline__ uint32_t at4(uint32_t w) const { return fma(w & 0x00F000F0u, 0x7D007D00u, minus); }
};

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

// The scales and zeros of a lane's four rows for a segment, as loaded.
template <typename S, int GPS>
struct GroupWords {
  static constexpr int W = (GPS * (int)sizeof(S) + 3) / 4;
  uint32_t s[4][W];
  uint32_t z[4];  // a byte per group
  __device__ __forceinline__ float scale(int row, int q) const {
    if constexpr (sizeof(S) == 4) {
      return __uint_as_float(s[row][q]);
    } else {
      const float2 v = elem::unpack2<S>(s[row][q / 2]);
      return q & 1 ? v.y : v.x;
    }
  }
  __device__ __forceinline__ uint32_t zero(int row, int q) const { return (z[row] >> (8 * q)) & 255u; }
};

// GROUP: columns per scale. NT: blocks of 8 tokens of a CTA. S: type of the scales.
template <typename T, typename S, int GROUP, int NT>
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
  const uint8_t* f_rows;  // the first of this lane's rows of the block, at its columns
  int f_more[4];          // bytes from there to each of the four
  auto set_rows = [&]() {
    // rows past the last are computed as the last and not stored
    const int64_t r0 = f_block * rows + rw * kRows + g;
    f_rows = p.packed + min(r0, p.N - 1) * (p.K / 2) + t * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) f_more[i] = (int)((min(r0 + 8 * i, p.N - 1) - min(r0, p.N - 1)) * (p.K / 2));
  };
  set_rows();
  if (f_seg >= seg_hi) f_block = p.blocks;  // no segment for this warp
  auto fetch = [&]() {
    if (f_block < p.blocks) {
      const bool in = f_seg * kSeg + t * 32 < p.K;
      const uint8_t* at = in ? f_rows + f_seg * (kSeg / 2) : p.packed;  // size 0: zeros are written
      const uint32_t to = ring_at + f_slot * kItem + g * 64 + ((t ^ swizzle) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) copy16(to + i * 512, at + (in ? f_more[i] : 0), in ? 16 : 0);
      f_seg += k_warps;
      if (f_seg >= seg_hi) {
        f_seg = seg_lo + kw;
        f_block += step;
        if (f_block < p.blocks) set_rows();
      }
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
    const int64_t row0 = block * rows + rw * kRows + g;
    const S* scales = static_cast<const S*>(p.scales) + min(row0, p.N - 1) * groups;
    const uint8_t* zeros = p.zeros + (p.zeros ? min(row0, p.N - 1) * groups : 0);
    int more[4];  // groups from the first of the four rows to each
#pragma unroll
    for (int i = 0; i < 4; ++i) more[i] = (int)((min(row0 + 8 * i, p.N - 1) - min(row0, p.N - 1)) * groups);
    GroupWords<S, GPS> words;
    auto load_groups = [&](int64_t seg) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const S* at = scales + more[i] + seg * GPS;
        if (GPS == 1 || p.whole_groups) {  // a segment's groups in one load
          if constexpr (words.W == 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(at));
            words.s[i][0] = v.x; words.s[i][1] = v.y; words.s[i][2] = v.z; words.s[i][3] = v.w;
          } else if constexpr (words.W == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
            words.s[i][0] = v.x; words.s[i][1] = v.y;
          } else if constexpr (GPS * sizeof(S) == 4) {
            words.s[i][0] = __ldg(reinterpret_cast<const uint32_t*>(at));
          } else {
            words.s[i][0] = __ldg(reinterpret_cast<const uint16_t*>(at));
          }
          if (p.zeros) {
            const uint8_t* z = zeros + more[i] + seg * GPS;
            if constexpr (GPS == 4) words.z[i] = __ldg(reinterpret_cast<const uint32_t*>(z));
            else if constexpr (GPS == 2) words.z[i] = __ldg(reinterpret_cast<const uint16_t*>(z));
            else words.z[i] = __ldg(z);
          }
        } else {
#pragma unroll
          for (int q = 0; q < words.W; ++q) words.s[i][q] = 0;
          words.z[i] = 0;
#pragma unroll
          for (int q = 0; q < GPS; ++q) {
            const int64_t in = min(seg * GPS + q, groups - 1) - seg * GPS;  // past the last: x is 0
            if constexpr (sizeof(S) == 4) words.s[i][q] = __ldg(reinterpret_cast<const uint32_t*>(at) + in);
            else words.s[i][q / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at) + in) << (16 * (q & 1));
            if (p.zeros) words.z[i] |= (uint32_t)__ldg(zeros + more[i] + seg * GPS + in) << (8 * q);
          }
        }
        if (!p.zeros) words.z[i] = 0x08080808u;
      }
    };
    if (seg_lo + kw < seg_hi) load_groups(seg_lo + kw);

    for (int64_t s = seg_lo + kw; s < seg_hi; s += k_warps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();  // the copies of all lanes have landed, and the slot before was read by all
      fetch();
      const GroupWords<S, GPS> cur = words;
      if (s + k_warps < seg_hi) load_groups(s + k_warps);
      const uint8_t* xs = smem + (s - seg_lo) * (kSeg * 2) + t * 16;
      const uint8_t* ws = ring + slot * kItem + g * 64 + t * 4;
      slot = slot + 1 == kStages ? 0 : slot + 1;
#pragma unroll
      for (int q = 0; q < GPS; ++q) {
        float sum[2][NT][4];
        const Unpack<H> u0(cur.zero(0, q)), u1(cur.zero(1, q)), u2(cur.zero(2, q)), u3(cur.zero(3, q));
#pragma unroll
        for (int jj = 0; jj < 4 / GPS; ++jj) {
          const int j = q * (4 / GPS) + jj;
          uint32_t a[2][2][4];  // [tile][step]
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t w0 = *reinterpret_cast<const uint32_t*>(ws + r * 1024 + ((j ^ swizzle) * 16));
            uint32_t w1 = *reinterpret_cast<const uint32_t*>(ws + r * 1024 + 512 + ((j ^ swizzle) * 16));
            const Unpack<H>&v0 = r ? u2 : u0, &v1 = r ? u3 : u1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              a[r][h][0] = v0.at0(w0);
              a[r][h][1] = v1.at0(w1);
              a[r][h][2] = v0.at4(w0);
              a[r][h][3] = v1.at4(w1);
              w0 >>= 8;
              w1 >>= 8;
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
                mma<H>(sum[r][n], a[r][0], b.x, b.y, jj > 0 || o > 0);
                mma<H>(sum[r][n], a[r][1], b.z, b.w, true);
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
              acc[r][n][i] = fmaf(cur.scale(2 * r + (i >> 1), q), sum[r][n][i], acc[r][n][i]);
      }
    }

    // sums of the column warps, then of the cluster, each in its order
    constexpr int C = 8 * NT;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* to = sums + (size_t)(kw * C + n * 8 + 2 * t) * rows + rw * kRows + r * 16 + g;
        to[0] = acc[r][n][0] * Unpack<H>::scale;
        to[rows] = acc[r][n][1] * Unpack<H>::scale;
        to[8] = acc[r][n][2] * Unpack<H>::scale;
        to[rows + 8] = acc[r][n][3] * Unpack<H>::scale;
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
template <typename T, typename S, int GROUP, int NT>
inline int launch_shape(Args a, cudaStream_t st) {
  auto kern = w4_kernel<T, S, GROUP, NT>;
  constexpr int GPS = kSeg / GROUP;
  a.whole_groups = a.K % kSeg == 0 && elem::aligned_to(a.scales, GPS * (int)sizeof(S)) &&
                   elem::aligned_to(a.zeros, GPS);
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

template <typename T, typename S>
inline int launch_typed(Args a, int group, cudaStream_t st) {
  // tokens of a CTA: fewer where a cluster cannot hold the share of more
  a.tokens = (int)(a.M < kMaxTokens ? a.M : kMaxTokens);
  const int64_t segs = (a.K + kSeg - 1) / kSeg;
  while (a.tokens > 1 && Mma<T>::parts * a.tokens * x_row_bytes((segs + kMaxCluster - 1) / kMaxCluster) > 160 * 1024)
    a.tokens /= 2;
  const bool one = a.tokens <= 8;
  if (group == 32) return one ? launch_shape<T, S, 32, 1>(a, st) : launch_shape<T, S, 32, 2>(a, st);
  if (group == 64) return one ? launch_shape<T, S, 64, 1>(a, st) : launch_shape<T, S, 64, 2>(a, st);
  return one ? launch_shape<T, S, 128, 1>(a, st) : launch_shape<T, S, 128, 2>(a, st);
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

inline int linear(const Args& a, int group, int dtype, int scale_dtype, cudaStream_t st) {
  const int rc = check_matrix("w4_linear", a.N, a.K, group, dtype, scale_dtype);
  if (rc != KT_OK) return rc;
  if (scale_dtype != KT_F32 && scale_dtype != dtype)
    return fail(KT_ERR_ARG, "w4_linear: scales are fp32 or of the tokens' type");
  if (a.M < 0) return fail(KT_ERR_ARG, "w4_linear: negative M=%lld", (long long)a.M);
  if (a.M == 0 || a.N == 0) return KT_OK;
  if (a.K == 0) return fail(KT_ERR_ARG, "w4_linear: K must be positive");
  if (!a.x || !a.packed || !a.scales || !a.y) return fail(KT_ERR_ARG, "w4_linear: null pointer");
  if (a.ldx < 0 || a.ldy < a.N) return fail(KT_ERR_ARG, "w4_linear: bad row strides");
  const int sz = elem::size_of(dtype);
  if (!aligned16(a.packed)) return fail(KT_ERR_ARG, "w4_linear: packed weights must be 16-byte aligned");
  if (!elem::aligned_to(a.x, sz) || !elem::aligned_to(a.y, sz) || !elem::aligned_to(a.bias, sz) ||
      !elem::aligned_to(a.scales, elem::size_of(scale_dtype)))
    return fail(KT_ERR_ARG, "w4_linear: a pointer is not aligned to its elements");
  const bool f32 = scale_dtype == KT_F32;
  if (dtype == KT_F32) return launch_typed<float, float>(a, group, st);
  if (dtype == KT_BF16) return f32 ? launch_typed<__nv_bfloat16, float>(a, group, st)
                                   : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, group, st);
  return f32 ? launch_typed<__half, float>(a, group, st) : launch_typed<__half, __half>(a, group, st);
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
