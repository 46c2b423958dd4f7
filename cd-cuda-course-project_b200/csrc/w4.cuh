// w4.cuh — products of a few tokens with a matrix of 4-bit weights:
//   y[m][n] = bias[n] + sum over groups G of s[n][G] sum over k in G of x[m][k] (q[n][k] - z[n][G])
// q in 0..15, two to a byte (even k in the low half), G of 32, 64 or 128
// columns, z = 8 where no zeros are given.
//
// Bound by memory: the weights are read once, N K / 2 bytes. At 6.5 TB/s that
// is 13 10^12 weights a second, which leaves 2.6 lane instructions for each;
// fp32 multiply-adds per token would exceed that from the second token on. So the
// sums run on the tensor cores (mma.sync m16n8k16: 16 weight rows by 8 tokens,
// fp32 accumulation, the weights unpacked straight into its operand registers; a
// tcgen05 tile would take them from tensor memory, 128 rows at a time, through a
// store and a wait for each group, which was not tried): q - z is exact in 16 bits,
// and so are its products with x; the scale multiplies each group's fp32 sum. fp32
// tokens are split into three bf16 parts: exactly from 2^-110 on, where the last of
// their 24 bits is at least bf16's least number 2^-133, and to less than 2^-133 below.
//
// Unpacking takes most of the instructions, so it costs 9 for 8 weights: one
// mask for each pair of nibbles (bits 0-3 and 4-7 of both halves of a word, then
// the same of the word shifted by 8) and one packed multiply-add. A 16-bit float
// of nothing but a nibble in its low 8 bits is q 2^-133 or q 2^-129 in bf16
// (whose subnormals and first binade are one linear range), q 2^-24 or q 2^-20
// in fp16; a power of two and -z make it (q - z) / 64 or / 512, exactly, and
// that factor comes back when the sums are done.
//
// A warp takes 32 rows and segments of 128 columns, 2 KB of weights, which one
// TMA load brings into a ring of its own, 2 to 4 deep: no warp waits for
// another, and the loads in flight cost neither registers nor address
// arithmetic. A step of m16n8k16 may take any 16 columns if x has the same
// order, so a lane reads the words of one group (TMA's 64-byte swizzle: no bank
// is read twice) and uses each as it is. x is staged once per CTA in shared
// memory, in the order of the steps; each 16 bytes of it serve two tiles of 16
// rows.
//
// One CTA of 16 warps per SM holds x. Its warps form groups of k_warps that split
// the columns of 32 rows; groups take their rows in turn, each at its own pace,
// and add their sums in a fixed order through shared memory. Where x does not
// fit one CTA, or rows are few, a cluster splits the columns as well: its CTAs go
// row by row together, and add their sums through distributed shared memory one
// turn late (a warp that has left its sums arrives at the cluster's barrier, goes
// on with the next rows, and waits there before it adds the sums before).
//
// Measured on a B200, 131072x8192: one token in bf16, groups of 128, 109 us
// (5.1 TB/s, 78 % of measured copy bandwidth); 8 tokens in fp16, groups of 64 with
// zeros, 142 us (4.2 TB/s; issue slots 66 % busy, the ALU pipe 52 %); 16 tokens in
// bf16 184 us. 4096x4096, one token: 5.5 us. 16 fp32 tokens, 32768x8192: 104 us; of
// its units the tensor pipe is the busiest (53 %, on 128 of 148 SMs; three products
// per weight), and warps wait for it most.
#pragma once
#include <cooperative_groups.h>

#include "elem.cuh"
#include "sm100.cuh"

namespace kt {
namespace w4 {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kSeg = 128;          // columns of a warp step
constexpr int kRows = 32;          // rows of a warp step
constexpr int kMinStages = 2, kMaxStages = 4;  // of a warp's ring
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
  int tokens;   // of a CTA
  int k_warps;  // warps that split the columns of 32 rows
  int units;    // of 32 rows
  int stages;
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

// Pairs of weights of one type H: `power` brings a nibble at bits 0-3 (low) and
// 4-7 (high) of both halves of a word, read as H, to q / scale.
template <typename H>
struct Nibbles;
template <>
struct Nibbles<__nv_bfloat16> {
  static constexpr float scale = 64.f;                               // 2^-133 2^127
  static constexpr uint32_t low = 0x7F007F00u, high = 0x7D007D00u;  // 2^127, 2^123
  __device__ __forceinline__ static uint32_t minus(uint32_t zero) {  // pair of -zero / scale
    return fma(zero * 0x00010001u, low ^ 0x80008000u, 0x80008000u);  // (+ -0)
  }
  __device__ __forceinline__ static uint32_t fma(uint32_t q, uint32_t power, uint32_t minus) {
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&q),
                                     *reinterpret_cast<const __nv_bfloat162*>(&power),
                                     *reinterpret_cast<const __nv_bfloat162*>(&minus));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Nibbles<__half> {
  static constexpr float scale = 512.f;                              // 2^-24 2^15
  static constexpr uint32_t low = 0x78007800u, high = 0x68006800u;  // 2^15, 2^11
  __device__ __forceinline__ static uint32_t minus(uint32_t zero) {
    return fma(zero * 0x00010001u, low ^ 0x80008000u, 0x80008000u);
  }
  __device__ __forceinline__ static uint32_t fma(uint32_t q, uint32_t power, uint32_t minus) {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&q), *reinterpret_cast<const __half2*>(&power),
                              *reinterpret_cast<const __half2*>(&minus));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// Eight columns of a token, in the order in which the steps read them.
template <typename H>
__device__ __forceinline__ uint4 order8(const float (&f)[8]) {
  return make_uint4(elem::pack2<H>(f[0], f[4]), elem::pack2<H>(f[1], f[5]), elem::pack2<H>(f[2], f[6]),
                    elem::pack2<H>(f[3], f[7]));
}

// Shared memory of a CTA: the warps' rings and their barriers, the sums
// [1 or 2 turns][warps][8 NT tokens][rows], x [parts][tokens][share of K + 32
// columns].
__host__ __device__ constexpr size_t x_row_bytes(int64_t segs) {
  return (size_t)segs * kSeg * 2 + 64;  // 64: the eight lanes of a read cover all banks
}
constexpr size_t kBarBytes = (size_t)kWarps * kMaxStages * 8;
__host__ __device__ constexpr size_t sums_bytes(int nt) { return (size_t)kWarps * kRows * 8 * nt * sizeof(float); }
constexpr size_t kAlign = 1024;  // of the rings, for the swizzle

// How scales and zeros are read: a segment's in one load (kWhole: no zeros), or,
// where a row's do not start on a boundary of such loads, one group by each of the
// four lanes of a row, which exchange them (16 tokens, 131072x8160, groups of 32
// with zeros: 324 us, and 587 with each lane loading all).
enum Groups { kWhole, kWholeZeros, kSingle };

// The scales and zeros of a lane's four rows for a segment, as loaded.
template <typename S, int GPS, Groups MODE>
struct GroupWords {
  static constexpr int W = MODE == kSingle ? 1 : (GPS * (int)sizeof(S) + 3) / 4;
  uint32_t s[4][W];
  uint32_t z[4];  // a byte per group (kSingle: of this lane's group, above a scale of 16 bits)

  __device__ __forceinline__ void load(const S* scales, const uint8_t* zeros, const uint32_t (&more)[4], int first,
                                       int groups, int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = more[i] + (uint32_t)first;
      if constexpr (MODE != kSingle) {
        const S* from = scales + at;
        if constexpr (W == 4) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(from));
          s[i][0] = v.x; s[i][1] = v.y; s[i][2] = v.z; s[i][3] = v.w;
        } else if constexpr (W == 2) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(from));
          s[i][0] = v.x; s[i][1] = v.y;
        } else if constexpr (GPS * sizeof(S) == 4) {
          s[i][0] = __ldg(reinterpret_cast<const uint32_t*>(from));
        } else {
          s[i][0] = __ldg(reinterpret_cast<const uint16_t*>(from));
        }
        if constexpr (MODE == kWholeZeros) {
          if constexpr (GPS == 4) z[i] = __ldg(reinterpret_cast<const uint32_t*>(zeros + at));
          else if constexpr (GPS == 2) z[i] = __ldg(reinterpret_cast<const uint16_t*>(zeros + at));
          else z[i] = __ldg(zeros + at);
        }
      } else {
        const int q = t % GPS;
        s[i][0] = 0;  // past the last: x is 0
        z[i] = 8;
        if (first + q < groups) {
          if (zeros) z[i] = __ldg(zeros + at + q);
          if constexpr (sizeof(S) == 4) s[i][0] = __ldg(reinterpret_cast<const uint32_t*>(scales) + at + q);
          else s[i][0] = __ldg(reinterpret_cast<const uint16_t*>(scales) + at + q) | z[i] << 16;
        }
      }
    }
  }
  // kSingle: the scale and the zero of group q, from the lane that has them
  __device__ __forceinline__ void exchange(int row, int q, float* scale, uint32_t* zero) const {
    const int from = ((int)threadIdx.x & 28) | q;
    const uint32_t w = __shfl_sync(0xffffffffu, s[row][0], from);
    if constexpr (sizeof(S) == 4) {
      *scale = __uint_as_float(w);
      *zero = __shfl_sync(0xffffffffu, z[row], from);
    } else {
      *scale = elem::unpack2<S>(w).x;
      *zero = w >> 16;
    }
  }
  __device__ __forceinline__ float scale(int row, int q) const {
    if constexpr (sizeof(S) == 4) {
      return __uint_as_float(s[row][q]);
    } else {
      const float2 v = elem::unpack2<S>(s[row][q / 2]);
      return q & 1 ? v.y : v.x;
    }
  }
  __device__ __forceinline__ uint32_t zero(int row, int q) const {
    if constexpr (MODE == kWhole) return 8;
    else if constexpr (GPS == 1) return z[row] & 255u;
    else return __byte_perm(z[row], 0, 0x4440 + q);
  }
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// GROUP: columns per scale. NT: blocks of 8 tokens of a CTA.
template <typename T, int GROUP, int NT, Groups MODE>
__global__ void __launch_bounds__(kThreads, 1) w4_kernel(const Args p, const __grid_constant__ CUtensorMap map) {
  namespace cg = cooperative_groups;
  using namespace sm100;
  using H = typename Mma<T>::type;
  constexpr int P = Mma<T>::parts;
  constexpr int GPS = kSeg / GROUP;  // groups of a segment
  constexpr int C = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((kAlign - (smem_u32(smem_raw) & (kAlign - 1))) & (kAlign - 1));
  const cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  const int g = lane >> 2, t = lane & 3;
  const int k_warps = p.k_warps, rw = warp / k_warps, kw = warp % k_warps;
  const int64_t m0 = (int64_t)blockIdx.y * p.tokens;
  const int tokens = (int)(p.M - m0 < p.tokens ? p.M - m0 : p.tokens);
  const int segs = (int)((p.K + kSeg - 1) / kSeg), most = (segs + split - 1) / split;
  const int seg_lo = min(part * most, segs), seg_hi = min(seg_lo + most, segs);
  const int64_t groups = p.K / GROUP;
  // units of 32 rows: this group's first, and how many are between two of its turns
  const int first = (int)(blockIdx.x / split) * (kWarps / k_warps) + rw;
  const int step = (int)(gridDim.x / split) * (kWarps / k_warps);

  const int stages = p.stages;
  const int row_bytes = (int)x_row_bytes(most);
  const int part_bytes = row_bytes * p.tokens;
  const uint32_t ring_bytes = (uint32_t)(kWarps * stages * kItem);
  const uint8_t* ring = smem + warp * stages * kItem;
  const uint32_t bars = smem_u32(smem) + ring_bytes + warp * kMaxStages * 8;
  float* sums = reinterpret_cast<float*>(smem + ring_bytes + kBarBytes);
  uint8_t* xsm = smem + ring_bytes + kBarBytes + sums_bytes(NT) * (split > 1 ? 2 : 1);
  const int swizzle = (g >> 1) & 3;

  // this warp's steps: its segments of a unit, unit after unit
  int f_unit = first, f_seg = seg_lo + kw, f_slot = 0;
  if (f_seg >= seg_hi) f_unit = p.units;  // none
  auto fetch = [&]() {  // rows and columns past the last are zeros
    if (f_unit >= p.units) return;
    if (lane == 0) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the slot's reads before TMA's write
      mbar_arrive_expect_tx(bars + 8 * f_slot, kItem);
      tma_load_2d(smem_u32(ring) + f_slot * kItem, &map, f_seg * (kSeg / 2), f_unit * kRows, bars + 8 * f_slot);
    }
    f_slot = f_slot + 1 == stages ? 0 : f_slot + 1;
    f_seg += k_warps;
    if (f_seg >= seg_hi) {
      f_seg = seg_lo + kw;
      f_unit += step;
    }
  };
  if (lane == 0) {
    tma_prefetch_desc(&map);
    for (int i = 0; i < stages; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  for (int i = 0; i < stages - 1; ++i) fetch();

  // x: eight columns at a time
  {
    const int units = (seg_hi - seg_lo) * (kSeg / 8);
    const bool vec = sizeof(T) == 2 && elem::misalign<T>(p.x) == 0 && p.ldx % 8 == 0;
    for (int i = threadIdx.x; i < units * tokens; i += kThreads) {
      const int m = i / units, u = i - m * units;
      const int64_t k0 = (int64_t)seg_lo * kSeg + u * 8;
      float f[8];
      const T* xr = static_cast<const T*>(p.x) + (m0 + m) * p.ldx + k0;
      if (sizeof(T) == 2 && vec && k0 < p.K) {  // K is a multiple of 32
        if constexpr (sizeof(T) == 2) elem::unpack_vec<T>(*reinterpret_cast<const uint4*>(xr), f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = k0 < p.K ? elem::to_f(xr[j]) : 0.f;
      }
      // of a segment's 16 units, lane t reads unit 4j + t at word j (4t + j: CHUNK); both at place 4j + t
      const int place = GROUP < kSeg ? u : (u & ~15) | ((u & 3) << 2) | ((u >> 2) & 3);
      uint8_t* to = xsm + m * row_bytes + place * 16;
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

  // adds the sums of `unit`, which its warps (in all CTAs of the cluster) have
  // left in turn `turn`, and stores the rows
  auto finish = [&](int unit, int turn) {
    const float* from = sums + (turn * kWarps + rw * k_warps) * (kRows * C);
    const int threads = k_warps * 32;  // of this CTA that share the work
    for (int i = (part * k_warps + kw) * 32 + lane; i < kRows * tokens; i += split * threads) {
      const int m = i / kRows;
      const int64_t n = (int64_t)unit * kRows + i % kRows;
      float v = 0.f;
      for (int q = 0; q < split; ++q) {
        const float* at = split > 1 ? cluster.map_shared_rank(from, q) : from;
        for (int w = 0; w < k_warps; ++w) v += at[w * (kRows * C) + i];
      }
      if (n < p.N) {
        v *= Nibbles<H>::scale;
        if (p.bias) v += elem::to_f(static_cast<const T*>(p.bias)[n]);
        static_cast<T*>(p.y)[(m0 + m) * p.ldy + n] = elem::from_f<T>(v);
      }
    }
  };
  auto group_sync = [&]() {
    if (k_warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + rw), "r"(k_warps * 32) : "memory");
  };

  const uint8_t* x_rows[NT];  // this lane's token of each block of 8; those past the last are not stored
#pragma unroll
  for (int n = 0; n < NT; ++n) x_rows[n] = xsm + (n * 8 + g < tokens ? n * 8 + g : 0) * row_bytes + t * 16;
  // this lane's words of its first row in a slot: word t of each 16-byte chunk j or,
  // where a group is the whole segment, chunk t (one load instead of four)
  constexpr bool CHUNK = GROUP == kSeg;
  const uint8_t* word_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) word_at[j] = ring + g * 64 + ((CHUNK ? t : j) ^ swizzle) * 16 + (CHUNK ? j : t) * 4;
  int slot = 0, turn = 0, before = -1;
  uint32_t parity = 0;
  bool ok = true;
  // in a cluster all groups make the same number of turns, some without rows
  for (int unit = first; split > 1 ? unit - first < p.units : unit < p.units; unit += step, turn ^= 1) {
    float acc[2][NT][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
    const int64_t row0 = (int64_t)unit * kRows;
    const T* scales = static_cast<const T*>(p.scales) + row0 * groups;
    const uint8_t* zeros = p.zeros + (p.zeros ? row0 * groups : 0);
    uint32_t more[4];  // groups from the unit's first row to this lane's four
#pragma unroll
    for (int i = 0; i < 4; ++i) more[i] = (uint32_t)((min(row0 + g + 8 * i, p.N - 1) - row0) * groups);
    const int seg_end = unit < p.units ? seg_hi : 0;
    GroupWords<T, GPS, MODE> words;
    if (seg_lo + kw < seg_end) words.load(scales, zeros, more, (seg_lo + kw) * GPS, (int)groups, t);

    // (unrolled: two segments share their address arithmetic, which takes 10 % less time)
#pragma unroll 2
    for (int s = seg_lo + kw; s < seg_end; s += k_warps) {
      if (ok && !__all_sync(0xffffffffu, mbar_wait(bars + 8 * slot, parity))) {
        // gave up: load nothing more, and wait (as long again) for what is in flight
        ok = false;
        f_unit = p.units;
        raise_device_error(DEV_MBAR_TIMEOUT);
        for (int i = 0; i < stages - 1; ++i) {
          const int at = (slot + i) % stages;
          (void)mbar_wait(bars + 8 * at, slot + i < stages ? parity : parity ^ 1);
        }
      }
      __syncwarp();  // all lanes have read the slot before this one, which fetch() fills
      fetch();
      const GroupWords<T, GPS, MODE> cur = words;
      if (s + k_warps < seg_hi) words.load(scales, zeros, more, (s + k_warps) * GPS, (int)groups, t);
      const int x_at = (s - seg_lo) * (kSeg * 2);
      const int slot_at = slot * kItem;
      uint4 chunk[4];  // [row]
      if constexpr (CHUNK) {
#pragma unroll
        for (int i = 0; i < 4; ++i) chunk[i] = *reinterpret_cast<const uint4*>(word_at[0] + slot_at + i * 512);
      }
      auto word = [&](int row, int j) -> uint32_t {
        if constexpr (CHUNK) {
          const uint4& c = chunk[row];
          return j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w;
        } else {
          return *reinterpret_cast<const uint32_t*>(word_at[j] + slot_at + row * 512);
        }
      };
      if (++slot == stages) {
        slot = 0;
        parity ^= 1;
      }
#pragma unroll
      for (int q = 0; q < GPS; ++q) {
        float sum[2][NT][4];
        uint32_t minus[4];
        float scale[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t zero;
          if constexpr (MODE == kSingle) {
            cur.exchange(i, q, &scale[i], &zero);
          } else {
            scale[i] = cur.scale(i, q);
            zero = cur.zero(i, q);
          }
          minus[i] = Nibbles<H>::minus(zero);
        }
#pragma unroll
        for (int jj = 0; jj < 4 / GPS; ++jj) {
          const int j = q * (4 / GPS) + jj;
          uint32_t a[2][2][4];  // [tile][step]
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t w0 = word(2 * r, j), w1 = word(2 * r + 1, j);
            const uint32_t z0 = minus[2 * r], z1 = minus[2 * r + 1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              a[r][h][0] = Nibbles<H>::fma(w0 & 0x000F000Fu, Nibbles<H>::low, z0);
              a[r][h][1] = Nibbles<H>::fma(w1 & 0x000F000Fu, Nibbles<H>::low, z1);
              a[r][h][2] = Nibbles<H>::fma(w0 & 0x00F000F0u, Nibbles<H>::high, z0);
              a[r][h][3] = Nibbles<H>::fma(w1 & 0x00F000F0u, Nibbles<H>::high, z1);
              w0 >>= 8;
              w1 >>= 8;
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int o = 0; o < P; ++o) {
              const uint4 b = *reinterpret_cast<const uint4*>(x_rows[n] + o * part_bytes + x_at + j * 64);
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
              acc[r][n][i] = fmaf(scale[2 * r + (i >> 1)], sum[r][n][i], acc[r][n][i]);
      }
    }

    auto leave = [&](int turn) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float* to = sums + (turn * kWarps + warp) * (kRows * C) + (n * 8 + 2 * t) * kRows + r * 16 + g;
          to[0] = acc[r][n][0];
          to[kRows] = acc[r][n][1];
          to[8] = acc[r][n][2];
          to[kRows + 8] = acc[r][n][3];
        }
    };
    if (split == 1) {
      leave(0);
      group_sync();
      finish(unit, 0);
      group_sync();
    } else {
      if (before >= 0) {
        cluster_wait();
        finish(before, turn ^ 1);
      }
      leave(turn);
      cluster_arrive();
      before = unit;
    }
  }
  if (split > 1) {
    cluster_wait();
    finish(before, turn ^ 1);
    cluster_arrive();  // the other CTAs read this one's sums
    cluster_wait();
  }
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
template <typename T, int GROUP, int NT, Groups MODE>
inline int launch_shape(Args a, cudaStream_t st) {
  auto kern = w4_kernel<T, GROUP, NT, MODE>;
  const int segs = (int)((a.K + kSeg - 1) / kSeg);
  auto bytes_for = [&](int split, int stages) {
    return Mma<T>::parts * a.tokens * x_row_bytes((segs + split - 1) / split) + (size_t)kWarps * stages * kItem +
           kBarBytes + sums_bytes(NT) * (split > 1 ? 2 : 1) + kAlign;
  };
  constexpr size_t kMost = 227 * 1024;
  int split = 1;
  while (split < kMaxCluster && bytes_for(split, kMinStages) > kMost) split *= 2;
  if (bytes_for(split, kMinStages) > kMost)
    return fail(KT_ERR_UNSUPPORTED, "w4_linear: K=%lld is too large", (long long)a.K);
  // How the columns are split: turns x (steps of a warp + what a turn costs
  // beside them, in steps), least. The last turn is mostly not full, and few
  // rows fill the device only with their columns split: one token by 8192x8192
  // takes 13 us with 8 warps to 32 rows and 25 with one, by 1024x16384 6.7 us with
  // the columns split over a cluster and 11.6 without; 16 tokens by 16384x16384
  // take 82 us with the one warp that this finds, and 242 with 16.
  const int64_t m_tiles = (a.M + a.tokens - 1) / a.tokens;
  a.units = (int)((a.N + kRows - 1) / kRows);
  const int sms = sm_count();
  int64_t least = INT64_MAX;
  int best_split = split;
  for (int sp = split; sp <= kMaxCluster; sp *= 2) {
    const int64_t ctas = sms / sp / m_tiles > 0 ? sms / sp / m_tiles : 1;
    for (int kw = 1; kw <= kWarps; kw *= 2) {
      const int64_t at_once = ctas * (kWarps / kw), turns = (a.units + at_once - 1) / at_once;
      const int64_t steps = ((segs + sp - 1) / sp + kw - 1) / kw;
      const int64_t cost = turns * (4 * steps + (kw > 1 ? 4 : 2) + (sp > 1 ? 8 : 0));
      if (cost < least) {
        least = cost;
        best_split = sp;
        a.k_warps = kw;
      }
    }
  }
  split = best_split;
  a.stages = kMaxStages;
  while (a.stages > kMinStages && bytes_for(split, a.stages) > kMost) --a.stages;
  const size_t bytes = bytes_for(split, a.stages);
  int resident = 0;
  int rc = resident_clusters((const void*)kern, kThreads, bytes, split, &resident, "w4_linear: launch shape");
  if (rc != KT_OK) return rc;
  if (resident < 1) return fail(KT_ERR_UNSUPPORTED, "w4_linear: no cluster fits");
  const int64_t need = (a.units + kWarps / a.k_warps - 1) / (kWarps / a.k_warps);
  const int64_t room = resident / m_tiles > 0 ? resident / m_tiles : 1;
  const int64_t clusters = need < room ? need : room;
  if (m_tiles > 65535) return fail(KT_ERR_UNSUPPORTED, "w4_linear: M=%lld is too large", (long long)a.M);
  if (a.N > INT32_MAX / 2) return fail(KT_ERR_UNSUPPORTED, "w4_linear: N=%lld is too large", (long long)a.N);
  CUtensorMap map;
  rc = make_tmap_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.packed, (uint64_t)a.N, (uint64_t)a.K / 2,
                    (uint64_t)a.K / 2, kSeg / 2, kRows, CU_TENSOR_MAP_SWIZZLE_64B);
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
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, a, map), "w4_linear launch");
}

template <typename T, int GROUP, int NT>
inline int launch_groups(const Args& a, cudaStream_t st) {
  constexpr int GPS = kSeg / GROUP;
  const bool whole = a.K % kSeg == 0 && elem::aligned_to(a.scales, GPS * (int)sizeof(T)) &&
                     elem::aligned_to(a.zeros, GPS);
  if (!whole) return launch_shape<T, GROUP, NT, kSingle>(a, st);
  return a.zeros ? launch_shape<T, GROUP, NT, kWholeZeros>(a, st) : launch_shape<T, GROUP, NT, kWhole>(a, st);
}

template <typename T>
inline int launch_typed(Args a, int group, cudaStream_t st) {
  // tokens of a CTA: fewer where a cluster cannot hold the share of more
  a.tokens = (int)(a.M < kMaxTokens ? a.M : kMaxTokens);
  const int64_t segs = (a.K + kSeg - 1) / kSeg;
  while (a.tokens > 1 && Mma<T>::parts * a.tokens * x_row_bytes((segs + kMaxCluster - 1) / kMaxCluster) > 96 * 1024)
    a.tokens /= 2;
  const bool one = a.tokens <= 8;
  if (group == 32) return one ? launch_groups<T, 32, 1>(a, st) : launch_groups<T, 32, 2>(a, st);
  if (group == 64) return one ? launch_groups<T, 64, 1>(a, st) : launch_groups<T, 64, 2>(a, st);
  return one ? launch_groups<T, 128, 1>(a, st) : launch_groups<T, 128, 2>(a, st);
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
  const int rc = check_matrix("w4_linear", a.N, a.K, group, dtype, dtype);
  if (rc != KT_OK) return rc;
  if (a.M < 0) return fail(KT_ERR_ARG, "w4_linear: negative M=%lld", (long long)a.M);
  if (a.M == 0 || a.N == 0) return KT_OK;
  if (a.K == 0) return fail(KT_ERR_ARG, "w4_linear: K must be positive");
  if (!a.x || !a.packed || !a.scales || !a.y) return fail(KT_ERR_ARG, "w4_linear: null pointer");
  if (a.ldx < 0 || a.ldy < a.N) return fail(KT_ERR_ARG, "w4_linear: bad row strides");
  const int sz = elem::size_of(dtype);
  if (!aligned16(a.packed)) return fail(KT_ERR_ARG, "w4_linear: packed weights must be 16-byte aligned");
  if (!elem::aligned_to(a.x, sz) || !elem::aligned_to(a.y, sz) || !elem::aligned_to(a.bias, sz) ||
      !elem::aligned_to(a.scales, sz))
    return fail(KT_ERR_ARG, "w4_linear: a pointer is not aligned to its elements");
  // CTAs read x while others store their rows of y
  const uintptr_t x0 = (uintptr_t)a.x, y0 = (uintptr_t)a.y;
  if (x0 < y0 + (uintptr_t)((a.M - 1) * a.ldy + a.N) * sz && y0 < x0 + (uintptr_t)((a.M - 1) * a.ldx + a.K) * sz)
    return fail(KT_ERR_ARG, "w4_linear: y overlaps x");
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
