// Attention of few queries over many keys: one new token per sequence over a paged cache, or a few
// queries over an encoder's states. o = sum_j p_j v_j / sum_j p_j, p_j = 2^(x_j - m), x_j = scale log2 e
// q.k_j, with m a running reference of the largest x.
//
// Bound: memory, every key and value read once for all query heads that share them. The rows of one key
// head (the heads of its group, times the queries) are the 16 columns of a 16x16 matrix instruction,
// whatever their number: it forms the sums over head_dim and over the keys without a lane exchange or
// an LDS round trip, and even with one row of 16 in use it has several times the rate the memory can
// feed (fp32, d 64: 512 bytes of a key and its value take 64 cycles of one SIMD, 20 TB/s over the
// chip). A lane loads what it will multiply, 16 bytes at a time from whole rows, straight into
// registers.
//
// For one 16x16xK instruction lane l (j = l % 16, g = l / 16) supplies row j of A and column j of B at
// its own K / 4 places of the contraction, and holds D[4 g + r][j], r = 0..3. The contraction's order is
// free, and so is the order of A's rows:
//   S^T = K Q^T: A = a tile's 16 keys, lane (j, g) key j; B = the rows; D: key 4 g + r of row j;
//   O^T += V^T P^T: B = P from those registers, so lane (j, g) supplies V of keys 4 g + r at the
//   head_dims that it has loaded of those keys (kC of them, one per instruction): D: row j again.
// Types: an fp32 cache takes the fp32 instruction. A 16-bit one takes the 16-bit instructions, with
// what is not of its type as a sum of 16-bit terms: fp32 queries as three bf16, or two f16 under a scale
// of the row (22 bits of its largest, and an error in a score is one of its size anyway; a third f16 term
// changed fp32 results' error from 7.3e-7 to 7.2e-7); weights, over bf16 values, as three bf16, which hold
// their 24 bits. (Two are off by 2^-17 of a weight, and a bf16 result that lies near a tie then rounds to
// the wrong side: 86 of 16384 results over 60000 to 131071 tokens, 15 so, where sums in fp32 give 46. Two /
// three, bf16, us: those contexts, d 128, 279.4 / 279.9; 64 sequences of 1 to 2048, d 64, 27.1 / 27.5.)
// Over f16 values the weights stay fp32 and the values are widened: f16 terms of a weight
// would end at 2^-24 of the largest one's size, and a key of all the weight but no value (an attention
// sink) would take the bits of all the others.
//
// Work: the sequences' 32-key tiles, end to end, are dealt in equal runs to a fixed number of
// workgroups, whatever the lengths; a workgroup's run crosses heads and sequences. Where a run ends
// inside a head the workgroup leaves its unnormalised sums in the workspace (at most two: its first
// and its last head), and a second kernel joins them in order. Reruns are bit-identical. A head counts
// kSplitWaves tiles more than it has, which is what beginning one costs: without, the workgroup that the
// shortest sequences fall to ends last (64 sequences of 1 to 2048, 6 heads, fp32 d 64: 79 us, 46 so).
//
// Measured (kernel and join): 4 contexts of 60000 to 131071, 32 heads in 8 groups, d 128 bf16, 263 to 273 + 5
// us (5.7 to 5.9 TB/s, by card); that ragged batch 45 + 5 us (4.5 TB/s); 8 x 6 heads 1 x 1536 fp32 12.4 + 3.9
// us (3.0 TB/s); one sequence of 240, 6 heads, 7.8 us, the latency of one workgroup, where the table has room
// for little more (split_plan); under one for 4096 or 131072 tokens the same sequence takes runs and a join,
// 10.5 us for 7.3 from a graph, 64 such sequences 20.1 for 12.6.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "fattn_device.h"
#include "fattn_internal.h"

namespace fattn {
namespace {

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int kSplitWaves = 4;
constexpr int kMostRuns = 1024;     // workgroups, with runs: 256 x kOccupancy
constexpr int kTile = kSplitTile;   // keys of a tile: two halves of 16
constexpr int kRowsMax = 16;        // rows of a block
constexpr float kRoom = 4.0f;       // log2 of what a weight may pass its reference by

__device__ __forceinline__ f4 mma_f32(float a, float b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4 mma_16(u4 a, u4 b, f4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c,
                                                0, 0, 0);
}
__device__ __forceinline__ f4 mma_16(u4 a, u4 b, f4 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b),
                                                 c, 0, 0, 0);
}

// Over the four lanes that hold one row (j, j + 16, j + 32, j + 48).
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float row_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// x and y as sums of N terms of type C, largest first, two values to a word. Each term but the last is
// cut off towards 0 and none is 0 where x is not (a rest of nothing counts as 2^-30 of x): all have x's
// sign, and an infinity that they multiply stays one.
__device__ __forceinline__ float rest(float x, float least) { return fabsf(x) > fabsf(least) ? x : least; }
template <int N>
__device__ __forceinline__ void terms2(float x, float y, unsigned (&w)[N], __bf16) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const float lx = x * 0x1p-30f, ly = y * 0x1p-30f;
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    const unsigned hx = __float_as_uint(x) & 0xffff0000u, hy = __float_as_uint(y) & 0xffff0000u;
    w[i] = __builtin_amdgcn_perm(hy, hx, 0x07060302u);
    x = rest(x - __uint_as_float(hx), lx), y = rest(y - __uint_as_float(hy), ly);
  }
  w[N - 1] = __builtin_bit_cast(unsigned, b2{static_cast<__bf16>(x), static_cast<__bf16>(y)});
}
template <int N>
__device__ __forceinline__ void terms2(float x, float y, unsigned (&w)[N], _Float16) {
  static_assert(N == 2, "two f16");
  const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
  w[0] = __builtin_bit_cast(unsigned, h);
  // (The least f16 is 2^-24.)
  const float lx = x == 0.0f ? 0.0f : copysignf(0x1p-24f, x), ly = y == 0.0f ? 0.0f : copysignf(0x1p-24f, y);
  x = rest(x - static_cast<float>(h.x), lx), y = rest(y - static_cast<float>(h.y), ly);
  w[1] = __builtin_bit_cast(unsigned, h2{static_cast<_Float16>(x), static_cast<_Float16>(y)});
}

// Tiles of sequence b, and its length; bad: a length that the cache cannot hold.
template <bool kPaged>
__device__ __forceinline__ int seq_tiles(const SplitArgs& a, int b, int& len, bool& bad) {
  len = a.lengths != nullptr ? a.lengths[b] : a.SK;
  bad = kPaged && (len < 0 || len > a.SK);
  len = bad ? 0 : min(max(len, 0), a.SK);
  return (len + kTile - 1) / kTile;
}
// A value that is one for the whole wave, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(x));
  const unsigned hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(static_cast<uint64_t>(x) >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
// x / y of values that are not negative: in 32 bits where they fit (a 64-bit division takes 0.3 us).
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  if (((x | y) >> 31) == 0) return static_cast<unsigned>(x) / static_cast<unsigned>(y);
  return x / y;
}
// What a sequence of n tiles counts for per key head: its tiles, and what beginning a head costs.
__device__ __forceinline__ int64_t cost(const SplitArgs& a, int n) { return n == 0 ? 0 : n + a.begin; }
// The length of a run.
__device__ __forceinline__ int64_t quota(const SplitArgs& a, int64_t units) {
  const int64_t q = quotient(units + a.wgs - 1, a.wgs);
  return q < a.min_run ? a.min_run : q;
}
// Row r of key head kvh: its query head and query.
__device__ __forceinline__ void row_of(const SplitArgs& a, int kvh, int r, int& head, int& i) {
  const int in = a.SQ == 1 ? r : r / a.SQ;
  head = kvh * a.G + in;
  i = r - in * a.SQ;
}
__device__ __forceinline__ void put_lse(const SplitArgs& a, int b, int head, int i, float m, float l) {
  if (a.lse == nullptr) return;
  // L = m ln 2 + ln l, with scale log2 e as rounded into the exponents taken out again.
  const float c2 = a.scale * kLog2e;
  const double mr = c2 == 0.0f ? 0.6931471805599453 : static_cast<double>(a.scale) / c2;
  a.lse[(static_cast<int64_t>(b) * a.H + head) * a.SQ + i] =
      l == 0.0f ? kNegInf : static_cast<float>(static_cast<double>(m) * mr + logf(l));
}
template <typename Q>
__device__ __forceinline__ Q* out_row(const SplitArgs& a, int b, int head, int i, int d) {
  return static_cast<Q*>(a.o) + ((static_cast<int64_t>(b) * a.SQ + i) * a.H + head) * d;
}
template <typename Q>
__device__ __forceinline__ void put4(Q* p, f4 x) {
  typedef Q q4 __attribute__((ext_vector_type(4)));
  const q4 y{static_cast<Q>(x[0]), static_cast<Q>(x[1]), static_cast<Q>(x[2]), static_cast<Q>(x[3])};
  *reinterpret_cast<q4*>(p) = y;
}

// The registers of one wave: a tile's keys and values, the rows, the sums.
template <typename Q, typename C, int D>
struct Wave {
  static constexpr bool kF32 = std::is_same<C, float>::value;
  static constexpr int kC = kF32 ? (D == 32 ? 2 : 4) : D / 16;  // head_dims of V per load
  static constexpr int kBlocks = D / (16 * kC);                 // loads of a V row
  static constexpr int kKLoads = kF32 ? D / 16 : D / 32;        // loads of a K row, 16 bytes a lane
  static constexpr int kVWords = kF32 ? kC : kC / 2;
  static constexpr int kAcc = D / 16;
  // Terms of the queries and of the weights (1: as they are).
  static constexpr bool kSame = std::is_same<Q, C>::value;
  static constexpr int kQT = kF32 || kSame ? 1 : std::is_same<C, __bf16>::value ? 3 : 2;
  static constexpr int kPT = 3;  // (bf16)

  u4 k[2][kKLoads];
  unsigned v[2][4][kBlocks][kVWords];
  u4 q[kQT][kKLoads];
  f4 o[kAcc];  // register r of o[kC T + n]: head_dim 16 kC T + kC (4 g + r) + n of row j
  float c2;    // scale log2 e over the row's scale
  float m, l;

  __device__ __forceinline__ void load_q(const Q* row, float scale, int g) {
    c2 = scale * kLog2e;
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) q[0][i] = *reinterpret_cast<const u4*>(row + 16 * i + 4 * g);
    } else if constexpr (kSame) {
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) q[0][i] = *reinterpret_cast<const u4*>(row + 32 * i + 8 * g);
    } else {
      f4 x[kKLoads][2];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        x[i][0] = ld4(row + 32 * i + 8 * g);
        x[i][1] = ld4(row + 32 * i + 8 * g + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e / 4][e % 4]));
      }
      float sc = 1.0f;
      if constexpr (std::is_same<C, _Float16>::value) {
        // The row's largest magnitude at 2^13: 22 bits of each value down to 2^-17 of it.
        const int e = min(max(static_cast<int>(__float_as_uint(row_max(top)) >> 23) - 127, -113), 126);
        sc = __int_as_float((13 - e + 127) << 23);
        c2 *= __int_as_float((e - 13 + 127) << 23);
      }
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        unsigned w[4][kQT];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          terms2(x[i][e / 2][2 * (e % 2)] * sc, x[i][e / 2][2 * (e % 2) + 1] * sc, w[e], C{});
        }
#pragma unroll
        for (int t = 0; t < kQT; ++t) q[t][i] = u4{w[0][t], w[1][t], w[2][t], w[3][t]};
      }
    }
  }
  __device__ __forceinline__ void clear() {
    m = kNegInf, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kAcc; ++i) o[i] = f4{};
  }
  // Half h of a tile, from the row of its first key (uniform, so a load is a scalar base and a 32-bit
  // offset of the lane); `live` of its 16 keys are there (the others repeat the last).
  __device__ __forceinline__ void load_k(int h, const C* p, unsigned ss, int live, int j, int g) {
    const char* base = reinterpret_cast<const char*>(p);
    const unsigned at = static_cast<unsigned>(min(j, live - 1)) * ss + 16u * g;
#pragma unroll
    for (int i = 0; i < kKLoads; ++i) k[h][i] = *reinterpret_cast<const u4*>(base + (at + 64u * i));
  }
  __device__ __forceinline__ void load_v(int h, const C* p, unsigned ss, int live, int j, int g) {
    const char* base = reinterpret_cast<const char*>(p);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const unsigned at =
          static_cast<unsigned>(min(4 * g + r, live - 1)) * ss + static_cast<unsigned>(kC * sizeof(C)) * j;
#pragma unroll
      for (int t = 0; t < kBlocks; ++t) {
        const char* row = base + (at + static_cast<unsigned>(16 * kC * sizeof(C)) * t);
        if constexpr (kVWords == 4) {
          const u4 x = *reinterpret_cast<const u4*>(row);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[h][r][t][i] = x[i];
        } else if constexpr (kVWords == 2) {
          const u2 x = *reinterpret_cast<const u2*>(row);
          v[h][r][t][0] = x[0], v[h][r][t][1] = x[1];
        } else {
          v[h][r][t][0] = *reinterpret_cast<const unsigned*>(row);
        }
      }
    }
  }
  __device__ __forceinline__ void scores(f4 (&s)[2]) const {
    s[0] = f4{}, s[1] = f4{};
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[h] = mma_f32(__uint_as_float(k[h][i][e]), __uint_as_float(q[0][i][e]), s[h]);
          }
        }
      }
    } else {
#pragma unroll
      for (int t = kQT - 1; t >= 0; --t) {  // small terms first
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h) s[h] = mma_16(k[h][i], q[t][i], s[h], C{});
        }
      }
    }
  }
  // Weights from scores, `live` keys of the tile.
  __device__ __forceinline__ void weights(f4 (&s)[2], int live, int g) {
    float top = kNegInf;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[h][r] = 16 * h + 4 * g + r < live ? s[h][r] * c2 : kNegInf;
        top = fmaxf(top, s[h][r]);
      }
    }
    // The reference moves only when a weight passes it by 2^kRoom (or there is none yet).
    if (__builtin_amdgcn_ballot_w64(top > m + kRoom) != 0) {
      const float to = fmaxf(m, row_max(top));
      const float f = m == kNegInf ? 0.0f : exp2_hw(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int i = 0; i < kAcc; ++i) o[i] *= f;
    }
    const float ref = m == kNegInf ? 0.0f : m;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[h][r] = exp2_hw(s[h][r] - ref);
        l += s[h][r];
      }
    }
  }
  // o += V^T P^T. Values of absent keys count as 0, whatever memory holds there.
  __device__ __forceinline__ void sums(const f4 (&p)[2], int live, int g) {
    if (live < kTile) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (16 * h + 4 * g + r >= live) {
#pragma unroll
            for (int t = 0; t < kBlocks; ++t) {
#pragma unroll
              for (int i = 0; i < kVWords; ++i) v[h][r][t][i] = 0;
            }
          }
        }
      }
    }
    if constexpr (kF32) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int t = 0; t < kBlocks; ++t) {
#pragma unroll
            for (int n = 0; n < kC; ++n) {
              o[kC * t + n] = mma_f32(__uint_as_float(v[h][r][t][n]), p[h][r], o[kC * t + n]);
            }
          }
        }
      }
    } else if constexpr (std::is_same<C, _Float16>::value) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int i = 0; i < kVWords; ++i) {
            const h2 x = __builtin_bit_cast(h2, v[h][r][0][i]);
            o[2 * i] = mma_f32(static_cast<float>(x.x), p[h][r], o[2 * i]);
            o[2 * i + 1] = mma_f32(static_cast<float>(x.y), p[h][r], o[2 * i + 1]);
          }
        }
      }
    } else {
      u4 b[kPT];
      unsigned w[4][kPT];
#pragma unroll
      for (int e = 0; e < 4; ++e) terms2(p[e / 2][2 * (e % 2)], p[e / 2][2 * (e % 2) + 1], w[e], C{});
#pragma unroll
      for (int t = 0; t < kPT; ++t) b[t] = u4{w[0][t], w[1][t], w[2][t], w[3][t]};
#pragma unroll
      for (int i = 0; i < kVWords; ++i) {
        // Two keys' values of one head_dim into one word: the low halves (n = 2 i), the high ones.
        u4 lo, hi;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned x = v[e / 2][2 * (e % 2)][0][i], y = v[e / 2][2 * (e % 2) + 1][0][i];
          lo[e] = __builtin_amdgcn_perm(y, x, 0x05040100u);
          hi[e] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        }
#pragma unroll
        for (int t = kPT - 1; t >= 0; --t) {
          o[2 * i] = mma_16(lo, b[t], o[2 * i], C{});
          o[2 * i + 1] = mma_16(hi, b[t], o[2 * i + 1], C{});
        }
      }
    }
  }
};

// Waves per SIMD (so workgroups per CU) that the registers allow.
template <typename Q, typename C, int D>
constexpr int kOccupancy = D == 32    ? 4
                           : D == 128 ? 2
                           : std::is_same<C, _Float16>::value || (std::is_same<C, __bf16>::value &&
                                                                  std::is_same<Q, C>::value)
                               ? 4
                               : 3;

template <typename Q, typename C, int D, bool kPaged>
__global__ void __launch_bounds__(64 * kSplitWaves)
    __attribute__((amdgpu_waves_per_eu(kOccupancy<Q, C, D>, kOccupancy<Q, C, D>)))
split_kernel(SplitArgs a) {
  typedef Wave<Q, C, D> W;
  constexpr int kPitch = D + 4;
  __shared__ __attribute__((aligned(16))) float so[kSplitWaves][kRowsMax][kPitch];
  __shared__ float sml[kSplitWaves][2][kRowsMax];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = a.HK * a.RB;

  // This workgroup's run: `left` of the sequences' costs end to end, from `off` into sequence b's.
  int b = 0;
  int64_t off = 0, left = 0;
  int early[2] = {};  // the pages of the wave's first tile
  if (a.wgs == 0) {  // one workgroup per key head and block of rows
    b = static_cast<int>(blockIdx.x) / heads;
    if constexpr (kPaged) {
      // Read beside the length, which says whether the tile is there: one load's latency less before the
      // first keys (one sequence of 240: 8.1 us without, 7.8 so).
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        early[h] = a.table[b * a.table_stride + divide(min(2 * w + h, a.SK / 16 - 1), a.by_page)];
      }
    }
  } else {
    // Each wave for itself, without LDS: a lane takes `each` sequences that follow one another.
    const int each = (a.B + 63) / 64, from = min(lane * each, a.B), to = min(from + each, a.B);
    auto costs = [&](int i) {
      int len;
      bool bad;
      return cost(a, seq_tiles<kPaged>(a, i, len, bad)) * heads;
    };
    long long mine = 0;
    for (int i = from; i < to; ++i) mine += costs(i);
    long long upto = mine;
    for (int i = 1; i < 64; i *= 2) {
      const long long y = __shfl_up(upto, i);
      if (lane >= i) upto += y;
    }
    const int64_t units = uniform(__shfl(upto, 63)), run = uniform(quota(a, units));
    const int64_t u = static_cast<int64_t>(blockIdx.x) * run;
    if (blockIdx.x == 0 && w == 0) {  // where each sequence begins, for the join
      int64_t at = upto - mine;
      for (int i = from; i < to; ++i) {
        a.before[i] = at;
        at += costs(i);
      }
      if (lane == 63) a.before[a.B] = units;
    }
    if (u >= units) return;
    left = units - u < run ? units - u : run;
    // The lane whose sequences u is in, and which of them.
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(u < upto));
    int64_t base = uniform(__shfl(upto - mine, at));
    b = __builtin_amdgcn_readfirstlane(at * each);
    for (int64_t c = uniform(costs(b)); u >= base + c; c = uniform(costs(b))) base += c, ++b;
    off = u - base;
  }

  while (true) {
    int len;
    bool bad;
    const int n = __builtin_amdgcn_readfirstlane(seq_tiles<kPaged>(a, b, len, bad));
    len = __builtin_amdgcn_readfirstlane(len);
    int hh, t0 = 0, t1 = n;
    if (a.wgs == 0) {
      hh = static_cast<int>(blockIdx.x) % heads;
    } else {
      if (left <= 0) return;
      const int64_t each = cost(a, n);
      if (off >= each * heads) {
        off -= each * heads;
        ++b;
        continue;
      }
      hh = __builtin_amdgcn_readfirstlane(static_cast<int>(quotient(off, each)));
      // The run's part of this head, [in, in + take) of begin + n: the tiles are what is past `begin`.
      const int64_t in = off - each * hh, take = left < each - in ? left : each - in;
      t0 = __builtin_amdgcn_readfirstlane(static_cast<int>(in > a.begin ? in - a.begin : 0));
      t1 = __builtin_amdgcn_readfirstlane(static_cast<int>(in + take > a.begin ? in + take - a.begin : 0));
      left -= take;
      off += take;
      if (t0 == t1) continue;
    }
    const int kvh = hh / a.RB, r0 = hh % a.RB * kRowsMax;
    const int rows = min(a.G * a.SQ - r0, kRowsMax);

    // --- The wave's tiles: t0 + w, t0 + w + 4, ...
    W x;
    x.clear();
    int wrong = 0;  // a page that the cache does not have
    {
      int head, i;
      row_of(a, kvh, r0 + min(j, rows - 1), head, i);
      x.load_q(static_cast<const Q*>(a.q) + b * a.qs[0] + head * a.qs[1] + i * a.qs[2], a.scale, g);
    }
    const C* kp = static_cast<const C*>(a.k) + kvh * a.ks[1];
    const C* vp = static_cast<const C*>(a.v) + kvh * a.vs[1];
    if constexpr (!kPaged) kp += b * a.ks[0], vp += b * a.vs[0];
    // The first key's row of half h of tile t, and how many keys the half has. A half past the end is
    // the last one that has keys.
    struct Half {
      const C *k, *v;
      int live;
    };
    auto half = [&](int t, int h) {
      const int at = min(2 * t + h, (len - 1) / 16);
      Half x;
      x.live = min(len - 16 * at, 16);
      if constexpr (kPaged) {
        const int pi = divide(at, a.by_page), slot = 16 * (at - pi * (a.page_size / 16));
        const bool had = a.wgs == 0 && at == 2 * w + h;
        int page = __builtin_amdgcn_readfirstlane(had ? early[h] : a.table[b * a.table_stride + pi]);
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) page = 0, wrong = 1;
        x.k = kp + page * a.ks[0] + slot * a.ks[2];
        x.v = vp + page * a.vs[0] + slot * a.vs[2];
      } else {
        x.k = kp + 16ll * at * a.ks[2];
        x.v = vp + 16ll * at * a.vs[2];
      }
      return x;
    };
    // A step: scores of the tile in hand, and over what follows the loads of the next tile's keys;
    // weights and sums; the loads of its values.
    const unsigned kss = static_cast<unsigned>(a.ks[2] * sizeof(C));
    const unsigned vss = static_cast<unsigned>(a.vs[2] * sizeof(C));
    int t = t0 + w;
    Half at[2];
    if (t < t1) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        at[h] = half(t, h);
        x.load_k(h, at[h].k, kss, at[h].live, j, g);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) x.load_v(h, at[h].v, vss, at[h].live, j, g);
    }
    for (; t < t1; t += kSplitWaves) {
      const int live = len - kTile * t;
      const bool more = t + kSplitWaves < t1;
      f4 s[2];
      x.scores(s);
      if (more) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          at[h] = half(t + kSplitWaves, h);
          x.load_k(h, at[h].k, kss, at[h].live, j, g);
        }
      }
      x.weights(s, live, g);
      x.sums(s, live, g);
      if (more) {
#pragma unroll
        for (int h = 0; h < 2; ++h) x.load_v(h, at[h].v, vss, at[h].live, j, g);
      }
    }

    // --- The waves' sums, through LDS.
    x.l = row_sum(x.l);
    if constexpr (kPaged) {
      if (wrong) x.l = __builtin_nanf("");
    }
    if (g == 0) sml[w][0][j] = x.m, sml[w][1][j] = x.l;
    if (j < rows) {
#pragma unroll
      for (int bl = 0; bl < W::kBlocks; ++bl) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int c = 0; c < W::kC; ++c) {
            so[w][j][16 * W::kC * bl + W::kC * (4 * g + r) + c] = x.o[W::kC * bl + c][r];
          }
        }
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == n;
    float* part = whole ? nullptr
                        : a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 == 0 ? 1 : 0)) *
                                       a.part_rows * (D + 4);
    for (int i = tid; i < rows * (D / 4); i += 64 * kSplitWaves) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      float m = kNegInf;
#pragma unroll
      for (int y = 0; y < kSplitWaves; ++y) m = fmaxf(m, sml[y][0][row]);
      f4 o{};
      float l = 0.0f;
#pragma unroll
      for (int y = 0; y < kSplitWaves; ++y) {
        const float my = sml[y][0][row], ly = sml[y][1][row];
        // (A wave without a finite score has sums of 0, or NaN for infinite values; its l may still be NaN,
        // for a page.)
        const float f = my == kNegInf ? 0.0f : my == m ? 1.0f : exp2_hw(my - m);
        l += my == kNegInf ? ly : ly * f;
        o += ld4(&so[y][row][d]) * f;
      }
      if (whole) {
        int head, q;
        row_of(a, kvh, r0 + row, head, q);
        // (l is 0 where every score is minus infinity: NaN, as the formula.)
        put4(out_row<Q>(a, b, head, q, D) + d, o * (1.0f / l));
        if (d == 0) put_lse(a, b, head, q, m, l);
      } else {
        st4(part + row * (D + 4) + d, o);
        if (d == 0) part[row * (D + 4) + D] = m, part[row * (D + 4) + D + 1] = l;
      }
    }
    if (a.wgs == 0) {
      if (n == 0) {  // no keys: zeros (a length outside the cache: NaN)
        for (int i = tid; i < rows * (D / 4); i += 64 * kSplitWaves) {
          const int row = i / (D / 4), d = i % (D / 4) * 4;
          int head, q;
          row_of(a, kvh, r0 + row, head, q);
          const float z = bad ? __builtin_nanf("") : 0.0f;
          put4(out_row<Q>(a, b, head, q, D) + d, f4{z, z, z, z});
        }
      }
      return;
    }
    __syncthreads();
  }
}

// The partial sums of one row (b, head, query), joined in the order of the keys: thread (group, lane)
// takes every kGroups-th, D / 4 lanes a group.
template <typename Q, int D, bool kPaged>
__global__ void __launch_bounds__(256) join_kernel(SplitArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ __attribute__((aligned(16))) float so[kGroups][D];
  __shared__ float sm[kGroups], sl[kGroups];
  const int tid = threadIdx.x, d = tid % kLanes * 4, grp = tid / kLanes;
  const int per = a.H * a.SQ;
  const int b = static_cast<int>(blockIdx.x) / per, in = static_cast<int>(blockIdx.x) % per;
  const int head = in / a.SQ, q = in % a.SQ, kvh = head / a.G;
  const int r = (head - kvh * a.G) * a.SQ + q, hh = kvh * a.RB + r / kRowsMax;
  // (All three before anything waits for one of them.)
  const int64_t at_b = a.before[b], units = a.before[a.B];
  int len;
  bool bad;
  const int n = seq_tiles<kPaged>(a, b, len, bad);
  if (n == 0) {
    const float z = bad ? __builtin_nanf("") : 0.0f;
    if (grp == 0) put4(out_row<Q>(a, b, head, q, D) + d, f4{z, z, z, z});
    if (tid == 0) put_lse(a, b, head, q, 0.0f, bad ? z : 0.0f);
    return;
  }
  const int64_t run = quota(a, units);
  const int64_t u0 = at_b + static_cast<int64_t>(hh) * (n + a.begin) + a.begin;
  const int w0 = static_cast<int>(quotient(u0, run)), w1 = static_cast<int>(quotient(u0 + n - 1, run));
  if (w0 == w1) return;  // written by its one workgroup
  const int64_t pitch = static_cast<int64_t>(a.part_rows) * (D + 4);
  const float* row = a.part + (r % kRowsMax) * (D + 4);
  auto slot = [&](int w) { return row + (static_cast<int64_t>(w) * 2 + (w == w0 ? 1 : 0)) * pitch; };
  float m = kNegInf, l = 0.0f;
  f4 o{};
  constexpr int kAtOnce = 4;  // parts in flight
  for (int w = w0 + grp; w <= w1; w += kGroups * kAtOnce) {
    float ms[kAtOnce], ls[kAtOnce];
    f4 os[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float* p = slot(min(w + i * kGroups, w1));
      ms[i] = p[D], ls[i] = p[D + 1], os[i] = ld4(p + d);
    }
    const float before = m;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (w + i * kGroups > w1) ms[i] = kNegInf, ls[i] = 0.0f, os[i] = f4{};
      m = fmaxf(m, ms[i]);
    }
    const float f = before == kNegInf ? 0.0f : exp2_hw(before - m);
    o *= f, l *= before == kNegInf ? 1.0f : f;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      // (As for the waves' sums.)
      const float fi = ms[i] == kNegInf ? 0.0f : exp2_hw(ms[i] - m);
      l += ms[i] == kNegInf ? ls[i] : ls[i] * fi;
      o += os[i] * fi;
    }
  }
  st4(&so[grp][d], o);
  if (d == 0) sm[grp] = m, sl[grp] = l;
  __syncthreads();
  if (grp != 0) return;
  float mm = kNegInf;
  for (int y = 0; y < kGroups; ++y) mm = fmaxf(mm, sm[y]);
  o = f4{}, l = 0.0f;
  for (int y = 0; y < kGroups; ++y) {
    const float f = sm[y] == kNegInf ? 0.0f : exp2_hw(sm[y] - mm);
    l += sm[y] == kNegInf ? sl[y] : sl[y] * f;
    o += ld4(&so[y][d]) * f;
  }
  put4(out_row<Q>(a, b, head, q, D) + d, o * (1.0f / l));
  if (tid == 0) put_lse(a, b, head, q, mm, l);
}

template <typename Q, typename C, int D, bool kPaged>
int run_split(const SplitArgs& a, hipStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(a.B) * a.HK * a.RB;
  SplitArgs args = a;
  if (args.wgs > 0) args.wgs = 256 * kOccupancy<Q, C, D>;
  void* kargs[] = {&args};
  const unsigned grid = static_cast<unsigned>(args.wgs == 0 ? pairs : args.wgs);
  hipError_t err = hipLaunchKernel(reinterpret_cast<const void*>(split_kernel<Q, C, D, kPaged>),
                                   dim3(grid), dim3(64 * kSplitWaves), kargs, 0, stream);
  if (err != hipSuccess || a.wgs == 0) return static_cast<int>(err);
  const unsigned rows = static_cast<unsigned>(static_cast<int64_t>(a.B) * a.H * a.SQ);
  return static_cast<int>(hipLaunchKernel(reinterpret_cast<const void*>(join_kernel<Q, D, kPaged>),
                                          dim3(rows), dim3(256), kargs, 0, stream));
}

template <typename Q, typename C, bool kPaged>
int by_dim(const SplitArgs& a, int d, hipStream_t s) {
  return d == 32   ? run_split<Q, C, 32, kPaged>(a, s)
         : d == 64 ? run_split<Q, C, 64, kPaged>(a, s)
                   : run_split<Q, C, 128, kPaged>(a, s);
}

}  // namespace

SplitPlan split_plan(int64_t b, int64_t hk, int64_t rows, int64_t d, int64_t capacity) {
  SplitPlan p{};
  p.row_blocks = static_cast<int>((rows + kRowsMax - 1) / kRowsMax);
  p.part_rows = static_cast<int>(rows < kRowsMax ? rows : kRowsMax);
  const int64_t tiles = (capacity + kTile - 1) / kTile;
  p.min_run = kSplitWaves;
  p.begin = kSplitWaves;
  // One workgroup per key head, and no join, where no sequence can have more than four tiles a wave, or
  // eight with a workgroup for most CUs: by what the tables have room for, since the lengths are on the
  // device. Direct / in runs, us (with 6 us of a graph's launch): fp32 d 64,
  // 384 heads of 1024 tokens 45.9 / 52.6, of 1 to 700 25.6 / 29.9; bf16 d 128, 256 of 1000 28.8 / 35.5,
  // 192 26.0 / 29.7; past it 384 of 1 to 2048 64.9 / 54.7, 48 of 1000 28.2 / 20.8, of 1500 37.8 / 23.0. (A
  // wave alone takes 2 us a tile, the memory's latency twice; eight waves a workgroup change little.)
  const int64_t direct = b * hk * p.row_blocks >= 192 ? 8 * kSplitWaves : 4 * kSplitWaves;
  p.wgs = tiles <= direct ? 0 : kMostRuns;
  p.before = static_cast<size_t>(p.wgs) * 2 * p.part_rows * static_cast<size_t>(d + 4) * sizeof(float);
  p.bytes = p.wgs == 0 ? 0 : p.before + static_cast<size_t>(b + 1) * sizeof(int64_t);
  return p;
}

int launch_split(const SplitArgs& a, int dtype, int cache_dtype, int d, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.table == nullptr) return by_dim<float, float, false>(a, d, s);
  if (dtype == kF16) return by_dim<_Float16, _Float16, true>(a, d, s);
  if (dtype == kBF16) return by_dim<__bf16, __bf16, true>(a, d, s);
  return cache_dtype == kF16    ? by_dim<float, _Float16, true>(a, d, s)
         : cache_dtype == kBF16 ? by_dim<float, __bf16, true>(a, d, s)
                                : by_dim<float, float, true>(a, d, s);
}

}  // namespace fattn
