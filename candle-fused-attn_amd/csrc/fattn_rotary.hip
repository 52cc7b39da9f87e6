// Rotary positions, and the append of keys and values to a paged cache with the rotation on the way.
//
// A rotated head has n = dim / 2 pairs of values, (x_i, x_{i + n}) or, interleaved, (x_2i, x_2i+1);
// pair i at position p turns by the angle a = p f_i:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,  c = magnitude cos a,  s = magnitude sin a
// and values past dim stay. The inverse (the gradient) turns by -a with the same magnitude.
//
// Bound: memory, each value read and written once. A workgroup takes a few tokens with all their
// heads, so that an angle's sine and cosine are formed once per token and pair (in LDS) and not once
// per head; positions need no table in memory and have no largest value.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "fattn_internal.h"

namespace fattn {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxTokens = 16;   // tokens of a workgroup
constexpr int kMaxAngles = 1024; // angles of a workgroup (LDS: 8 bytes each)
constexpr int kUnroll = 4;       // items a thread has in flight

// cos and sin of p f, times the magnitude. The angle is formed and reduced in 64 bits, since in 32 one
// of 10^5 radians is off by 4e-3: t = a / 2 pi turns, less its nearest quarter, leaves |y| <= pi / 4,
// where the Taylor series to y^13 and y^12 are exact to 1e-12.
__device__ __forceinline__ float2 turn(double p, double f, double magnitude) {
  const double t = p * f * 0.15915494309189533577;
  const double q = rint(4.0 * t);
  const double y = fma(q, -0.25, t) * 6.28318530717958647693, z = y * y;
  double s = 1.0 / 6227020800.0, c = 1.0 / 479001600.0;
  s = fma(s, z, -1.0 / 39916800.0), c = fma(c, z, -1.0 / 3628800.0);
  s = fma(s, z, 1.0 / 362880.0), c = fma(c, z, 1.0 / 40320.0);
  s = fma(s, z, -1.0 / 5040.0), c = fma(c, z, -1.0 / 720.0);
  s = fma(s, z, 1.0 / 120.0), c = fma(c, z, 1.0 / 24.0);
  s = fma(s, z, -1.0 / 6.0), c = fma(c, z, -0.5);
  s = fma(s * z, y, y), c = fma(c, z, 1.0);
  // q mod 4 quarters (of a double: an angle of 2^33 turns has a q past 32 bits).
  const int k = static_cast<int>(q - 4.0 * floor(0.25 * q));
  const double cc = (k & 1) ? s : c, ss = (k & 1) ? c : s;
  return float2{static_cast<float>(((k == 1 || k == 2) ? -cc : cc) * magnitude),
                static_cast<float>((k >= 2 ? -ss : ss) * magnitude)};
}

// N values moved at once: wide accesses need their alignment, one or two values only their own.
template <typename T, int N>
struct alignas(N >= 4 ? sizeof(T) * N : sizeof(T)) Vec {
  T v[N];
};
// One rounding to the stored type, to nearest; none where it is the loaded one and nothing turned.
template <typename C, typename T>
__device__ __forceinline__ C convert(T x) {
  return static_cast<C>(static_cast<float>(x));
}
template <>
__device__ __forceinline__ float convert<float, float>(float x) { return x; }
template <>
__device__ __forceinline__ _Float16 convert<_Float16, _Float16>(_Float16 x) { return x; }
template <>
__device__ __forceinline__ __bf16 convert<__bf16, __bf16>(__bf16 x) { return x; }

// x c + y in 32 bits, rounded there before any rounding to 16 (an instruction that fuses the two is
// taken for some widths of access and not for others: results would depend on a tensor's alignment).
__device__ __forceinline__ float turned(float x, float c, float y) {
  float r = fmaf(x, c, y);
  asm("" : "+v"(r));
  return r;
}

// A workgroup: `tokens` tokens, and the share blockIdx.y of their items. An item is VEC pairs of a
// rotated head in the half layout (two vectors, n apart), else VEC values. Items of a token, part by
// part and head by head, run over a head's values, so a wave reads whole rows.
template <typename T, typename C, int VEC, bool kInterleaved, bool kPaged>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[kMaxAngles];
  __shared__ int64_t pos_of[kMaxTokens], at_of[2][kMaxTokens];  // at: k's and v's place in the pages
  __shared__ int seq_of[kMaxTokens], in_of[kMaxTokens];
  const int tid = threadIdx.x, n = a.pairs;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens, all = static_cast<int64_t>(a.B) * a.S;
  const int nt = static_cast<int>(all - t0 < a.tokens ? all - t0 : a.tokens);
  if (tid < nt) {
    const int64_t t = t0 + tid;
    const int b = static_cast<int>(t / a.S), i = static_cast<int>(t % a.S);
    int64_t p;
    if constexpr (kPaged) {
      const int held = a.lengths[b];
      p = static_cast<int64_t>(held) + i;
      // A token past its sequence's count, or whose page the table or the cache does not have, is not
      // written.
      int64_t page = -1;
      const bool counted = a.counts == nullptr || i < a.counts[b];
      if (counted && held >= 0 && p / a.page_size < a.table_width) {
        page = a.table[b * a.table_stride + p / a.page_size];
      }
      const bool live = page >= 0 && page < a.pages;
      const int64_t slot = p % a.page_size;
      at_of[0][tid] = live ? page * a.page_strides[0] + slot * a.page_strides[2] : -1;
      at_of[1][tid] = live ? page * a.page_strides[3] + slot * a.page_strides[5] : -1;
    } else {
      const int64_t at = b * a.pos_strides[0] + i * a.pos_strides[1];
      p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                  : static_cast<const int32_t*>(a.positions)[at];
    }
    pos_of[tid] = p, seq_of[tid] = b, in_of[tid] = i;
  }
  __syncthreads();
  for (int i = tid; i < nt * n; i += kRotThreads) {
    float2 x = turn(static_cast<double>(pos_of[i / n]), a.frequencies[i % n], a.magnitude);
    if (a.inverse) x.y = -x.y;
    cs[i] = x;
  }
  __syncthreads();

  typedef Vec<T, VEC> In;
  // Items per head: rotated ones first, then copies of the rest.
  const int turns = kInterleaved ? 2 * n / VEC : n / VEC, rest = (a.D - 2 * n) / VEC, plain = a.D / VEC;
  const int n0 = a.part[0].heads * (a.part[0].rotate ? turns + rest : plain);
  const int n1 = a.part[1].heads * (a.part[1].rotate ? turns + rest : plain);
  const int n2 = a.part[2].heads * (a.part[2].rotate ? turns + rest : plain);
  const int per = n0 + n1 + n2, items = nt * per;
  const int share = (items + static_cast<int>(gridDim.y) - 1) / static_cast<int>(gridDim.y);
  const int first = static_cast<int>(blockIdx.y) * share;
  const int last = first + share < items ? first + share : items;

  struct Item {
    In x[2];
    void* to;   // null: nothing to write
    int angle;  // of the first pair, -1: a copy
    bool own;   // the row is of the activations' type, not the cache's
  };
  for (int base = first + tid; base < last; base += kRotThreads * kUnroll) {
    Item it[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int item = base + u * kRotThreads;
      it[u].to = nullptr, it[u].angle = -1, it[u].own = true;
      if (item >= last) continue;
      const int t = item / per;
      int r = item % per;
      const int pi = r < n0 ? 0 : r < n0 + n1 ? 1 : 2;
      r -= pi == 0 ? 0 : pi == 1 ? n0 : n0 + n1;
      const RotaryPart& part = a.part[pi];
      const int of = part.rotate ? turns + rest : plain, head = r / of, c = r % of;
      const bool rotated = part.rotate && c < turns;
      // The item's first value in its head.
      const int e = part.rotate && !rotated ? 2 * n + (c - turns) * VEC : c * VEC;
      const int64_t b = seq_of[t], i = in_of[t];
      const T* from = static_cast<const T*>(part.x) + b * part.xs[0] + head * part.xs[1] +
                      i * part.xs[2] + e;
      if (kPaged && pi != 0) {
        const int64_t at = at_of[pi - 1][t];
        if (at < 0) continue;
        it[u].to = static_cast<C*>(part.y) + at + head * a.page_strides[3 * pi - 2] + e;
        it[u].own = false;
      } else {
        it[u].to = static_cast<T*>(part.y) + b * part.ys[0] + head * part.ys[1] + i * part.ys[2] + e;
      }
      it[u].x[0] = *reinterpret_cast<const In*>(from);
      if (rotated) {
        if constexpr (!kInterleaved) it[u].x[1] = *reinterpret_cast<const In*>(from + n);
        it[u].angle = t * n + (kInterleaved ? e / 2 : e);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (it[u].to == nullptr) continue;
      const int at = it[u].angle;
      auto put = [&](auto* out) {
        typedef std::remove_pointer_t<decltype(out)> R;
        Vec<R, VEC> y;
        if (at < 0) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) y.v[i] = convert<R, T>(it[u].x[0].v[i]);
        } else if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float2 w = cs[at + i];
            const float p = static_cast<float>(it[u].x[0].v[2 * i]);
            const float q = static_cast<float>(it[u].x[0].v[2 * i + 1]);
            y.v[2 * i] = static_cast<R>(turned(p, w.x, -(q * w.y)));
            y.v[2 * i + 1] = static_cast<R>(turned(q, w.x, p * w.y));
          }
        } else {
          Vec<R, VEC> z;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float2 w = cs[at + i];
            const float p = static_cast<float>(it[u].x[0].v[i]);
            const float q = static_cast<float>(it[u].x[1].v[i]);
            y.v[i] = static_cast<R>(turned(p, w.x, -(q * w.y)));
            z.v[i] = static_cast<R>(turned(q, w.x, p * w.y));
          }
          *reinterpret_cast<Vec<R, VEC>*>(out + n) = z;
        }
        *reinterpret_cast<Vec<R, VEC>*>(out) = y;
      };
      if (!kPaged || it[u].own) {
        put(static_cast<T*>(it[u].to));
      } else {
        put(static_cast<C*>(it[u].to));
      }
    }
  }
}

template <typename T, typename C, bool kPaged>
const void* rotary_fn(int vec, bool interleaved) {
  auto fn = [&](auto v) {
    constexpr int V = decltype(v)::value;
    return interleaved ? reinterpret_cast<const void*>(rotary_kernel<T, C, V, true, kPaged>)
                       : reinterpret_cast<const void*>(rotary_kernel<T, C, V, false, kPaged>);
  };
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return fn(std::integral_constant<int, 8>{});
  }
  if (vec >= 4) return fn(std::integral_constant<int, 4>{});
  // (Interleaved, a vector holds whole pairs.)
  if (interleaved) return reinterpret_cast<const void*>(rotary_kernel<T, C, 2, true, kPaged>);
  return reinterpret_cast<const void*>(rotary_kernel<T, C, 1, false, kPaged>);
}

}  // namespace

int launch_rotary(RotaryArgs a, int dtype, int cache_dtype, int vec, void* stream) {
  const bool paged = a.table != nullptr;
  const void* fn = nullptr;
  const bool il = a.interleaved != 0;
  if (!paged) {
    fn = dtype == kF32   ? rotary_fn<float, float, false>(vec, il)
         : dtype == kF16 ? rotary_fn<_Float16, _Float16, false>(vec, il)
                         : rotary_fn<__bf16, __bf16, false>(vec, il);
  } else if (dtype == kF32) {
    fn = cache_dtype == kF32   ? rotary_fn<float, float, true>(vec, il)
         : cache_dtype == kF16 ? rotary_fn<float, _Float16, true>(vec, il)
                               : rotary_fn<float, __bf16, true>(vec, il);
  } else {
    fn = dtype == kF16 ? rotary_fn<_Float16, _Float16, true>(vec, il)
                       : rotary_fn<__bf16, __bf16, true>(vec, il);
  }
  // Tokens per workgroup: about two rounds of items per thread, angles within LDS, and no more than
  // leave 1024 workgroups; few tokens share out their items over blockIdx.y.
  const int64_t all = static_cast<int64_t>(a.B) * a.S;
  int64_t per = 0;
  for (const RotaryPart& p : a.part) {
    const int pairs = a.interleaved ? a.pairs : a.pairs / 2;
    per += static_cast<int64_t>(p.heads) * ((p.rotate ? a.D - 2 * a.pairs + 2 * pairs : a.D) / vec);
  }
  if (per == 0) per = 1;
  int64_t tokens = 2 * kUnroll * kRotThreads / per;
  if (a.pairs > 0 && tokens > kMaxAngles / a.pairs) tokens = kMaxAngles / a.pairs;
  if (tokens > kMaxTokens) tokens = kMaxTokens;
  if (tokens > all / 1024) tokens = all / 1024;
  if (tokens < 1) tokens = 1;
  a.tokens = static_cast<int>(tokens);
  const int64_t blocks = (all + tokens - 1) / tokens;
  int64_t shares = (tokens * per + kRotThreads - 1) / kRotThreads;
  const int64_t want = (1024 + blocks - 1) / blocks;
  if (shares > want) shares = want;
  // (A workgroup's share of items stays far inside 32 bits.)
  void* args[] = {&a};
  return static_cast<int>(hipLaunchKernel(fn, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(shares)),
                                          dim3(kRotThreads), args, 0,
                                          static_cast<hipStream_t>(stream)));
}

}  // namespace fattn
