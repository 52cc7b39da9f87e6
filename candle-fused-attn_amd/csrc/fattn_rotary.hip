// Rotary positions, and the append of keys and values to a paged cache with the rotation on the way.
//
// A rotated head has n = dim / 2 pairs of values, (x_i, x_{i + n}) or, interleaved, (x_2i, x_2i+1);
// pair i at position p turns by the angle a = p f_i:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,  c = magnitude cos a,  s = magnitude sin a
// and values past dim stay. The inverse (the gradient) turns by -a with the same magnitude.
//
// Bound: memory, each value read and written once: b 64 s 240 h 6 d 64, q and k turned and v copied, 30 us
// (4.7 TB/s; a large copy 4.9), b 2 s 8191 32 + 8 heads d 128 bf16 66 us (5.1 TB/s), prompts of 16 x 2048
// tokens into pages 150 us (4.6 TB/s); for a few tokens 3.5 to 4.5 us, a launch. A workgroup takes some
// tokens of one operand with all their heads, so that an angle's sine and cosine are formed once per
// token and pair (in LDS) and not once per head; positions need no table in memory and have no largest
// value. (All operands in one workgroup, items found by division, and the loads after the angles: 40, 94
// and 200 us.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "fattn_internal.h"

namespace fattn {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxTokens = 64;    // tokens of a workgroup
constexpr int kMaxAngles = 2048;  // angles of a workgroup (LDS: 8 bytes each)
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

// A workgroup: `tokens` tokens of one operand (blockIdx.y: the operand, and which share of the items). An
// item is VEC pairs of a rotated head in the half layout (two vectors, n apart), else VEC values; a head's
// items follow one another, so a wave moves whole rows. The first items are loaded before the angles
// are formed, over whose latency they come in.
template <typename T, typename C, int VEC, bool kInterleaved, bool kPaged>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[kMaxAngles];
  __shared__ int64_t at_of[kMaxTokens];  // paged: the token's slot, -1: none
  __shared__ int64_t pos_of[kMaxTokens];
  const int tid = threadIdx.x, n = a.pairs;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens, all = static_cast<int64_t>(a.B) * a.S;
  const int nt = static_cast<int>(all - t0 < a.tokens ? all - t0 : a.tokens);
  const int y = static_cast<int>(blockIdx.y);
  const int pi = y < a.first_share[1] ? 0 : y < a.first_share[2] ? 1 : 2;
  const RotaryPart& part = a.part[pi];
  const bool to_pages = kPaged && pi != 0;  // (part 0 is q)
  const bool turns = part.rotate != 0;
  // A head's items: its turned values first, then the copies.
  const int turned_items = kInterleaved ? 2 * n / VEC : n / VEC;
  const int of = a.items[pi], per = of * part.heads, items = nt * per;
  const int shares = a.first_share[pi + 1] - a.first_share[pi];
  const int share = (items + shares - 1) / shares;
  const int first = (y - a.first_share[pi]) * share;
  const int last = first + share < items ? first + share : items;

  typedef Vec<T, VEC> In;
  struct Item {
    In x[2];
    int64_t to;     // (not the pages': the row's offset in y)
    int t, e, head; // token, first value (-1: no item), head
  };
  Item it[kUnroll];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int item = base + u * kRotThreads;
      it[u].e = -1;
      if (item >= last) continue;
      const int t = divide(item, a.by_per[pi]);
      const int r = item - t * per, head = divide(r, a.by_items[pi]), c = r - head * of;
      const int e = turns && c >= turned_items ? 2 * n + (c - turned_items) * VEC : c * VEC;
      const int tok = static_cast<int>(t0) + t, b = divide(tok, a.by_seq), i = tok - b * a.S;
      it[u].t = t, it[u].e = e, it[u].head = head;
      it[u].to = b * part.ys[0] + head * part.ys[1] + i * part.ys[2];
      const T* from = static_cast<const T*>(part.x) + b * part.xs[0] + head * part.xs[1] +
                      i * part.xs[2] + e;
      it[u].x[0] = *reinterpret_cast<const In*>(from);
      if (!kInterleaved && turns && e < n) it[u].x[1] = *reinterpret_cast<const In*>(from + n);
    }
  };
  load(first + tid);

  if (tid < nt) {
    const int tok = static_cast<int>(t0) + tid, b = divide(tok, a.by_seq), i = tok - b * a.S;
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
      const int64_t* st = a.page_strides + (pi == 2 ? 3 : 0);
      at_of[tid] = page >= 0 && page < a.pages ? page * st[0] + p % a.page_size * st[2] : -1;
    } else {
      const int64_t at = b * a.pos_strides[0] + i * a.pos_strides[1];
      p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                  : static_cast<const int32_t*>(a.positions)[at];
    }
    pos_of[tid] = p;
  }
  __syncthreads();
  if (turns) {
    for (int i = tid; i < nt * n; i += kRotThreads) {
      const int t = divide(i, a.by_pairs);
      float2 x = turn(static_cast<double>(pos_of[t]), a.frequencies[i - t * n], a.magnitude);
      if (a.inverse) x.y = -x.y;
      cs[i] = x;
    }
    __syncthreads();
  }

  auto store = [&](auto* base, const Item& x, int64_t at) {
    typedef std::remove_pointer_t<decltype(base)> R;
    R* out = base + at + x.e;
    const float2* w = cs + x.t * n + (kInterleaved ? x.e / 2 : x.e);
    Vec<R, VEC> y;
    if (!turns || x.e >= (kInterleaved ? 2 * n : n)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) y.v[i] = convert<R, T>(x.x[0].v[i]);
    } else if constexpr (kInterleaved) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float p = static_cast<float>(x.x[0].v[2 * i]), q = static_cast<float>(x.x[0].v[2 * i + 1]);
        y.v[2 * i] = static_cast<R>(turned(p, w[i].x, -(q * w[i].y)));
        y.v[2 * i + 1] = static_cast<R>(turned(q, w[i].x, p * w[i].y));
      }
    } else {
      Vec<R, VEC> z;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float p = static_cast<float>(x.x[0].v[i]), q = static_cast<float>(x.x[1].v[i]);
        y.v[i] = static_cast<R>(turned(p, w[i].x, -(q * w[i].y)));
        z.v[i] = static_cast<R>(turned(q, w[i].x, p * w[i].y));
      }
      *reinterpret_cast<Vec<R, VEC>*>(out + n) = z;
    }
    *reinterpret_cast<Vec<R, VEC>*>(out) = y;
  };
  for (int base = first + tid; base < last; base += kRotThreads * kUnroll) {
    if (base != first + tid) load(base);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (it[u].e < 0) continue;
      if (to_pages) {
        const int64_t at = at_of[it[u].t];
        if (at >= 0) store(static_cast<C*>(part.y), it[u], at + it[u].head * a.page_strides[pi == 2 ? 4 : 1]);
      } else {
        store(static_cast<T*>(part.y), it[u], it[u].to);
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
  // Tokens per workgroup: about two rounds of items per thread for the operand of most heads, angles
  // within LDS, and no more than leave 1024 workgroups, but an item for every thread; few tokens share
  // out an operand's items.
  const int64_t all = static_cast<int64_t>(a.B) * a.S;
  int64_t most = 1;
  for (int i = 0; i < 3; ++i) {
    const int turned = a.interleaved ? 2 * a.pairs / vec : a.pairs / vec;
    a.items[i] = a.part[i].rotate ? turned + (a.D - 2 * a.pairs) / vec : a.D / vec;
    most = std::max<int64_t>(most, static_cast<int64_t>(a.items[i]) * a.part[i].heads);
  }
  const int64_t fill = (kRotThreads + most - 1) / most;
  int64_t tokens = std::min(std::max(fill, all / 1024), std::max(fill, 2 * kUnroll * kRotThreads / most));
  if (a.pairs > 0) tokens = std::min<int64_t>(tokens, kMaxAngles / a.pairs);
  tokens = std::min<int64_t>(tokens, kMaxTokens);
  a.tokens = static_cast<int>(tokens);
  const int64_t blocks = (all + tokens - 1) / tokens;
  a.first_share[0] = 0;
  for (int i = 0; i < 3; ++i) {
    const int64_t per = static_cast<int64_t>(a.items[i]) * a.part[i].heads;
    const int64_t rounds = (tokens * per + kRotThreads - 1) / kRotThreads;
    const int64_t shares = std::min(rounds, (512 + blocks - 1) / blocks);
    a.first_share[i + 1] = a.first_share[i] + static_cast<int>(shares);
    a.by_per[i] = divider(per), a.by_items[i] = divider(a.items[i]);
  }
  a.by_seq = divider(a.S), a.by_pairs = divider(a.pairs);
  const int shares = a.first_share[3];
  void* args[] = {&a};
  return static_cast<int>(hipLaunchKernel(fn, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(shares)),
                                          dim3(kRotThreads), args, 0,
                                          static_cast<hipStream_t>(stream)));
}

}  // namespace fattn
