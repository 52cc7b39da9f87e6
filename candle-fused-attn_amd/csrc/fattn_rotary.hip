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

// --- The append to a 4-bit cache ---------------------------------------------------------------------
// 32 values share a scale 2^e, e the least with none of them past 7 2^e (so 6, the largest magnitude, is the
// nearest to each that passes it), and are stored as the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, the even code
// where two are as near: what the conversion instruction gives, times 2^-e. Which code is nearest is decided
// by the exact value: of a rotated key by its value in 64 bits (its angle p f rounded once, reduced in two
// terms of pi / 2), brought to 32 bits by rounding to odd, so that no second rounding moves a value across
// the border between two codes, and a token has the same codes on whatever path it came.
//
// Bound: memory, and for few tokens the launch. A thread has 8 values, so that four neighbours share a scale
// and a head's scales are one word; the values that a rotation pairs with them are read by the neighbours too.

// cos and sin of the angle p f (rounded once), times the magnitude, in 64 bits: less q quarter turns, |y| <=
// pi / 4, where the Taylor series to y^17 and y^16 are exact to 1e-17.
__device__ __forceinline__ double2 turn64(double p, double f, double magnitude) {
  const double a = p * f, q = rint(a * 0.63661977236758134308);
  const double y = fma(q, -6.123233995736766036e-17, fma(q, -1.57079632679489661923, a)), z = y * y;
  double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, z, -1.0 / 1307674368000.0), c = fma(c, z, -1.0 / 87178291200.0);
  s = fma(s, z, 1.0 / 6227020800.0), c = fma(c, z, 1.0 / 479001600.0);
  s = fma(s, z, -1.0 / 39916800.0), c = fma(c, z, -1.0 / 3628800.0);
  s = fma(s, z, 1.0 / 362880.0), c = fma(c, z, 1.0 / 40320.0);
  s = fma(s, z, -1.0 / 5040.0), c = fma(c, z, -1.0 / 720.0);
  s = fma(s, z, 1.0 / 120.0), c = fma(c, z, 1.0 / 24.0);
  s = fma(s, z, -1.0 / 6.0), c = fma(c, z, -0.5);
  s = fma(s * z, y, y), c = fma(c, z, 1.0);
  const int k = static_cast<int>(q - 4.0 * floor(0.25 * q));
  const double cc = (k & 1) ? s : c, ss = (k & 1) ? c : s;
  return double2{((k == 1 || k == 2) ? -cc : cc) * magnitude, (k >= 2 ? -ss : ss) * magnitude};
}
// x in 32 bits, rounded to odd: where it is not exact, towards 0 and with the last bit set.
__device__ __forceinline__ float to_odd(double x) {
  const float r = static_cast<float>(x);
  const double back = static_cast<double>(r);
  if (!(back != x) || x != x) return r;
  const unsigned u = __float_as_uint(r) - (fabs(back) > fabs(x) ? 1u : 0u);
  return __uint_as_float(u | 1u);
}
// Eight values, of a group of 32 that four neighbouring lanes have: their codes, and the group's scale byte.
__device__ __forceinline__ unsigned codes_of(const float (&x)[8], unsigned& scale) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, true)));
  top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x4E, 0xF, 0xF, true)));
  // (1.m 2^E <= 7 2^(E - 2) up to 1.75.)
  const int e = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  const bool finite = top < 0x7f800000u;
  scale = finite ? static_cast<unsigned>(max(e, 0)) : 255u;
  const float s = __uint_as_float(scale << 23);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  // No negative zeros: a token has one code for 0.
  const unsigned some = (w | w >> 1 | w >> 2) & 0x11111111u;
  w &= 0x77777777u | some << 3;
  return finite ? w : 0u;
}

constexpr int kMaxAngles64 = 1024;

// As rotary_kernel, an item 8 values of a head: of part 0 (q) written turned, of parts 1 and 2 as codes.
// kWide: an operand's values are moved 8 at a time.
template <typename T, bool kWide, bool kInterleaved>
__global__ void __launch_bounds__(kRotThreads) append_four_kernel(RotaryArgs a) {
  __shared__ double2 cs[kMaxAngles64];
  __shared__ int64_t at_of[kMaxTokens];
  __shared__ int pos_of[kMaxTokens];
  const int tid = threadIdx.x, n = a.pairs, D = a.D;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens, all = static_cast<int64_t>(a.B) * a.S;
  const int nt = static_cast<int>(all - t0 < a.tokens ? all - t0 : a.tokens);
  const int y = static_cast<int>(blockIdx.y);
  const int pi = y < a.first_share[1] ? 0 : y < a.first_share[2] ? 1 : 2;
  const RotaryPart& part = a.part[pi];
  const bool turns = part.rotate != 0 && n > 0;
  const int of = a.items[pi], per = of * part.heads, items = nt * per;
  const int shares = a.first_share[pi + 1] - a.first_share[pi];
  const int share = (items / of + shares - 1) / shares * of;  // (whole heads)
  const int first = (y - a.first_share[pi]) * share;
  const int last = first + share < items ? first + share : items;
  constexpr int kInFlight = 2;

  struct Item {
    T x[8], z[8];  // the values, and those that they turn with
    int64_t to;
    int t, e, head, low;  // token, first value (-1: no item), head; low: (half layout) the first of the pairs
  };
  Item it[kInFlight];
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int item = base + u * kRotThreads;
      it[u].e = -1;
      if (item >= last) continue;
      const int t = divide(item, a.by_per[pi]);
      const int r = item - t * per, head = divide(r, a.by_items[pi]), e = 8 * (r - head * of);
      const int tok = static_cast<int>(t0) + t, b = divide(tok, a.by_seq), i = tok - b * a.S;
      it[u].t = t, it[u].e = e, it[u].head = head;
      it[u].to = pi == 0 ? b * part.ys[0] + head * part.ys[1] + i * part.ys[2] : 0;
      const T* row = static_cast<const T*>(part.x) + b * part.xs[0] + head * part.xs[1] + i * part.xs[2];
      if constexpr (kWide) {
        typedef Vec<T, 16 / sizeof(T)> In;
        constexpr int kIn = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += kIn) {
          const In x = *reinterpret_cast<const In*>(row + e + k);
#pragma unroll
          for (int c = 0; c < kIn; ++c) it[u].x[k + c] = x.v[c];
        }
        if (!kInterleaved && turns && e < 2 * n) {
          const T* other = row + (e < n ? e + n : e - n);
#pragma unroll
          for (int k = 0; k < 8; k += kIn) {
            const In x = *reinterpret_cast<const In*>(other + k);
#pragma unroll
            for (int c = 0; c < kIn; ++c) it[u].z[k + c] = x.v[c];
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int c = e + k;
          it[u].x[k] = row[c];
          if (!kInterleaved && turns && c < 2 * n) it[u].z[k] = row[c < n ? c + n : c - n];
        }
      }
    }
  };
  load(first + tid);

  if (tid < nt) {
    const int tok = static_cast<int>(t0) + tid, b = divide(tok, a.by_seq), i = tok - b * a.S;
    const int held = a.lengths[b];
    const int64_t p = static_cast<int64_t>(held) + i;
    // (As in rotary_kernel.)
    int64_t page = -1;
    const bool counted = a.counts == nullptr || i < a.counts[b];
    if (counted && held >= 0 && p / a.page_size < a.table_width) {
      page = a.table[b * a.table_stride + p / a.page_size];
    }
    const int64_t* st = a.page_strides + (pi == 2 ? 3 : 0);
    at_of[tid] = page >= 0 && page < a.pages ? page * st[0] + p % a.page_size * st[2] : -1;
    pos_of[tid] = held;
  }
  __syncthreads();
  // Angles: q's in 32 bits, as fused_rotary's.
  float2* cs32 = reinterpret_cast<float2*>(cs);
  if (turns) {
    for (int i = tid; i < nt * n; i += kRotThreads) {
      const int t = divide(i, a.by_pairs);
      const int tok = static_cast<int>(t0) + t, b = divide(tok, a.by_seq);
      const double p = static_cast<double>(static_cast<int64_t>(pos_of[t]) + (tok - b * a.S));
      const double f = a.frequencies[i - t * n];
      if (pi == 0) {
        cs32[i] = turn(p, f, a.magnitude);
      } else {
        cs[i] = turn64(p, f, a.magnitude);
      }
    }
    __syncthreads();
  }

  // fn(k, value, its partner, whether it is the first of the pair, its pair) of an item's turned values.
  auto each = [&](const Item& x, auto turned_value, auto plain_value) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = x.e + k;
      if (!turns || c >= 2 * n) {
        plain_value(k);
      } else if (kInterleaved) {
        turned_value(k, x.x[k], x.x[k ^ 1], (k & 1) == 0, x.t * n + c / 2);
      } else {
        turned_value(k, x.x[k], x.z[k], c < n, x.t * n + (c < n ? c : c - n));
      }
    }
  };
  for (int base = first + tid; base < last; base += kRotThreads * kInFlight) {
    if (base != first + tid) load(base);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const Item& x = it[u];
      if (x.e < 0) continue;
      if (pi == 0) {
        T out[8];
        each(
            x,
            [&](int k, T v, T o, bool low, int at) {
              const float2 w = cs32[at];
              const float fv = static_cast<float>(v), fo = static_cast<float>(o);
              out[k] = static_cast<T>(turned(fv, w.x, low ? -(fo * w.y) : fo * w.y));
            },
            [&](int k) { out[k] = x.x[k]; });
        T* to = static_cast<T*>(part.y) + x.to + x.e;
        if constexpr (kWide) {
          constexpr int kOut = 16 / sizeof(T);
#pragma unroll
          for (int k = 0; k < 8; k += kOut) {
            Vec<T, kOut> v;
#pragma unroll
            for (int c = 0; c < kOut; ++c) v.v[c] = out[k + c];
            *reinterpret_cast<Vec<T, kOut>*>(to + k) = v;
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) to[k] = out[k];
        }
      } else {
        float v[8];
        each(
            x,
            [&](int k, T p, T o, bool low, int at) {
              const double2 w = cs[at];
              const double dp = static_cast<double>(static_cast<float>(p));
              const double dq = static_cast<double>(static_cast<float>(o)) * w.y;
              v[k] = to_odd(fma(dp, w.x, low ? -dq : dq));
            },
            [&](int k) { v[k] = static_cast<float>(x.x[k]); });
        unsigned scale;
        const unsigned codes = codes_of(v, scale);
        // The head's scale bytes, in order, from its groups' lanes.
        unsigned word = scale << (x.e / 32 * 8);
        if (D >= 64) word |= static_cast<unsigned>(__shfl_xor(static_cast<int>(word), 4));
        if (D == 128) word |= static_cast<unsigned>(__shfl_xor(static_cast<int>(word), 8));
        const int64_t at = at_of[x.t];
        if (at >= 0) {
          unsigned char* row = static_cast<unsigned char*>(part.y) + at + x.head * a.page_strides[pi == 2 ? 4 : 1];
          *reinterpret_cast<unsigned*>(row + x.e / 2) = codes;
          if (x.e == 0) *reinterpret_cast<unsigned*>(row + D / 2) = word;
        }
      }
    }
  }
}

// --- Tokens back out of a paged cache ------------------------------------------------------------------
// Bound: memory, each row read and each result written once. A thread has 8 values of a token's head; the
// results of one (sample, head) are contiguous, and those of neighbouring tokens lie in one page, so a wave
// reads and writes whole rows one after the other.
template <typename C, typename O, int D>
__global__ void __launch_bounds__(256) read_kernel(PagedReadArgs a) {
  constexpr int kOf = D / 8, kInFlight = 4;
  const int pair = static_cast<int>(blockIdx.x) / a.blocks, in = static_cast<int>(blockIdx.x) - pair * a.blocks;
  const int b = pair / a.HK, head = pair - b * a.HK, which = static_cast<int>(blockIdx.y);
  const int64_t* st = which == 0 ? a.ks : a.vs;
  const C* pages = static_cast<const C*>(which == 0 ? a.k_pages : a.v_pages) + head * st[1];
  O* out = static_cast<O*>(which == 0 ? a.k : a.v) + static_cast<int64_t>(pair) * a.S * D;
  const int len = a.lengths[b];
  const int64_t start = a.starts != nullptr ? a.starts[b] : 0;
  const int item0 = in * (256 * kInFlight) + static_cast<int>(threadIdx.x), items = a.S * kOf;
  const C* row[kInFlight];  // (null: zeros; with `bad`: NaN)
  bool bad[kInFlight];
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) {
    const int item = item0 + 256 * u;
    row[u] = nullptr, bad[u] = false;
    const int64_t t = start + item / kOf;
    if (item >= items || t < 0 || t >= len) continue;
    const int at = divide(static_cast<int>(t), a.by_page);
    bad[u] = true;
    if (at >= a.table_width) continue;
    const int page = a.table[b * a.table_stride + at];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) continue;
    bad[u] = false;
    row[u] = pages + page * st[0] + (static_cast<int>(t) - at * a.page_size) * st[2];
  }
  struct alignas(16) Values {
    C v[8];
  };
  struct Codes {
    unsigned w, scale;
  };
  std::conditional_t<std::is_same<C, four>::value, Codes, Values> x[kInFlight];
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) {
    const int e = (item0 + 256 * u) % kOf * 8;
    if (row[u] == nullptr) continue;
    if constexpr (std::is_same<C, four>::value) {
      const char* p = reinterpret_cast<const char*>(row[u]);
      x[u].w = *reinterpret_cast<const unsigned*>(p + e / 2);
      x[u].scale = *reinterpret_cast<const unsigned char*>(p + D / 2 + e / 32);
    } else {
      x[u] = *reinterpret_cast<const Values*>(row[u] + e);
    }
  }
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) {
    const int item = item0 + 256 * u;
    if (item >= items) continue;
    struct alignas(16) Out {
      O v[8];
    } y;
    if (row[u] == nullptr) {
      const O z = static_cast<O>(bad[u] ? __builtin_nanf("") : 0.0f);
#pragma unroll
      for (int k = 0; k < 8; ++k) y.v[k] = z;
    } else if constexpr (std::is_same<C, four>::value) {
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      const float s = __uint_as_float(x[u].scale << 23);
      const b2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x[u].w, s, 0),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x[u].w, s, 1),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x[u].w, s, 2),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x[u].w, s, 3)};
#pragma unroll
      for (int k = 0; k < 8; ++k) y.v[k] = convert<O, __bf16>(p[k / 2][k % 2]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) y.v[k] = convert<O, C>(x[u].v[k]);
    }
    *reinterpret_cast<Out*>(out + static_cast<int64_t>(item) * 8) = y;
  }
}

template <typename C, typename O>
const void* read_fn(int d) {
  return d == 32    ? reinterpret_cast<const void*>(read_kernel<C, O, 32>)
         : d == 128 ? reinterpret_cast<const void*>(read_kernel<C, O, 128>)
                    : reinterpret_cast<const void*>(read_kernel<C, O, 64>);
}
template <typename C>
const void* read_fn(int dtype, int d) {
  return dtype == kF16 ? read_fn<C, _Float16>(d) : dtype == kBF16 ? read_fn<C, __bf16>(d) : read_fn<C, float>(d);
}

template <typename T>
const void* append_four_fn(bool wide, bool interleaved) {
  return wide ? (interleaved ? reinterpret_cast<const void*>(append_four_kernel<T, true, true>)
                             : reinterpret_cast<const void*>(append_four_kernel<T, true, false>))
              : (interleaved ? reinterpret_cast<const void*>(append_four_kernel<T, false, true>)
                             : reinterpret_cast<const void*>(append_four_kernel<T, false, false>));
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
  const bool paged = a.table != nullptr, to_four = cache_dtype == kFP4;
  const void* fn = nullptr;
  const bool il = a.interleaved != 0;
  if (to_four) {
    const bool wide = vec == 8;
    fn = dtype == kF32   ? append_four_fn<float>(wide, il)
         : dtype == kF16 ? append_four_fn<_Float16>(wide, il)
                         : append_four_fn<__bf16>(wide, il);
    vec = 8;
  } else if (!paged) {
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
    a.items[i] = a.part[i].rotate && !to_four ? turned + (a.D - 2 * a.pairs) / vec : a.D / vec;
    most = std::max<int64_t>(most, static_cast<int64_t>(a.items[i]) * a.part[i].heads);
  }
  const int64_t fill = (kRotThreads + most - 1) / most;
  int64_t tokens = std::min(std::max(fill, all / 1024), std::max(fill, 2 * kUnroll * kRotThreads / most));
  if (a.pairs > 0) tokens = std::min<int64_t>(tokens, (to_four ? kMaxAngles64 : kMaxAngles) / a.pairs);
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

int launch_paged_read(PagedReadArgs a, int cache_dtype, int dtype, int d, void* stream) {
  const void* fn = cache_dtype == kF32    ? read_fn<float>(dtype, d)
                   : cache_dtype == kF16  ? read_fn<_Float16>(dtype, d)
                   : cache_dtype == kBF16 ? read_fn<__bf16>(dtype, d)
                                          : read_fn<four>(dtype, d);
  a.blocks = static_cast<int>(paged_read_blocks(a.S, d));
  a.by_page = divider(a.page_size);
  void* args[] = {&a};
  return static_cast<int>(hipLaunchKernel(fn, dim3(static_cast<unsigned>(a.B) * a.HK * a.blocks, 2), dim3(256),
                                          args, 0, static_cast<hipStream_t>(stream)));
}
int64_t paged_read_blocks(int64_t s, int64_t d) { return (s * (d / 8) + 1023) / 1024; }

}  // namespace fattn
