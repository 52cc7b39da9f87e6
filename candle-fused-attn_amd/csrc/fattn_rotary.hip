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
// 32 bits decide nearly every code: with the bound on what they are off by, both ends of a value's interval have
// the same one. Only where that leaves a doubt (an item of a wave in some hundreds; a group of values below 2^-100, all
// zeros among them; any turned by a magnitude below 2^-100) is it formed in 64.
//
// Bound: memory, and for few tokens the launch. A thread has 16 values, in two halves that turn together, so that
// four neighbours share a scale, a head's scales are one word and each value is read once. 16 x 2048 tokens, 32
// + 8 heads d 128 bf16, into pages: 139 to 147 us (4.7 TB/s; all codes in 64 bits 8 values at a time 200; four items in
// flight for two 179; queries in a launch of their own 198); 64 single tokens of 6 + 6 heads fp32 d 64 5.6 us.

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
// Of a group of 32 values that four neighbouring lanes have eight each of, the bits of whose largest magnitude
// are `top`: over all four.
__device__ __forceinline__ unsigned group_top(unsigned top) {
  top = max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, true)));
  return max(top, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x4E, 0xF, 0xF, true)));
}
__device__ __forceinline__ unsigned bits_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// Its scale byte (1.m 2^E <= 7 2^(E - 2) up to 1.75), 255 where a value is not finite.
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
  const int e = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return top < 0x7f800000u ? static_cast<unsigned>(max(e, 0)) : 255u;
}
// The eight's codes under it, no negative zeros among them (a token has one code for 0).
__device__ __forceinline__ unsigned codes_of(const float (&x)[8], unsigned scale) {
  const float s = __uint_as_float(scale << 23);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  const unsigned some = (w | w >> 1 | w >> 2) & 0x11111111u;
  w &= 0x77777777u | some << 3;
  return scale != 255u ? w : 0u;
}
// The same, and the scale they take.
__device__ __forceinline__ unsigned scaled_codes(const float (&x)[8], unsigned& scale) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, bits_of(x[i]));
  scale = scale_byte(group_top(top));
  return codes_of(x, scale);
}
// Codes of values that are within `off` of x, and whether these decide them: the same scale and codes at both
// ends (and no overflow, nor values among the least, where `off` does not hold).
__device__ __forceinline__ unsigned codes_within(const float (&x)[8], const float (&off)[8], unsigned& scale,
                                                 bool& sure) {
  float lo[8], hi[8];
  unsigned most = 0, least = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = x[i] - off[i], hi[i] = x[i] + off[i];
    most = max(most, bits_of(fabsf(x[i]) + off[i]));
    least = max(least, __float_as_uint(fmaxf(fabsf(x[i]) - off[i], 0.0f)));
  }
  most = group_top(most), least = group_top(least);
  scale = scale_byte(most);
  const unsigned w = codes_of(lo, scale);
  sure = scale == scale_byte(least) && w == codes_of(hi, scale) && most < 0x7f800000u && most > 0x0d800000u;
  return w;
}

// What a workgroup of an append has: `nt` tokens from t0 of operand pi (as rotary_kernel's), items first ..
// last (whole heads), where its tokens go and their angles.
struct AppendBlock {
  int64_t t0;
  int nt, pi, of, per, first, last;
  bool turns;
  __device__ __forceinline__ explicit AppendBlock(const RotaryArgs& a) {
    const int64_t all = static_cast<int64_t>(a.B) * a.S;
    t0 = static_cast<int64_t>(blockIdx.x) * a.tokens;
    nt = static_cast<int>(all - t0 < a.tokens ? all - t0 : a.tokens);
    const int y = static_cast<int>(blockIdx.y);
    pi = y < a.first_share[1] ? 0 : y < a.first_share[2] ? 1 : 2;
    turns = a.part[pi].rotate != 0 && a.pairs > 0;
    of = a.items[pi], per = of * a.part[pi].heads;
    const int items = nt * per, shares = a.first_share[pi + 1] - a.first_share[pi];
    const int share = (items / of + shares - 1) / shares * of;
    first = (y - a.first_share[pi]) * share;
    last = first + share < items ? first + share : items;
  }
};
struct AppendSmem {
  float2 cs[kMaxAngles];
  int64_t at_of[kMaxTokens];  // the token's slot, -1: none
  int pos_of[kMaxTokens];     // what its sequence holds before
};
__device__ __forceinline__ void append_tokens(const RotaryArgs& a, const AppendBlock& k, AppendSmem& sm) {
  const int tid = threadIdx.x, n = a.pairs;
  if (tid < k.nt) {
    const int tok = static_cast<int>(k.t0) + tid, b = divide(tok, a.by_seq), i = tok - b * a.S;
    const int held = a.lengths[b];
    const int64_t p = static_cast<int64_t>(held) + i;
    // (As in rotary_kernel.)
    int64_t page = -1;
    const bool counted = a.counts == nullptr || i < a.counts[b];
    if (counted && held >= 0 && p / a.page_size < a.table_width) {
      page = a.table[b * a.table_stride + p / a.page_size];
    }
    const int64_t* st = a.page_strides + (k.pi == 2 ? 3 : 0);
    sm.at_of[tid] = page >= 0 && page < a.pages ? page * st[0] + p % a.page_size * st[2] : -1;
    sm.pos_of[tid] = held;
  }
  __syncthreads();
  if (!k.turns) return;
  for (int i = tid; i < k.nt * n; i += kRotThreads) {
    const int t = divide(i, a.by_pairs);
    const int tok = static_cast<int>(k.t0) + t, b = divide(tok, a.by_seq);
    const double p = static_cast<double>(static_cast<int64_t>(sm.pos_of[t]) + (tok - b * a.S));
    const double f = a.frequencies[i - t * n];
    if (k.pi == 0) {  // (q's as fused_rotary's)
      sm.cs[i] = turn(p, f, a.magnitude);
    } else {
      const double2 w = turn64(p, f, a.magnitude);
      sm.cs[i] = float2{static_cast<float>(w.x), static_cast<float>(w.y)};
    }
  }
  __syncthreads();
}
// The position of the block's token t.
__device__ __forceinline__ double position_of(const RotaryArgs& a, const AppendBlock& k, const AppendSmem& sm, int t) {
  const int tok = static_cast<int>(k.t0) + t, b = divide(tok, a.by_seq);
  return static_cast<double>(static_cast<int64_t>(sm.pos_of[t]) + (tok - b * a.S));
}
// Eight values to 16-byte aligned memory.
template <typename T>
__device__ __forceinline__ void put8(T* to, const T (&x)[8]) {
  constexpr int kOut = 16 / sizeof(T);
#pragma unroll
  for (int k = 0; k < 8; k += kOut) {
    Vec<T, kOut> v;
#pragma unroll
    for (int c = 0; c < kOut; ++c) v.v[c] = x[k + c];
    *reinterpret_cast<Vec<T, kOut>*>(to + k) = v;
  }
}
template <typename T>
__device__ __forceinline__ void get8(T (&x)[8], const T* from) {
  constexpr int kIn = 16 / sizeof(T);
#pragma unroll
  for (int k = 0; k < 8; k += kIn) {
    const Vec<T, kIn> v = *reinterpret_cast<const Vec<T, kIn>*>(from + k);
#pragma unroll
    for (int c = 0; c < kIn; ++c) x[k + c] = v.v[c];
  }
}
// Eight values of a key, y = x c + z s (w(k): c, and s with z's sign), as codes, formed in 32 bits: off by 3 x
// 2^-24 of |x| + |z| at most, times the magnitude; `bound(k)`: 2^-21 of that, or 0 of values that are not turned (c
// 1, s 0 and z of the same scale: y is x, and in doubt it would be at every border, where 1 of 90 bf16 values lies).
// `sure`: that leaves no code in doubt. A scale's four lanes come here together, since they exchange its largest
// magnitude: a branch that some of them take would hide the others' values.
// (Of a magnitude below 2^-100 the bound and the factors lose their bits: nothing is sure.)
constexpr float kLeastBound = 0x1p-121f;
template <typename T, typename B, typename W>
__device__ __forceinline__ unsigned turned_codes(const T (&x)[8], const T (&z)[8], B bound, W w, unsigned& scale,
                                                 bool& sure) {
  float v[8], off[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 c = w(k);
    const float fx = static_cast<float>(x[k]), fz = static_cast<float>(z[k]);
    v[k] = fmaf(fx, c.x, fz * c.y);
    off[k] = (fabsf(fx) + fabsf(fz)) * bound(k);
  }
  bool here;
  const unsigned codes = codes_within(v, off, scale, here);
  sure = sure && here;
  return codes;
}
// Value c of a turned head: its pair (-1: not turned), whether it is the pair's first, the other's place.
template <bool kInterleaved>
struct Pairing {
  int pair, other;
  bool low;
  __device__ __forceinline__ Pairing(int c, int n, bool turns) {
    pair = !turns || c >= 2 * n ? -1 : kInterleaved ? c / 2 : c < n ? c : c - n;
    low = kInterleaved ? c % 2 == 0 : c < n;
    other = pair < 0 ? c : kInterleaved ? (low ? c + 1 : c - 1) : low ? c + n : c - n;
  }
};
// The codes of values e .. e + 7 of the block's token t, formed in 64 bits.
template <typename T, bool kInterleaved>
__device__ __forceinline__ unsigned exact_codes(const RotaryArgs& a, const AppendBlock& blk, const AppendSmem& sm,
                                                int t, const T* row, int e, unsigned& scale) {
  const double p = position_of(a, blk, sm, t);
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const Pairing<kInterleaved> at(e + k, a.pairs, blk.turns);
    const float x = static_cast<float>(row[e + k]);
    v[k] = x;
    if (at.pair >= 0) {
      const double2 c = turn64(p, a.frequencies[at.pair], a.magnitude);
      const double z = static_cast<double>(static_cast<float>(row[at.other])) * c.y;
      v[k] = to_odd(fma(static_cast<double>(x), c.x, at.low ? -z : z));
    }
    __builtin_amdgcn_sched_barrier(0);  // (one after the other: registers)
  }
  return scaled_codes(v, scale);
}
template <typename T>
__device__ __forceinline__ unsigned plain_codes(const T (&x)[8], unsigned& scale) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = static_cast<float>(x[k]);
  return scaled_codes(v, scale);
}

// An item: 8 values from e and 8 from e + gap on of one head: of the turned part, in the half layout, those that
// turn together (gap n); of the rest, or of a head that is not turned or turned in neighbours, its halves.
// Four neighbours have a scale's values: in the half layout every part's half is a multiple of 32; in
// neighbours the turned part may end within a scale, and its lanes, whose eight values are turned or not, go one
// way. All is moved 16 bytes at a time.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kRotThreads)
append_four_kernel(RotaryArgs a) {
  __shared__ AppendSmem sm;
  const AppendBlock blk(a);
  const RotaryPart& part = a.part[blk.pi];
  const int n = a.pairs, D = a.D, pi = blk.pi;
  const bool halves = !kInterleaved && blk.turns;  // the turned part's halves turn together
  constexpr int kInFlight = 2;
  struct Item {
    T x[8], z[8];
    int64_t to;
    int t, e, head, gap;  // e -1: no item
  };
  Item it[kInFlight];
  // An item's token, head, first value and gap; its row.
  auto place = [&](int item, int& t, int& head, int& e, int& gap) {
    t = divide(item, a.by_per[pi]);
    const int r = item - t * blk.per;
    head = divide(r, a.by_items[pi]);
    e = 8 * (r - head * blk.of), gap = D / 2;
    if (halves) {
      const bool rest = e >= n;
      gap = rest ? D / 2 - n : n;
      e += rest ? n : 0;
    }
  };
  auto row_of = [&](int t, int head, int64_t& to) {
    const int tok = static_cast<int>(blk.t0) + t, b = divide(tok, a.by_seq), i = tok - b * a.S;
    to = pi == 0 ? b * part.ys[0] + head * part.ys[1] + i * part.ys[2] : 0;
    return static_cast<const T*>(part.x) + b * part.xs[0] + head * part.xs[1] + i * part.xs[2];
  };
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int item = base + u * kRotThreads;
      it[u].e = -1;
      if (item >= blk.last) continue;
      place(item, it[u].t, it[u].head, it[u].e, it[u].gap);
      const T* row = row_of(it[u].t, it[u].head, it[u].to) + it[u].e;
      get8(it[u].x, row);
      get8(it[u].z, row + it[u].gap);
    }
  };
  load(blk.first + static_cast<int>(threadIdx.x));
  append_tokens(a, blk, sm);
  const float bound = fabsf(static_cast<float>(a.magnitude)) * 0x1p-21f;

  // Sixteen values, turned where they are turned, of q.
  auto put_q = [&](const Item& x) {
    T* to = static_cast<T*>(part.y) + x.to + x.e;
    T y[8], w[8];
    const float2* cs = sm.cs + x.t * n + x.e;
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = x.x[k], w[k] = x.z[k];
    if (halves && x.e < n) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float p = static_cast<float>(x.x[k]), q = static_cast<float>(x.z[k]);
        y[k] = static_cast<T>(turned(p, cs[k].x, -(q * cs[k].y)));
        w[k] = static_cast<T>(turned(q, cs[k].x, p * cs[k].y));
      }
    } else if (kInterleaved && blk.turns) {
      auto pairs = [&](T (&y)[8], int e) {
        if (e >= 2 * n) return;
        const float2* cs = sm.cs + x.t * n + e / 2;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = static_cast<float>(y[2 * k]), q = static_cast<float>(y[2 * k + 1]);
          y[2 * k] = static_cast<T>(turned(p, cs[k].x, -(q * cs[k].y)));
          y[2 * k + 1] = static_cast<T>(turned(q, cs[k].x, p * cs[k].y));
        }
      };
      pairs(y, x.e);
      pairs(w, x.e + x.gap);
    }
    put8(to, y);
    put8(to + x.gap, w);
  };
  // Codes and scales of a key's or value's item.
  auto put = [&](int t, int head, int e, int gap, unsigned cx, unsigned cz, unsigned sx, unsigned sz) {
    unsigned word = sx << (e / 32 * 8) | sz << ((e + gap) / 32 * 8);
    // (The head's scale bytes, in order, from its groups' lanes.)
    if (D == 128) word |= static_cast<unsigned>(__shfl_xor(static_cast<int>(word), 4));
    unsigned char* row =
        static_cast<unsigned char*>(part.y) + sm.at_of[t] + head * a.page_strides[pi == 2 ? 4 : 1];
    *reinterpret_cast<unsigned*>(row + e / 2) = cx;
    *reinterpret_cast<unsigned*>(row + (e + gap) / 2) = cz;
    if (e == 0) *reinterpret_cast<unsigned*>(row + D / 2) = word;
  };
  auto put_codes = [&](const Item& x) {
    unsigned cx, cz, sx, sz;
    bool sure = !blk.turns || bound >= kLeastBound;
    const float2* cs = sm.cs + x.t * n;
    if (halves && x.e < n) {
      cs += x.e;
      auto off = [&](int) { return bound; };
      cx = turned_codes(x.x, x.z, off, [&](int k) { return float2{cs[k].x, -cs[k].y}; }, sx, sure);
      cz = turned_codes(x.z, x.x, off, [&](int k) { return cs[k]; }, sz, sure);
    } else if (kInterleaved && blk.turns) {
      auto pairs = [&](const T (&y)[8], int e, unsigned& scale) {
        const bool in = e < 2 * n;
        if (n % 16 == 0 && !in) return plain_codes(y, scale);  // (no scale has both: four lanes alike)
        T other[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) other[k] = y[k ^ 1];
        return turned_codes(
            y, other, [&](int) { return in ? bound : 0.0f; },
            [&](int k) {
              const float2 w = in ? cs[(e + k) / 2] : float2{1.0f, 0.0f};
              return k % 2 == 0 ? float2{w.x, -w.y} : w;
            },
            scale, sure);
      };
      cx = pairs(x.x, x.e, sx);
      cz = pairs(x.z, x.e + x.gap, sz);
    } else {
      cx = plain_codes(x.x, sx);
      cz = plain_codes(x.z, sz);
    }
    const bool done = __builtin_amdgcn_ballot_w64(!sure) == 0;
    if (done) put(x.t, x.head, x.e, x.gap, cx, cz, sx, sz);
    return done;
  };
  for (int base = blk.first + static_cast<int>(threadIdx.x); base < blk.last; base += kRotThreads * kInFlight) {
    if (base != blk.first + static_cast<int>(threadIdx.x)) load(base);
    unsigned doubt = 0;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (it[u].e < 0) continue;
      if (pi == 0) {
        put_q(it[u]);
      } else if (sm.at_of[it[u].t] >= 0) {  // (a token's lanes alike)
        if (!put_codes(it[u])) doubt |= 1u << u;
      }
    }
    // What is in doubt (an item of a wave in some hundreds) once more, in 64 bits.
#pragma clang loop unroll(disable)
    for (int u = 0; doubt != 0; ++u, doubt >>= 1) {
      if ((doubt & 1u) == 0) continue;
      int t, head, e, gap;
      int64_t to;
      place(base + u * kRotThreads, t, head, e, gap);
      const T* row = row_of(t, head, to);
      unsigned codes[2], scale[2];
#pragma clang loop unroll(disable)
      for (int i = 0; i < 2; ++i) {
        unsigned s;
        const unsigned c = exact_codes<T, kInterleaved>(a, blk, sm, t, row, e + i * gap, s);
        (i == 0 ? codes[0] : codes[1]) = c, (i == 0 ? scale[0] : scale[1]) = s;
      }
      put(t, head, e, gap, codes[0], codes[1], scale[0], scale[1]);
    }
  }
}

// The same for every other head, rotation and alignment (d 32, half layouts whose parts are no whole scales twice): an
// item 8 values, moved one by one, which is what bounds it. 16 x 2048 tokens, 32 + 8 heads, bf16, half layout: d 32 130
// us (1.4 TB/s), d 64 with 32 turned 290 (1.2 TB/s), d 128 with 96 571; f32 224, 385 and 814.
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kRotThreads)
append_four_any_kernel(RotaryArgs a) {
  __shared__ AppendSmem sm;
  const AppendBlock blk(a);
  const RotaryPart& part = a.part[blk.pi];
  const int n = a.pairs, D = a.D, pi = blk.pi;
  append_tokens(a, blk, sm);
  const float bound = fabsf(static_cast<float>(a.magnitude)) * 0x1p-21f;
  for (int item = blk.first + static_cast<int>(threadIdx.x); item < blk.last; item += kRotThreads) {
    const int t = divide(item, a.by_per[pi]);
    const int r = item - t * blk.per, head = divide(r, a.by_items[pi]), e = 8 * (r - head * blk.of);
    if (pi != 0 && sm.at_of[t] < 0) continue;
    const int tok = static_cast<int>(blk.t0) + t, b = divide(tok, a.by_seq), i = tok - b * a.S;
    const T* row = static_cast<const T*>(part.x) + b * part.xs[0] + head * part.xs[1] + i * part.xs[2];
    T x[8], z[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const Pairing<kInterleaved> p(e + k, n, blk.turns);
      x[k] = row[e + k];
      z[k] = p.pair < 0 ? static_cast<T>(0.0f) : row[p.other];
    }
    auto w = [&](int k) {
      const Pairing<kInterleaved> p(e + k, n, blk.turns);
      if (p.pair < 0) return float2{1.0f, 0.0f};
      const float2 c = sm.cs[t * n + p.pair];
      return float2{c.x, p.low ? -c.y : c.y};
    };
    if (pi == 0) {
      T* to = static_cast<T*>(part.y) + b * part.ys[0] + head * part.ys[1] + i * part.ys[2] + e;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 c = w(k);
        to[k] = !blk.turns || e + k >= 2 * n
                    ? x[k]
                    : static_cast<T>(turned(static_cast<float>(x[k]), c.x, static_cast<float>(z[k]) * c.y));
      }
      continue;
    }
    unsigned scale, codes;
    bool sure = bound >= kLeastBound;
    if (blk.turns) {
      auto off = [&](int k) { return Pairing<kInterleaved>(e + k, n, true).pair < 0 ? 0.0f : bound; };
      codes = turned_codes(x, z, off, w, scale, sure);
      if (__builtin_amdgcn_ballot_w64(!sure) != 0) {
        codes = exact_codes<T, kInterleaved>(a, blk, sm, t, row, e, scale);
      }
    } else {
      codes = plain_codes(x, scale);
    }
    unsigned word = scale << (e / 32 * 8);
    if (D >= 64) word |= static_cast<unsigned>(__shfl_xor(static_cast<int>(word), 4));
    if (D == 128) word |= static_cast<unsigned>(__shfl_xor(static_cast<int>(word), 8));
    unsigned char* to = static_cast<unsigned char*>(part.y) + sm.at_of[t] + head * a.page_strides[pi == 2 ? 4 : 1];
    *reinterpret_cast<unsigned*>(to + e / 2) = codes;
    if (e == 0) *reinterpret_cast<unsigned*>(to + D / 2) = word;
  }
}

// --- Tokens back out of a paged cache ------------------------------------------------------------------
// Bound: memory, each row read and each result written once. A thread has 8 values of a token's head; the
// results of one (sample, head) are contiguous, and those of neighbouring tokens lie in one page, so a wave
// reads and writes whole rows one after the other. Results are stored past the caches, which they would sweep. 4
// x 8 heads 20000 to 32767 tokens of 4 bits to bf16, d 128: 157 us a call, 4.2 TB/s (the kernel itself 88: what
// it wrote drains behind it); 5 x 12 heads 333 tokens f16 d 32 4.4 us.
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
    O* to = out + static_cast<int64_t>(item) * 8;
    typedef unsigned w4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(O)) / 2; ++i) {
      w4 v;
      __builtin_memcpy(&v, reinterpret_cast<const char*>(&y) + 16 * i, 16);
      __builtin_nontemporal_store(v, reinterpret_cast<w4*>(to) + i);
    }
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
const void* append_four_fn(bool pairs, bool interleaved) {
  return pairs ? (interleaved ? reinterpret_cast<const void*>(append_four_kernel<T, true>)
                              : reinterpret_cast<const void*>(append_four_kernel<T, false>))
               : (interleaved ? reinterpret_cast<const void*>(append_four_any_kernel<T, true>)
                              : reinterpret_cast<const void*>(append_four_any_kernel<T, false>));
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
    const bool pairs = vec == 16;
    fn = dtype == kF32   ? append_four_fn<float>(pairs, il)
         : dtype == kF16 ? append_four_fn<_Float16>(pairs, il)
                         : append_four_fn<__bf16>(pairs, il);
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
