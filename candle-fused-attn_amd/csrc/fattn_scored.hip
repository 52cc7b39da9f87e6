// Attention of scores of other forms, forward and backward: queries the last SQ of SK positions, key heads
// shared by groups of query heads. With x = scale q.k, i the query's position and j the key's:
//   y = cap tanh(x / cap) - slope_h |i - j|        (or x itself; no slope)
//   i sees j where (j <= i, or j < prefix_b, or it is not causal) and documents[b][i] = documents[b][j] >= 0
//   P = softmax(y) over what is seen, O = P V; a row that sees nothing is 0.
//   dV = P^T dO, dY = P o (dO V^T - rowsum(dO o O)), dX = dY (1 - tanh^2(x / cap)), dQ = scale dX K,
//   dK = scale dX^T Q.
// The products, scales, staging and sums are those of fattn_pair_kernels.h (fp32 as pairs of f16, blocks of
// four waves of 32 rows, a backward of two kinds of workgroup that share no sum); here are the scores and
// the walks. What a block can see is a range of tiles: from its positions, and, with documents, from the
// first to the last place of the ids between its least and its largest (so ids in order, as packed
// documents have them, leave only their own tiles; other orders are walked over and masked). A tile's ids
// are staged beside it: a wave passes over a tile in which it sees nothing, and takes one in which it sees
// everything without a mask.
//
// Bound: the vector units. A step of 32 x 32 pairs has 24 (forward), 36 and 48 (backward) matrix instructions at
// d 64, 32 cycles each, and 300 to 600 others of 4 and more: the staged tiles' split into f16, the scores'
// tanh and exponent, the weights' split; at d 64 two waves of the backward share a SIMD, at d 128 one has it alone
// and waits for its LDS reads besides. One body per walk, whose masked scores are minus infinity, and a kernel
// per kind of score (slopes, cap): bodies with and without a mask side by side took registers for both.
// Measured (kernels in a queue; the first twenty or so run at a lower clock, up to 20 % slower): 8 x 12 heads of 2048,
// d 64, causal, plain scores, forward 204 us, backward 646 (252 and 200 TFLOP/s of 4 d and 10 d operations a pair,
// each as three products of f16; fused_attention 198 and 635), capped 231 and 723; in documents of 600, capped, 124
// and 347; 4 x 16 heads in 4 groups of 777, d 128, slopes and prefixes, 81 and 235 + 10 (the sum of the chunks); 2 x
// 32 heads in 8 groups 512 x 4097, d 128, slopes, forward 280 and 16 its join (218 TFLOP/s). Cards differ by some
// percent; figures side by side are of one card.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "fattn_internal.h"
#include "fattn_pair_kernels.h"

namespace fattn {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
constexpr int kW = 4;                    // waves of a workgroup
constexpr int kBlock = kW * kRows;       // its rows
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kUnseen = -__builtin_inf();  // L of a row that sees nothing (in a chunk)
constexpr float kFirstRef = -3e38f;           // the softmax's reference before the first score
enum { kNone, kSome, kAll };                  // what a wave sees of a tile

// --- Who sees whom -----------------------------------------------------------------------------
// (Sixteen lanes by DPP, their four results as scalars. By six shuffles each, and with find_ids() waiting for
// each load, 8 x 12 heads of 2048 in documents took 147 us forward and 426 backward, 142 and 408 so.)
template <typename F>
__device__ __forceinline__ int over_wave(int x, F fn) {
  x = fn(x, __builtin_amdgcn_update_dpp(x, x, 0xB1, 0xF, 0xF, true));   // of two lanes
  x = fn(x, __builtin_amdgcn_update_dpp(x, x, 0x4E, 0xF, 0xF, true));   // of four
  x = fn(x, __builtin_amdgcn_update_dpp(x, x, 0x141, 0xF, 0xF, true));  // of eight, mirrored
  x = fn(x, __builtin_amdgcn_update_dpp(x, x, 0x140, 0xF, 0xF, true));  // of sixteen
  return fn(fn(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
            fn(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
__device__ __forceinline__ int wave_least(int x) {
  return over_wave(x, [](int a, int b) { return min(a, b); });
}
__device__ __forceinline__ int wave_most(int x) {
  return over_wave(x, [](int a, int b) { return max(a, b); });
}
// LDS of the ids: those of the staged tiles, and what the waves find.
struct IdSmem {
  __attribute__((aligned(16))) int tile[2][kRows];
  int found[2][kW][2];
};
// A wave's ids (one per lane j, both halves alike) and its block's.
struct Ids {
  int mine;          // of the lane's row
  int least, most;   // of the wave's rows that have a document; most -1: none
  bool one;          // all 32 rows have the same
  __device__ __forceinline__ void take(int id) {
    mine = id;
    least = wave_least(id >= 0 ? id : INT_MAX);
    most = wave_most(id);
    one = most >= 0 && __builtin_amdgcn_ballot_w64(id != most) == 0;
  }
};
// The block's rows' ids lie in [*lo, *hi]; the first and the last + 1 of ids[from .. to) that do (none:
// first >= last). For the whole workgroup.
__device__ __forceinline__ void find_ids(IdSmem& sm, const Ids& ids, const int32_t* all, int from, int to, int w,
                                         int tid, int& first, int& last) {
  if ((tid & 63) == 0) sm.found[0][w][0] = ids.least, sm.found[0][w][1] = ids.most;
  __syncthreads();
  int lo = sm.found[0][0][0], hi = sm.found[0][0][1];
#pragma unroll
  for (int i = 1; i < kW; ++i) lo = min(lo, sm.found[0][i][0]), hi = max(hi, sm.found[0][i][1]);
  int f = INT_MAX, l = -1;
  constexpr int kAtOnce = 8;  // (loads in flight; past the end the last again)
  for (int i0 = from + tid; i0 < to; i0 += 64 * kW * kAtOnce) {
    int id[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) id[u] = all[min(i0 + 64 * kW * u, to - 1)];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = min(i0 + 64 * kW * u, to - 1);
      if (id[u] >= lo && id[u] <= hi) f = min(f, i), l = i;
    }
  }
  f = wave_least(f), l = wave_most(l);
  if ((tid & 63) == 0) sm.found[1][w][0] = f, sm.found[1][w][1] = l;
  __syncthreads();
  first = sm.found[1][0][0], last = sm.found[1][0][1];
#pragma unroll
  for (int i = 1; i < kW; ++i) first = min(first, sm.found[1][i][0]), last = max(last, sm.found[1][i][1]);
  last += 1;
  first = __builtin_amdgcn_readfirstlane(first), last = __builtin_amdgcn_readfirstlane(last);
}
// What a wave with `ids` sees of a tile with id `id` in lane j, where positions let it see `sees` of it.
__device__ __forceinline__ int among(int id, const Ids& ids, int sees) {
  if (__builtin_amdgcn_ballot_w64(id >= ids.least && id <= ids.most) == 0) return kNone;
  return ids.one && __builtin_amdgcn_ballot_w64(id != ids.most) == 0 ? sees : kSome;
}
// The last key that the query at position p sees (but for documents).
__device__ __forceinline__ int last_key(const ScoredArgs& a, int p, int prefix) {
  return a.causal ? max(p, prefix - 1) : a.SK - 1;
}
__device__ __forceinline__ int prefix_of(const ScoredArgs& a, int b) {
  return a.prefix != nullptr ? min(max(a.prefix[b], 0), a.SK) : 0;
}
__device__ __forceinline__ const int32_t* ids_of(const ScoredArgs& a, int b) {
  return a.documents != nullptr ? a.documents + b * a.document_stride : nullptr;
}
__device__ __forceinline__ float slope_of(const ScoredArgs& a, int h) {
  return a.slopes != nullptr ? slope_log2(a.slopes[h]) : 0.0f;
}

// --- Scores ------------------------------------------------------------------------------------
// MODS, bits: 1, less a slope times the distance; 2, capped; 4 (with both), by a cap of which a part is multiplied
// last, ScoredArgs::unit_rest. With a cap the products' factor gives x / cap, a walk holds tanh of it, and cap2 of that
// (cap log2 e) enters with what the exponent adds anyway. (A kernel of its own: as a branch of the others that part
// takes 473 -> 486 us forward and backward, 8 x 12 heads of 2048 in documents.)
// One score in units of log2 e by its definition, for the rows in fp32, and dy / dx.
__device__ __forceinline__ float score_fp32(const ScoredArgs& a, float dot, float slope2, int far, float& slope) {
  float y = dot * (a.scale * kLog2e * a.unit) * a.unit_rest;
  slope = 1.0f;
  if (a.cap2 != 0.0f) y = a.cap2 * tanh_any(y, slope);
  return fmaf(-slope2, fabsf(static_cast<float>(far)), y);
}
// The sign of the scale goes with a wave's own rows: what is hidden, minus infinity, meets a factor above 0.
__device__ __forceinline__ float sign_of(float scale) { return scale < 0.0f ? -1.0f : 1.0f; }
// That factor, without a cap or slopes: of two rows' units, of which the product may be below the least float (two rows
// of zeros, as padding has them: 2^-252) or the scale 0. The least float more changes none that counts, and costs
// nothing beside a product. (8 x 12 heads of 2048, the second half zeros: 1566 and 5770 us without, every wave of zeros
// once more in fp32; 175 and 575 so.)
__device__ __forceinline__ float factor(float own, float staged) { return fmaf(own, staged, 0x1p-149f); }
// Nothing is scheduled across: sixteen polynomials side by side take more registers than there are.
__device__ __forceinline__ void few_at_once() { __builtin_amdgcn_sched_barrier(0); }
// x / cap of a wave's tile to its tanh t and `fn(r, dt / dx)`. (Nearly always every |x| / cap is small, where a
// polynomial does it: of degree 7 or 11 in x, against those and an exponential and a quotient besides.)
template <typename F>
__device__ __forceinline__ void capped(f16v& x, F fn) {
  const float most = max_weight(x);
  if (__builtin_amdgcn_ballot_w64(most > kTanhTiny) == 0) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = tanh_tiny(x[r]);
      fn(r, fmaf(-x[r], x[r], 1.0f));
      if (r % 4 == 3) few_at_once();
    }
  } else if (__builtin_amdgcn_ballot_w64(most > kTanhSmall) == 0) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = tanh_small(x[r]);
      fn(r, fmaf(-x[r], x[r], 1.0f));
      if (r % 4 == 3) few_at_once();
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float slope;
      x[r] = tanh_any(x[r], slope);
      fn(r, slope);
      if (r % 2 == 1) few_at_once();
    }
  }
}
// The slope's part. Register r is 8 (r / 4) + r % 4 places from the lane's base; where no seen pair of the
// tile has its key after its query, the distance is a sum of both, and slope x place (one value for the wave)
// is added to the score while the lane's part goes with what the exponent adds: no instruction of its own. Both
// parts are of the tile's places, up to 32 slopes, and their roundings stay where they cancel; so a steep slope
// (past 1 in the exponent: 2^-19 then) takes the distance itself, whose rounding is one of the score.
constexpr float kSteep = 1.0f;
__device__ __forceinline__ int place_of(int r) { return 8 * (r >> 2) + (r & 3); }
// Minus infinity to the registers of places outside [least, most]; to those of other ids than the lane's.
__device__ __forceinline__ void hide(f16v& s, int least, int most) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = place_of(r) >= least && place_of(r) <= most ? s[r] : kNegInf;
}
__device__ __forceinline__ void hide_others(f16v& s, const int* tile, int mine, int g) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const i4 id = *reinterpret_cast<const i4*>(&tile[8 * i + 4 * g]);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * i + e] = id[e] == mine ? s[4 * i + e] : kNegInf;
  }
}
struct Places {
  float by[16];  // slope2 times the place of register r, in scalar registers
  __device__ __forceinline__ void set(float slope2) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      by[r] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(slope2 * static_cast<float>(place_of(r)))));
    }
  }
};
// Otherwise: less slope2 |base + SIGN place|.
template <int SIGN>
__device__ __forceinline__ float far_by(int r, float slope2, float base) {
  return -slope2 * fabsf(base + static_cast<float>(SIGN * place_of(r)));
}
// s[r] = s[r] f + by(r), f as fn(i)[c] of register 4 i + c.
template <typename F, typename B>
__device__ __forceinline__ void scale_add(f16v& s, F fn, B by) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f4 f = fn(i);
#pragma unroll
    for (int c = 0; c < 4; ++c) s[4 * i + c] = fmaf(s[4 * i + c], f[c], by(4 * i + c));
  }
}

// --- Rows in fp32 (see fattn_pair_kernels.h) -----------------------------------------------------
// L of a row; of a chunk in 64 bits, since the join takes differences of it.
__device__ __forceinline__ void put_l(const ScoredArgs& a, int chunk, int64_t at, double L) {
  if (a.nc > 1) {
    a.l_part[chunk * (static_cast<int64_t>(a.B) * a.H * a.SQ) + at] = L;
  } else {
    __builtin_nontemporal_store(static_cast<float>(L), a.lse + at);
  }
}
// O and L of 32 queries from qg over the tiles from t0 to t1.
template <int D, typename Store>
__device__ __forceinline__ void scored_rows_fp32(const ScoredArgs& a, int b, int h, int qg, int t0, int t1,
                                                 int chunk, float* so, int lane, Store store) {
  const int j = lane & 31, g = lane >> 5, qc = min(qg + j, a.SQ - 1), p = qc + a.SK - a.SQ, hk = h / a.G;
  const float* qp = a.q.p + b * a.q.sb + h * a.q.sh + qc * a.q.ss;
  const float* kp = a.k.p + b * a.k.sb + hk * a.k.sh;
  const float* vp = a.v.p + b * a.v.sb + hk * a.v.sh;
  const int lim = last_key(a, p, prefix_of(a, b));
  const int32_t* ids = ids_of(a, b);
  const int id = ids != nullptr ? ids[p] : 0;
  const float slope2 = slope_of(a, h);
  f16v acc[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) acc[dt] = zero16();
  float m = kNegInf, l = 0.0f;
  auto live = [&](int key) {
    return key <= lim && id >= 0 && (ids == nullptr || ids[min(key, a.SK - 1)] == id);
  };
#pragma clang loop unroll(disable)
  for (int t = t0; t < t1; ++t) {
    const int k0 = t * kRows;
    f16v s = dots_fp32<D>(kp + min(k0 + j, a.SK - 1) * a.k.ss, qp, g);
    float mn = m;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = k0 + tile_row(r, g);
      const bool is = live(key);
      float d;
      s[r] = is ? score_fp32(a, s[r], slope2, p - key, d) : kNegInf;
      mn = fmaxf(mn, s[r]);
    }
    mn = pair_max(fmaxf(mn, kNegInf));
    const float alpha = mn == m ? 1.0f : m == kNegInf ? 0.0f : exp2_hw(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) acc[dt] *= alpha;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = s[r] == kNegInf ? 0.0f : exp2_hw(s[r] - mn);
      l += s[r];
    }
    sum_fp32<D, false>(s, vp, a.v.ss, k0, a.SK, live, so, acc, j, g);
  }
  l = pair_sum(l);
  // (Every row with a document sees itself. One whose every score is minus infinity is NaN, as its formula:
  // 0 / 0; a chunk of such weighs nothing.)
  store(acc, l == 0.0f && (id < 0 || a.nc > 1) ? 1.0f : 1.0f / l);
  if (g == 0 && qg + j < a.SQ) {
    const double L = l == 0.0f ? kUnseen : static_cast<double>(m) * kLn2 + logf(l);
    put_l(a, chunk, (static_cast<int64_t>(b) * a.H + h) * a.SQ + qg + j, L);
  }
}

// dK and dV of 32 keys from kw0, over steps u0 .. u1 of the walk of n tiles from t0 of each head of the group,
// in fp32.
template <int D>
__device__ __forceinline__ void scored_keys_fp32(const ScoredArgs& a, int b, int hk, int kw0, int t0, int n,
                                                 int u0, int u1, float* so, f16v (&dk)[D / 32], f16v (&dv)[D / 32], int lane) {
  const int j = lane & 31, g = lane >> 5, key = kw0 + j, kc = min(key, a.SK - 1), off = a.SK - a.SQ;
  const float* kr = a.k.p + b * a.k.sb + hk * a.k.sh + kc * a.k.ss;
  const float* vr = a.v.p + b * a.v.sb + hk * a.v.sh + kc * a.v.ss;
  const int prefix = prefix_of(a, b);
  const int32_t* ids = ids_of(a, b);
  const int id = key < a.SK ? (ids != nullptr ? ids[kc] : 0) : -1;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) dk[dt] = zero16(), dv[dt] = zero16();
  auto live = [&](int qi) {
    return qi < a.SQ && id >= 0 && key <= last_key(a, qi + off, prefix) &&
           (ids == nullptr || ids[min(qi, a.SQ - 1) + off] == id);
  };
#pragma clang loop unroll(disable)
  for (int u = u0; u < u1; ++u) {
    const int h = hk * a.G + u / n, q0 = (t0 + u % n) * kRows;
    const float* qp = a.q.p + b * a.q.sb + h * a.q.sh;
    const float* gp = a.d_o.p + b * a.d_o.sb + h * a.d_o.sh;
    const float* op = a.o + (static_cast<int64_t>(b) * a.SQ * a.H + h) * D;
    const float* lp = a.lse + (static_cast<int64_t>(b) * a.H + h) * a.SQ;
    const float slope2 = slope_of(a, h);
    const int64_t qr = min(q0 + j, a.SQ - 1);
    f16v s = dots_fp32<D>(qp + qr * a.q.ss, kr, g), dp = dots_fp32<D>(gp + qr * a.d_o.ss, vr, g);
    float dd = 0.0f;
#pragma clang loop unroll(disable)
    for (int c = 4 * g; c < D; c += 8) {
      const f4 x = ld4(gp + qr * a.d_o.ss + c), y = ld4(op + qr * a.H * D + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) dd = fmaf(x[e], y[e], dd);
    }
    dd = pair_sum(dd);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int t = tile_row(r, g), qi = min(q0 + t, a.SQ - 1);
      float slope;
      const float y = score_fp32(a, s[r], slope2, qi + off - key, slope);
      const float p = exp2_hw(y + shifted_l(lp[qi], 0.0f));
      const float w = p * (dp[r] - __shfl(dd, t)) * slope;  // (every lane takes part in the shuffle)
      const bool is = live(q0 + t);
      s[r] = is ? p : 0.0f;
      dp[r] = is ? w : 0.0f;
    }
    sum_fp32<D, false>(s, gp, a.d_o.ss, q0, a.SQ, live, so, dv, j, g);
    sum_fp32<D, false>(dp, qp, a.q.ss, q0, a.SQ, live, so, dk, j, g);
  }
}
// dQ of 32 queries from qw0 over the tiles t0 .. t1, in fp32 (without the scale).
template <int D>
__device__ __forceinline__ void scored_queries_fp32(const ScoredArgs& a, int b, int h, int qw0, int t0, int t1,
                                                    float* so, f16v (&dq)[D / 32], int lane) {
  const int j = lane & 31, g = lane >> 5, hk = h / a.G, off = a.SK - a.SQ;
  const int64_t qc = min(qw0 + j, a.SQ - 1);
  const int p = static_cast<int>(qc) + off;
  const float* qr = a.q.p + b * a.q.sb + h * a.q.sh + qc * a.q.ss;
  const float* gr = a.d_o.p + b * a.d_o.sb + h * a.d_o.sh + qc * a.d_o.ss;
  const float* kp = a.k.p + b * a.k.sb + hk * a.k.sh;
  const float* vp = a.v.p + b * a.v.sb + hk * a.v.sh;
  const float* orow = a.o + ((static_cast<int64_t>(b) * a.SQ + qc) * a.H + h) * D;
  const float L = shifted_l(a.lse[(static_cast<int64_t>(b) * a.H + h) * a.SQ + qc], 0.0f);
  const int lim = last_key(a, p, prefix_of(a, b));
  const int32_t* ids = ids_of(a, b);
  const int id = ids != nullptr ? ids[p] : 0;
  const float slope2 = slope_of(a, h);
  float dd = 0.0f;
#pragma clang loop unroll(disable)
  for (int c = 4 * g; c < D; c += 8) {
    const f4 x = ld4(gr + c), y = ld4(orow + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) dd = fmaf(x[e], y[e], dd);
  }
  dd = pair_sum(dd);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) dq[dt] = zero16();
  auto live = [&](int key) {
    return key <= lim && id >= 0 && (ids == nullptr || ids[min(key, a.SK - 1)] == id);
  };
#pragma clang loop unroll(disable)
  for (int t = t0; t < t1; ++t) {
    const int64_t kr = min(t * kRows + j, a.SK - 1);
    const f16v s = dots_fp32<D>(kp + kr * a.k.ss, qr, g);
    f16v dp = dots_fp32<D>(vp + kr * a.v.ss, gr, g);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = t * kRows + tile_row(r, g);
      float slope;
      const float y = score_fp32(a, s[r], slope2, p - key, slope);
      const float w = exp2_hw(y + L) * (dp[r] - dd) * slope;
      dp[r] = live(key) ? w : 0.0f;
    }
    sum_fp32<D, false>(dp, kp, a.k.ss, t * kRows, a.SK, live, so, dq, j, g);
  }
}

// --- Forward -----------------------------------------------------------------------------------
// A workgroup: 128 queries of one head, over a range of key tiles; where the blocks are too few for the
// chip the tiles are cut into chunks, whose O and L a second kernel joins in order.
template <int D, int MODS>
__device__ __forceinline__ void scored_fwd(const ScoredArgs& a) {
  constexpr int kKS = D / 16, kDT = D / 32, kOPitch = (D < 64 ? D : 64) + 4;
  struct Kv {
    Tile<D> k, v;
  };
  union Tiles {
    Kv kv[2];
    float o[kW][kRows * kOPitch];
  };
  struct Smem {
    Tiles t;
    float uk[2][kRows], uv[2][kRows];
    IdSmem ids;
  };
  __shared__ __attribute__((aligned(16))) Smem sm;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int BH = a.B * a.H, off = a.SK - a.SQ;
  // (Causal: the blocks that see most first, and the heads of a group, which read the same keys, in one XCD's L2
  // where the key heads are a multiple of the XCDs. 2 x 32 heads in 8 groups 512 x 4097 d 128 so 97 MB from
  // memory and, on one card, 286 us with the join, group heads side by side 780 and 289; the backward's query
  // blocks, 4 x 16 heads in 4 groups of 777, take 2 % longer so.)
  const int id = static_cast<int>(blockIdx.x), per = a.nqb * a.nc, pairs = a.B * (a.H / a.G), in_pair = id / pairs;
  const int item = a.causal ? (id % pairs * a.G + in_pair % a.G) * per + per - 1 - in_pair / a.G
                            : xcd_remap(id, per * BH);
  const int bh = item / per, in = item - bh * per, qb = in / a.nc, chunk = in - qb * a.nc;
  const int b = bh / a.H, h = bh % a.H, hk = h / a.G;
  const int qw0 = qb * kBlock + w * kRows, qi = qw0 + j, pos = min(qi, a.SQ - 1) + off;
  const int prefix = prefix_of(a, b);
  const int32_t* all_ids = ids_of(a, b);
  // The keys: of the block to `end`, of the wave's first and last query to `lo` and `hi`.
  const int end = last_key(a, min(qb * kBlock + kBlock, a.SQ) - 1 + off, prefix) + 1;
  const int lim = last_key(a, pos, prefix);
  const int lo = last_key(a, min(qw0, a.SQ - 1) + off, prefix);
  const int hi = last_key(a, min(qw0 + kRows, a.SQ) - 1 + off, prefix);
  // No key that is seen after its query; the wave's first position (past the last query: the last).
  const bool ordered = a.causal && prefix == 0;
  const int lo_pos = min(qw0, a.SQ - 1) + off;
  const bool wave_live = qw0 < a.SQ;
  int t0 = 0, t1 = (end + kRows - 1) / kRows;
  Ids ids{0, 0, 0, true};
  if (all_ids != nullptr) {
    ids.take(all_ids[pos]);
    int first, last;
    find_ids(sm.ids, ids, all_ids, 0, end, w, tid, first, last);
    t0 = first / kRows, t1 = first < last ? (last + kRows - 1) / kRows : t0;
  }
  if (a.nc > 1) t0 = max(t0, chunk * a.chunk), t1 = min(t1, (chunk + 1) * a.chunk);
  float* out = a.nc > 1 ? a.o_part + chunk * (static_cast<int64_t>(BH) * a.SQ * D) : a.out;
  if (t0 >= t1) {  // no key to see: O is 0, L -infinity (a chunk: L alone)
    if (a.nc == 1) {
      for (int i = lane; i < min(a.SQ - qw0, kRows) * (D / 4); i += 64) {
        const int64_t row = static_cast<int64_t>(b) * a.SQ + qw0 + i / (D / 4);
        st4(out + (row * a.H + h) * D + i % (D / 4) * 4, f4{});
      }
    }
    if (lane < min(a.SQ - qw0, kRows)) put_l(a, chunk, static_cast<int64_t>(bh) * a.SQ + qw0 + lane, kUnseen);
    return;
  }
  const float* qp = a.q.p + b * a.q.sb + h * a.q.sh;
  const Operand kop{reinterpret_cast<const char*>(a.k.p + b * a.k.sb + hk * a.k.sh),
                    static_cast<unsigned>(a.k.ss) * 4u};
  const Operand vop{reinterpret_cast<const char*>(a.v.p + b * a.v.sb + hk * a.v.sh),
                    static_cast<unsigned>(a.v.ss) * 4u};

  Stage<D, kW> st;
  int id_next = 0;
  auto load = [&](int t) {
    st.load(kop, vop, t * kRows, a.SK - 1, w, lane);
    if (all_ids != nullptr && w == 0) id_next = all_ids[min(t * kRows + j, a.SK - 1)];
  };
  auto store = [&](int t) {
    const int put = t & 1;
    st.store(sm.t.kv[put].k, sm.t.kv[put].v, sm.uk[put], sm.uv[put], w, lane);
    if (all_ids != nullptr && w == 0) sm.ids.tile[put][j] = t * kRows + j < a.SK ? id_next : -1;
  };
  Pair q[kKS];
  float cq;  // |scale| log2 e over the query's scale, with a cap over that too
  {
    OwnRows<D> own;
    load(t0);
    own.load(qp + min(qi, a.SQ - 1) * a.q.ss, g);
    store(t0);
    load(t0 + 1);
    cq = own.split(sign_of(a.scale), q) * (fabsf(a.scale) * kLog2e * ((MODS & 2) != 0 ? a.unit : 1.0f));
  }
  const float slope2 = (MODS & 1) != 0 ? slope_of(a, h) : 0.0f;
  const float f2 = (MODS & 2) != 0 ? a.cap2 : 1.0f;
  Places places;
  if constexpr ((MODS & 1) != 0) places.set(slope2);
  f16v acc[kDT];  // O^T, in units of p / wsc and 2^-kTop
  float m = kFirstRef, lsum = 0.0f, wsc = kMaxScale;
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt) acc[dt] = zero16();
  const int roff0 = row_off<D>(j, g), coff0 = col_off<D>(lane);

  auto stage = [&](int t) {
    store(t + 1);
    load(t + 2);
    pin_loads();
  };
  // (See fattn_pair_kernels.h for the sums' scales.)
  auto tile = [&](int t, int sees) {
    const int roff = late(roff0), coff = late(coff0), kt0 = t * kRows, cur = t & 1;
    const Kv& kv = sm.t.kv[cur];
    stage(t);
    f16v s = zero16();
    {
      h8 kh[kKS];
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const Pair k = ld_row<D>(kv.k, roff ^ row_step(ks));
        kh[ks] = k.h;
        s = mma_small(k, q[ks], s);
      }
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) s = mma(kh[ks], q[ks].h, s);
    }
    float shift = 0.0f;  // of what is held less the score
    if constexpr ((MODS & 2) != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 uk = ld4(&sm.uk[cur][8 * i + 4 * g]);
#pragma unroll
        for (int c = 0; c < 4; ++c) s[4 * i + c] *= cq * uk[c];
      }
      if constexpr ((MODS & 4) != 0) s *= a.unit_rest;
      capped(s, [](int, float) {});
    }
    if constexpr ((MODS & 1) != 0) {
      auto f = [&](int i) {
        if constexpr ((MODS & 2) != 0) return f4{f2, f2, f2, f2};
        return ld4(&sm.uk[cur][8 * i + 4 * g]) * cq;
      };
      const float base = static_cast<float>(pos - 4 * g - kt0);
      if (fabsf(slope2) <= kSteep && (ordered || kt0 + kRows - 1 <= lo_pos)) {
        shift = slope2 * base;
        scale_add(s, f, [&](int r) { return places.by[r]; });
      } else {
        scale_add(s, f, [&](int r) { return far_by<-1>(r, slope2, base); });
      }
    }
    // What is not seen is minus infinity: register r's key is kt0 + 4 g + 8 (r / 4) + r % 4.
    if (sees == kSome) {
      hide(s, 0, ids.mine >= 0 ? lim - kt0 - 4 * g : -1);
      if (all_ids != nullptr) hide_others(s, sm.ids.tile[cur], ids.mine, g);
    }
    f16v e;
    float psum = 0.0f, wmax = 0.0f;
    auto exps = [&] {
      wmax = 0.0f;
      int r0 = 4 * g;
      asm("" : "+v"(r0));
      const float ref = m + shift;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 uv = ld4(&sm.uv[cur][8 * i + r0]);
        f4 uk{};
        if constexpr (MODS == 0) uk = ld4(&sm.uk[cur][8 * i + r0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = 4 * i + c;
          const float p = exp2_hw(MODS == 0   ? fmaf(s[r], factor(cq, uk[c]), -m)
                                  : MODS == 2 ? fmaf(s[r], f2, -m)
                                              : s[r] - ref);
          psum = r == 0 ? p : psum + p;
          e[r] = p * uv[c];
        }
        asm("v_max3_f32 %0, %1, %2, %0" : "+v"(wmax) : "v"(e[4 * i]), "v"(e[4 * i + 1]));
        asm("v_max3_f32 %0, %1, %2, %0" : "+v"(wmax) : "v"(e[4 * i + 2]), "v"(e[4 * i + 3]));
      }
    };
    exps();
    if (__builtin_amdgcn_ballot_w64(!(psum <= kRowTop && wmax * wsc <= kMaxWeight)) != 0) {
      float tmax = kNegInf;
      int r0 = 4 * g;
      asm("" : "+v"(r0));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        tmax = fmaxf(tmax, MODS != 0 ? s[r] : s[r] * factor(cq, sm.uk[cur][8 * (r >> 2) + r0 + (r & 3)]));
      }
      if constexpr (MODS == 2) tmax *= f2;
      const float ref = pair_max(tmax - shift) - kRefTop;
      float to = wsc, alpha = 1.0f;
      if (!(pair_sum(psum) <= kRowTop) && ref > m) {
        alpha = exp2_hw(m - ref);  // (0 from the first one)
        to = alpha > 0.0f ? fminf(to * pow2(-exponent(alpha)), kMaxScale) : kMaxScale;
        m = ref;
        lsum *= alpha;
        exps();
      }
      wmax = pair_max(fmaxf(wmax, 0.0f));
      if (wmax * to > kMaxWeight) to = pow2(kWTop - exponent(wmax));
      const float f = alpha > 0.0f ? alpha * (to / wsc) : 0.0f;
      wsc = to;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) acc[dt] *= f;
    }
    lsum += psum;
    const Pair p0 = split_acc<0>(e, wsc), p1 = split_acc<1>(e, wsc);
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt) {
      acc[dt] = mma3(ld_col<D>(kv.v, coff ^ col_step(dt), 0), p0, acc[dt]);
      acc[dt] = mma3(ld_col<D>(kv.v, coff ^ col_step(dt), 1), p1, acc[dt]);
    }
  };
  auto seen = [&](int t) {
    const int sees = !wave_live || t * kRows > hi ? kNone : t * kRows + kRows - 1 <= lo ? kAll : kSome;
    return all_ids == nullptr || sees == kNone ? sees : among(sm.ids.tile[t & 1][j], ids, sees);
  };
  __syncthreads();  // tile t0
  int t = t0, sees;
  while (t < t1) {
    while (t < t1 && (sees = seen(t)) != kNone) {
      tile(t, sees);
      __syncthreads();  // tile t + 1 is staged; every wave is done with tile t
      ++t;
    }
    while (t < t1 && seen(t) == kNone) {
      stage(t);
      __syncthreads();
      ++t;
    }
  }
  if (!wave_live) return;

  // L = (m + log2 l) ln 2, to one rounding: the backward takes 2^(y - L log2 e).
  const float l = pair_sum(lsum);
  float* so = sm.t.o[w];
  const int lane_e = late(lane);
  auto put = [&](const f16v (&x)[kDT], float f, float f2) {
    store_rows<D>(x, f, f2, so, out + ((static_cast<int64_t>(b) * a.SQ + qw0) * a.H + h) * D,
                  static_cast<int64_t>(a.H) * D, a.SQ - qw0, lane_e);
  };
  const bool lost = l == 0.0f && ids.mine >= 0 && a.nc == 1;  // (every score is minus infinity)
  if (__builtin_amdgcn_ballot_w64(qi < a.SQ && (lost || !(probe_finite<kDT>(acc, l * 0.0f) == 0.0f))) != 0) {
    scored_rows_fp32<D>(a, b, h, qw0, t0, t1, chunk, so, late(lane),
                        [&](const f16v (&x)[kDT], float inv) { put(x, inv, 1.0f); });
    return;
  }
  // (A row that saw nothing has sums of 0. Two factors: their product may be subnormal.)
  put(acc, l == 0.0f ? 1.0f : 1.0f / l, pow2(-kTop) / wsc);
  if (g == 0 && qi < a.SQ) {
    int le = exponent(l);
    float f = l * pow2(-le);  // [1, 2), then [0.75, 1.5)
    if (f > 1.5f) f *= 0.5f, ++le;
    const double L = l == 0.0f ? kUnseen : fma(static_cast<double>(m), kLn2, fma(le, kLn2, logf(f)));
    put_l(a, chunk, static_cast<int64_t>(bh) * a.SQ + qi, L);
  }
}
template <int D, int MODS, int WAVES>
__global__ void __launch_bounds__(64 * kW) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))
fwd_scored_kernel(ScoredArgs a) {
  scored_fwd<D, MODS>(a);
}

// O and L of the chunks' [nc][b, s, h, d] and [nc][b, h, s]: O = sum_c w_c O_c / sum_c w_c, w_c =
// exp(L_c - max), L = max + log sum; a chunk in which a row saw nothing (L -infinity) has no O. D / 4 lanes a
// row.
template <int D>
__global__ void __launch_bounds__(256) join_scored_kernel(ScoredArgs a) {
  constexpr int kLanes = D / 4, kAtOnce = 4;  // (chunks in flight)
  const int rows = a.B * a.SQ * a.H, row = static_cast<int>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (row >= rows) return;
  const int d = threadIdx.x % kLanes * 4;
  const int r = row / a.H, h = row - r * a.H, b = r / a.SQ, i = r - b * a.SQ;
  const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.SQ + i;
  f4 o[kAtOnce];
  auto load = [&](int c0) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      o[u] = ld4(a.o_part + (static_cast<int64_t>(min(c0 + u, a.nc - 1)) * rows + row) * D + d);
    }
  };
  auto l_of = [&](int c) { return a.l_part[static_cast<int64_t>(min(c, a.nc - 1)) * rows + at]; };
  load(0);
  double top = kUnseen;
  for (int c0 = 0; c0 < a.nc; c0 += 2 * kAtOnce) {
    double L[2 * kAtOnce];
#pragma unroll
    for (int u = 0; u < 2 * kAtOnce; ++u) L[u] = l_of(c0 + u);
#pragma unroll
    for (int u = 0; u < 2 * kAtOnce; ++u) top = L[u] > top || L[u] != L[u] ? L[u] : top;
  }
  float sum = 0.0f;
  f4 x{};
  for (int c0 = 0; c0 < a.nc; c0 += kAtOnce) {
    if (c0 > 0) load(c0);
    double L[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) L[u] = l_of(c0 + u);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      // (What lies in the O of a chunk that saw nothing is not looked at.)
      if (c0 + u >= a.nc || L[u] == kUnseen) continue;
      const float w = expf(static_cast<float>(L[u] - top));
      sum += w;
      x += o[u] * w;
    }
  }
  // (No chunk saw anything: a row without a document, or, NaN, scores that are all minus infinity.)
  const int32_t* ids = ids_of(a, b);
  const bool none = top == kUnseen && ids != nullptr && ids[i + a.SK - a.SQ] < 0;
  st4(a.out + static_cast<int64_t>(row) * D + d, none ? f4{} : x * (1.0f / sum));
  if (d == 0) a.lse[at] = top == kUnseen ? kNegInf : static_cast<float>(top + logf(sum));
}

// --- Backward ----------------------------------------------------------------------------------
// Key blocks walk the query tiles that see them, of each head of their group in turn, and hold dK and dV;
// query blocks walk the key tiles that they see and hold dQ.
template <int D>
union ScoredTiles {
  struct {
    Tile<D> a, b;
  } t[2];
  float o[kW][kRows * ((D < 64 ? D : 64) + 4)];
};
template <int D>
struct ScoredSmem {
  ScoredTiles<D> u;
  float ua[2][kRows], ub[2][kRows], l[2][kRows], d[2][kRows];
  float ls[2][kRows];  // (key blocks) l less the slope times the row's place in the tile
  IdSmem ids;
};

template <int D, int MODS>
__device__ __forceinline__ void scored_keys(const ScoredArgs& a, ScoredSmem<D>& sm, int item, int chunk) {
  constexpr int kKS = D / 16, kDT = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int HK = a.H / a.G, off = a.SK - a.SQ, SQ = a.SQ;
  const int bh = item / a.nkb, kb = item % a.nkb, b = bh / HK, hk = bh % HK, h0 = hk * a.G;
  const int k0 = kb * kBlock, kw0 = k0 + w * kRows, key = kw0 + j, kc = min(key, a.SK - 1);
  const int prefix = prefix_of(a, b);
  const int32_t* all_ids = ids_of(a, b);
  const bool wave_live = kw0 < a.SK;
  // The queries: all, or from the first at or past the block's first key.
  int q_first = a.causal && k0 >= prefix ? max(k0 - off, 0) : 0, q_end = SQ;
  Ids ids{0, 0, 0, true};
  if (all_ids != nullptr) {
    ids.take(key < a.SK ? all_ids[kc] : -1);
    int first, last;
    find_ids(sm.ids, ids, all_ids, q_first + off, a.SK, w, tid, first, last);
    q_first = first - off, q_end = last - off;
  }
  // The walk: n tiles from t0 of each head of the group, or a chunk of these steps, from u0 on.
  const int t0 = q_first / kRows, n = (q_end + kRows - 1) / kRows - t0, u0 = chunk * a.chk;
  const int steps = q_first < q_end ? min(n * a.G - u0, a.chk) : 0;
  float* dkv = a.dkv + ((static_cast<int64_t>(chunk) * a.B + b) * a.SK + kw0) * 2 * HK * D +
               static_cast<int64_t>(hk) * D;
  if (steps <= 0) {  // keys that no query sees
    for (int i = lane; i < min(a.SK - kw0, kRows) * (D / 4); i += 64) {
      float* row = dkv + static_cast<int64_t>(i / (D / 4)) * 2 * HK * D + i % (D / 4) * 4;
      st4(row, f4{});
      st4(row + static_cast<int64_t>(HK) * D, f4{});
    }
    return;
  }
  const Operand qop{reinterpret_cast<const char*>(a.q.p + b * a.q.sb + h0 * a.q.sh),
                    static_cast<unsigned>(a.q.ss) * 4u};
  const Operand gop{reinterpret_cast<const char*>(a.d_o.p + b * a.d_o.sb + h0 * a.d_o.sh),
                    static_cast<unsigned>(a.d_o.ss) * 4u};
  const float* op = a.o + (static_cast<int64_t>(b) * SQ * a.H + h0) * D;
  const float* lp = a.lse + (static_cast<int64_t>(b) * a.H + h0) * SQ;

  const int kp = half_log2(a.SK);
  Stage<D, kW> st;
  RowDots<D, kW> ro;
  float lreg, slope_next = 0.0f;
  int id_next = 0;
  // Step u's head in the group (past the last step: the last) and its tile's first row.
  auto place = [&](int u, int& hh) {
    hh = min((u + u0) / n, a.G - 1);
    return (t0 + u + u0 - hh * n) * kRows;
  };
  auto load = [&](int u) {
    int hh;
    const int r0 = place(u, hh);
    st.load(Operand{qop.p + hh * a.q.sh * 4, qop.ss4}, Operand{gop.p + hh * a.d_o.sh * 4, gop.ss4}, r0, SQ - 1, w,
            lane);
    if (all_ids != nullptr && w == 0) id_next = r0 + j < SQ ? all_ids[r0 + j + off] : -1;
  };
  auto load_o = [&](int u) {
    int hh;
    const int r0 = place(u, hh);
    ro.load(op + hh * D, static_cast<unsigned>(a.H) * D, r0, SQ - 1, w, lane);
    lreg = lp[hh * static_cast<int64_t>(SQ) + min(r0 + j, SQ - 1)];
    if constexpr ((MODS & 1) != 0) {
      if (w == 0) slope_next = slope_of(a, h0 + hh);
    }
  };
  auto store = [&](int u) {
    const int put = u & 1;
    st.store(sm.u.t[put].a, sm.u.t[put].b, sm.ua[put], sm.ub[put], w, lane);
    ro.put(st, sm.d[put], w, lane);
    if (w == 0 && g == 0) {
      // (A row that sees nothing has an L of minus infinity, and scores of it too.)
      const float l = id_next < 0 ? 0.0f : shifted_l(lreg, kp);
      sm.l[put][j] = l;
      if constexpr ((MODS & 1) != 0) sm.ls[put][j] = fmaf(-slope_next, static_cast<float>(j), l);
      if (all_ids != nullptr) sm.ids.tile[put][j] = id_next;
    }
  };
  Pair kB[kKS], vB[kKS];
  float uk, uv;  // 1 / the key's scales
  {
    OwnRows<D> ok, ov;
    load(0);
    load_o(0);
    ok.load(a.k.p + b * a.k.sb + hk * a.k.sh + kc * a.k.ss, g);
    ov.load(a.v.p + b * a.v.sb + hk * a.v.sh + kc * a.v.ss, g);
    uk = ok.split(sign_of(a.scale), kB);
    uv = ov.split(1.0f, vB);
    store(0);
    load(1);
    load_o(1);
  }
  f16v dk[kDT], dv[kDT];
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt) dk[dt] = zero16(), dv[dt] = zero16();
  const float cs = fabsf(a.scale) * kLog2e * ((MODS & 2) != 0 ? a.unit : 1.0f) * uk, cg = uv;
  const float f2 = (MODS & 2) != 0 ? a.cap2 : 1.0f;
  const bool ordered = a.causal && prefix == 0;
  float psc = kMaxScale, dsc = kMaxScale;
  const int roff0 = row_off<D>(j, g), coff0 = col_off<D>(lane);

  auto tile = [&](int u, int q0, int hh, int sees) {
    const int roff = late(roff0), coff = late(coff0), cur = u & 1;
    store(u + 1);
    const Tile<D>&Q = sm.u.t[cur].a, &G = sm.u.t[cur].b;
    f16v s = zero16(), dp = zero16();
    {
      h8 x[kKS];
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const Pair q = ld_row<D>(Q, roff ^ row_step(ks));
        x[ks] = q.h;
        // (The forward's order: its A operand is this B.)
        s = mma(q.l, kB[ks].h, s);
        s = mma(q.h, kB[ks].l, s);
      }
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) s = mma(x[ks], kB[ks].h, s);
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const Pair y = ld_row<D>(G, roff ^ row_step(ks));
        x[ks] = y.h;
        dp = mma_small(y, vB[ks], dp);
      }
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) dp = mma(x[ks], vB[ks].h, dp);
    }
    // The loads of the step after next from here on (its O later still): held across the products above as
    // well, they do not fit.
    load(u + 2);
    pin_loads();
    if constexpr ((MODS & 2) != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 uq = ld4(&sm.ua[cur][8 * i + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * i + e] *= cs * uq[e];
      }
      if constexpr ((MODS & 4) != 0) s *= a.unit_rest;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 Dv = ld4(&sm.d[cur][8 * i + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * i + e] = fmaf(dp[4 * i + e], cg, -Dv[e]);
    }
    if constexpr ((MODS & 2) != 0) capped(s, [&](int r, float slope) { dp[r] *= slope; });
    // The slope's part: a row's (staged with its L) and the lane's, or, where a key may be after a query that
    // sees it, of the distance.
    // (With a slope s becomes the whole exponent.)
    if constexpr ((MODS & 1) != 0) {
      const float slope2 = slope_of(a, h0 + hh);
      auto f = [&](int i) {
        if constexpr ((MODS & 2) != 0) return f4{f2, f2, f2, f2};
        return ld4(&sm.ua[cur][8 * i + 4 * g]) * cs;
      };
      if (fabsf(slope2) <= kSteep && (ordered || kw0 + kRows - 1 <= q0 + off)) {
        const float shift = slope2 * static_cast<float>(key - q0 - off);
        scale_add(s, f, [&](int r) { return sm.ls[cur][place_of(r) + 4 * g] + shift; });
      } else {
        const float base = static_cast<float>(q0 + 4 * g + off - key);
        scale_add(s, f, [&](int r) { return sm.l[cur][place_of(r) + 4 * g] + far_by<1>(r, slope2, base); });
      }
    }
    // Register r's query is q0 + 4 g + 8 i + e: seen below SQ and, causal, not before the key.
    if (sees == kSome) {
      hide(s, a.causal && key >= prefix ? key - off - q0 - 4 * g : 0,
           key < a.SK && ids.mine >= 0 ? SQ - 1 - q0 - 4 * g : -1);
      if (all_ids != nullptr) hide_others(s, sm.ids.tile[cur], ids.mine, g);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 uq = ld4(&sm.ua[cur][8 * i + 4 * g]), ug = ld4(&sm.ub[cur][8 * i + 4 * g]);
      f4 L{};
      if constexpr ((MODS & 1) == 0) L = ld4(&sm.l[cur][8 * i + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * i + e;
        s[r] = exp2_hw((MODS & 1) != 0 ? s[r] : fmaf(s[r], MODS == 0 ? factor(cs, uq[e]) : f2, L[e])) * ug[e];
        dp[r] = s[r] * dp[r] * uq[e];
      }
    }
    pin_acc(dv);
    pin_acc(dk);
    const float mp = max_weight(s), md = max_weight(dp);
    if (__builtin_amdgcn_ballot_w64(mp * psc > kMaxWeight || md * dsc > kMaxWeight) != 0) {
      fit_scale(mp, psc, dv);
      fit_scale(md, dsc, dk);
      pin_acc(dv);
      pin_acc(dk);
    }
    {
      const Pair p0 = split_acc<0>(s, psc), p1 = split_acc<1>(s, psc);
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) {
        dv[dt] = mma3(ld_col<D>(G, coff ^ col_step(dt), 0), p0, dv[dt]);
        dv[dt] = mma3(ld_col<D>(G, coff ^ col_step(dt), 1), p1, dv[dt]);
      }
    }
    load_o(u + 2);
    pin_loads();
    {
      const Pair p0 = split_acc<0>(dp, dsc), p1 = split_acc<1>(dp, dsc);
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) {
        dk[dt] = mma3(ld_col<D>(Q, coff ^ col_step(dt), 0), p0, dk[dt]);
        dk[dt] = mma3(ld_col<D>(Q, coff ^ col_step(dt), 1), p1, dk[dt]);
      }
    }
  };
  // What the wave's keys are seen by, of a step's tile.
  auto seen = [&](int u, int q0) {
    if (!wave_live) return static_cast<int>(kNone);
    const bool before = a.causal && kw0 >= prefix;  // (else some key of the wave is in the prefix)
    if (before && q0 + kRows - 1 + off < kw0) return static_cast<int>(kNone);
    const bool whole = q0 + kRows <= SQ && kw0 + kRows <= a.SK &&
                       (!a.causal || kw0 + kRows - 1 <= q0 + off || kw0 + kRows <= prefix);
    const int sees = whole ? kAll : kSome;
    return all_ids == nullptr ? sees : among(sm.ids.tile[u & 1][j], ids, sees);
  };
  __syncthreads();
  int u = 0, hh, q0 = place(0, hh), sees;
  auto next = [&] {
    ++u, q0 += kRows;
    if (q0 == (t0 + n) * kRows) q0 = t0 * kRows, ++hh;
  };
  while (u < steps) {
    while (u < steps && (sees = seen(u, q0)) != kNone) {
      tile(u, q0, hh, sees);
      __syncthreads();
      next();
    }
    while (u < steps && seen(u, q0) == kNone) {
      store(u + 1);
      load(u + 2);
      load_o(u + 2);
      pin_loads();
      __syncthreads();
      next();
    }
  }
  if (!wave_live) return;
  // The two factors of dK and of dV: the second is a power of two, exact where it is subnormal.
  float fk = pow2(-kTop) * a.scale, fk2 = pow2(-kp) / dsc, fv = pow2(-kTop - kp), fv2 = 1.0f / psc;
  const float z = probe_finite<kDT>(dk, probe_finite<kDT>(dv, fk * 0.0f));
  if (__builtin_amdgcn_ballot_w64(key < a.SK && !(z == 0.0f)) != 0) {
    scored_keys_fp32<D>(a, b, hk, kw0, t0, n, u0, u0 + steps, sm.u.o[w], dk, dv, late(lane));
    fk = a.scale, fk2 = fv = fv2 = 1.0f;
  }
  const int lane_e = late(lane);
  const int64_t stride = static_cast<int64_t>(2) * HK * D;
  store_rows<D>(dk, fk, fk2, sm.u.o[w], dkv, stride, a.SK - kw0, lane_e);
  store_rows<D>(dv, fv, fv2, sm.u.o[w], dkv + stride / 2, stride, a.SK - kw0, lane_e);
}

template <int D, int MODS>
__device__ __forceinline__ void scored_queries(const ScoredArgs& a, ScoredSmem<D>& sm, int item, int chunk) {
  constexpr int kKS = D / 16, kDT = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int off = a.SK - a.SQ, bh = item / a.nqb, qb = item % a.nqb, b = bh / a.H, h = bh % a.H, hk = h / a.G;
  const int qw0 = qb * kBlock + w * kRows, qi = qw0 + j, qc = min(qi, a.SQ - 1), pos = qc + off;
  const int prefix = prefix_of(a, b);
  const int32_t* all_ids = ids_of(a, b);
  const int end = last_key(a, min(qb * kBlock + kBlock, a.SQ) - 1 + off, prefix) + 1;
  const int lim = last_key(a, pos, prefix);
  const int lo = last_key(a, min(qw0, a.SQ - 1) + off, prefix);
  const int hi = last_key(a, min(qw0 + kRows, a.SQ) - 1 + off, prefix);
  // No key that is seen after its query; the wave's first position (past the last query: the last).
  const bool ordered = a.causal && prefix == 0;
  const int lo_pos = min(qw0, a.SQ - 1) + off;
  const bool wave_live = qw0 < a.SQ;
  int t0 = 0, t1 = (end + kRows - 1) / kRows;
  Ids ids{0, 0, 0, true};
  if (all_ids != nullptr) {
    ids.take(all_ids[pos]);
    int first, last;
    find_ids(sm.ids, ids, all_ids, 0, end, w, tid, first, last);
    t0 = first / kRows, t1 = first < last ? (last + kRows - 1) / kRows : t0;
  }
  t0 += chunk * a.chq, t1 = min(t1, t0 + a.chq);
  float* dq_rows = a.dq + (((static_cast<int64_t>(chunk) * a.B + b) * a.SQ + qw0) * a.H + h) * D;
  if (t0 >= t1) {  // no key was seen
    for (int i = lane; i < min(a.SQ - qw0, kRows) * (D / 4); i += 64) {
      st4(dq_rows + static_cast<int64_t>(i / (D / 4)) * a.H * D + i % (D / 4) * 4, f4{});
    }
    return;
  }
  const Operand kop{reinterpret_cast<const char*>(a.k.p + b * a.k.sb + hk * a.k.sh),
                    static_cast<unsigned>(a.k.ss) * 4u};
  const Operand vop{reinterpret_cast<const char*>(a.v.p + b * a.v.sb + hk * a.v.sh),
                    static_cast<unsigned>(a.v.ss) * 4u};
  Stage<D, kW> st;
  int id_next = 0;
  auto load = [&](int t) {
    st.load(kop, vop, t * kRows, a.SK - 1, w, lane);
    if (all_ids != nullptr && w == 0) id_next = all_ids[min(t * kRows + j, a.SK - 1)];
  };
  auto store = [&](int t) {
    const int put = t & 1;
    st.store(sm.u.t[put].a, sm.u.t[put].b, sm.ua[put], sm.ub[put], w, lane);
    if (all_ids != nullptr && w == 0) sm.ids.tile[put][j] = t * kRows + j < a.SK ? id_next : -1;
  };
  Pair qB[kKS], gB[kKS];
  const int kp = half_log2(a.SK);
  float uq, ug, L, Dq;  // L: kp - L log2 e
  {
    OwnRows<D> oq, og, oo;
    load(t0);
    oq.load(a.q.p + b * a.q.sb + h * a.q.sh + qc * a.q.ss, g);
    og.load(a.d_o.p + b * a.d_o.sb + h * a.d_o.sh + qc * a.d_o.ss, g);
    oo.load(a.o + ((static_cast<int64_t>(b) * a.SQ + qc) * a.H + h) * D, g);
    L = a.lse[static_cast<int64_t>(bh) * a.SQ + qc];
    Dq = 0.0f;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) {
#pragma unroll
      for (int e = 0; e < 8; ++e) Dq = fmaf(og.x[ks][e / 4][e % 4], oo.x[ks][e / 4][e % 4], Dq);
    }
    Dq = pair_sum(Dq) * pow2(kTop);  // (dP and D times 2^kTop meet K's unit)
    L = ids.mine < 0 ? 0.0f : shifted_l(L, kp);  // (as for the key blocks)
    uq = oq.split(sign_of(a.scale), qB);
    ug = og.split(1.0f, gB);
    store(t0);
    load(t0 + 1);
  }
  f16v dq[kDT];
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt) dq[dt] = zero16();
  const float cs = fabsf(a.scale) * kLog2e * ((MODS & 2) != 0 ? a.unit : 1.0f) * uq, cg = ug;
  const float slope2 = (MODS & 1) != 0 ? slope_of(a, h) : 0.0f;
  const float f2 = (MODS & 2) != 0 ? a.cap2 : 1.0f;
  Places places;
  if constexpr ((MODS & 1) != 0) places.set(slope2);
  float dsc = kMaxScale;
  const int roff0 = row_off<D>(j, g), coff0 = col_off<D>(lane);

  auto tile = [&](int t, int sees) {
    const int roff = late(roff0), coff = late(coff0), cur = t & 1, kt0 = t * kRows;
    store(t + 1);
    const Tile<D>&K = sm.u.t[cur].a, &V = sm.u.t[cur].b;
    f16v s = zero16(), dp = zero16();
    {
      h8 x[kKS];
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const Pair k = ld_row<D>(K, roff ^ row_step(ks));
        x[ks] = k.h;
        s = mma_small(k, qB[ks], s);
      }
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) s = mma(x[ks], qB[ks].h, s);
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        const Pair v = ld_row<D>(V, roff ^ row_step(ks));
        x[ks] = v.h;
        // (The key blocks' order: their A operand is this B.)
        dp = mma(v.l, gB[ks].h, dp);
        dp = mma(v.h, gB[ks].l, dp);
      }
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) dp = mma(x[ks], gB[ks].h, dp);
    }
    load(t + 2);
    pin_loads();
    if constexpr ((MODS & 2) != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 uk = ld4(&sm.ua[cur][8 * i + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * i + e] *= cs * uk[e];
      }
      if constexpr ((MODS & 4) != 0) s *= a.unit_rest;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 uv = ld4(&sm.ub[cur][8 * i + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * i + e] = fmaf(dp[4 * i + e], cg * uv[e], -Dq);
    }
    if constexpr ((MODS & 2) != 0) capped(s, [&](int r, float slope) { dp[r] *= slope; });
    float l = L;
    if constexpr ((MODS & 1) != 0) {
      auto f = [&](int i) {
        if constexpr ((MODS & 2) != 0) return f4{f2, f2, f2, f2};
        return ld4(&sm.ua[cur][8 * i + 4 * g]) * cs;
      };
      const float base = static_cast<float>(pos - 4 * g - kt0);
      if (fabsf(slope2) <= kSteep && (ordered || kt0 + kRows - 1 <= lo_pos)) {
        l = fmaf(-slope2, base, L);
        scale_add(s, f, [&](int r) { return places.by[r]; });
      } else {
        scale_add(s, f, [&](int r) { return far_by<-1>(r, slope2, base); });
      }
    }
    if (sees == kSome) {
      hide(s, 0, ids.mine >= 0 ? lim - kt0 - 4 * g : -1);
      if (all_ids != nullptr) hide_others(s, sm.ids.tile[cur], ids.mine, g);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f4 uk = ld4(&sm.ua[cur][8 * i + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * i + e;
        dp[r] = exp2_hw(MODS == 0   ? fmaf(s[r], factor(cs, uk[e]), L)
                        : MODS == 2 ? fmaf(s[r], f2, L)
                                    : s[r] + l) * dp[r] * uk[e];
      }
    }
    pin_acc(dq);
    const float md = max_weight(dp);
    if (__builtin_amdgcn_ballot_w64(md * dsc > kMaxWeight) != 0) {
      fit_scale(md, dsc, dq);
      pin_acc(dq);
    }
    const Pair p0 = split_acc<0>(dp, dsc), p1 = split_acc<1>(dp, dsc);
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt) {
      dq[dt] = mma3(ld_col<D>(K, coff ^ col_step(dt), 0), p0, dq[dt]);
      dq[dt] = mma3(ld_col<D>(K, coff ^ col_step(dt), 1), p1, dq[dt]);
    }
  };
  auto seen = [&](int t) {
    const int sees = !wave_live || t * kRows > hi ? kNone : t * kRows + kRows - 1 <= lo ? kAll : kSome;
    return all_ids == nullptr || sees == kNone ? sees : among(sm.ids.tile[t & 1][j], ids, sees);
  };
  __syncthreads();
  int t = t0, sees;
  while (t < t1) {
    while (t < t1 && (sees = seen(t)) != kNone) {
      tile(t, sees);
      __syncthreads();
      ++t;
    }
    while (t < t1 && seen(t) == kNone) {
      store(t + 1);
      load(t + 2);
      pin_loads();
      __syncthreads();
      ++t;
    }
  }
  if (!wave_live) return;
  float f = pow2(-kTop) * a.scale, fq = pow2(-kp) / dsc;
  if (__builtin_amdgcn_ballot_w64(qi < a.SQ && !(probe_finite<kDT>(dq, f * 0.0f) == 0.0f)) != 0) {
    scored_queries_fp32<D>(a, b, h, qw0, t0, t1, sm.u.o[w], dq, late(lane));
    f = a.scale, fq = 1.0f;
  }
  store_rows<D>(dq, f, fq, sm.u.o[w], dq_rows, static_cast<int64_t>(a.H) * D, a.SQ - qw0, late(lane));
}

template <int D, int MODS, int WAVES>
__global__ void __launch_bounds__(64 * kW) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES)))
bwd_scored_kernel(ScoredArgs a) {
  __shared__ __attribute__((aligned(16))) ScoredSmem<D> sm;
  const int id = static_cast<int>(blockIdx.x), pairs = a.B * (a.H / a.G);
  const int per_k = a.nkb * a.nck, per_q = a.nqb * a.ncq, keys = per_k * pairs;
  if (id < keys) {
    // Causal: the low blocks (they are seen by every later query) first.
    const int item = a.causal ? id % pairs * per_k + id / pairs : xcd_remap(id, keys);
    const int pair = item / per_k, in = item - pair * per_k, kb = in / a.nck;
    scored_keys<D, MODS>(a, sm, pair * a.nkb + kb, in - kb * a.nck);
  } else {
    const int BH = a.B * a.H, i = id - keys;
    const int item = a.causal ? i % BH * per_q + per_q - 1 - i / BH : xcd_remap(i, per_q * BH);
    const int bh = item / per_q, in = item - bh * per_q, qb = in / a.ncq;
    scored_queries<D, MODS>(a, sm, bh * a.nqb + qb, in - qb * a.ncq);
  }
}
// out = sum_c part[c], of `n` vectors of four, chunks in order.
__global__ void __launch_bounds__(256) sum_scored_kernel(const float* part, float* out, int64_t n, int nc) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  f4 x{};
#pragma unroll 4
  for (int c = 0; c < nc; ++c) x += ld4(part + (c * n + i) * 4);
  st4(out + i * 4, x);
}

template <int MODS>
const void* fwd_fn(int d) {
  return d == 32    ? reinterpret_cast<const void*>(fwd_scored_kernel<32, MODS, 4>)
         : d == 128 ? reinterpret_cast<const void*>(fwd_scored_kernel<128, MODS, 2>)
                    : reinterpret_cast<const void*>(fwd_scored_kernel<64, MODS, 3>);
}
template <int MODS>
const void* bwd_fn(int d) {
  return d == 32    ? reinterpret_cast<const void*>(bwd_scored_kernel<32, MODS, 3>)
         : d == 128 ? reinterpret_cast<const void*>(bwd_scored_kernel<128, MODS, 1>)
                    : reinterpret_cast<const void*>(bwd_scored_kernel<64, MODS, 2>);
}
int mods(const ScoredArgs& a) {
  if (a.unit_rest != 1.0f) return 7;
  return (a.slopes != nullptr ? 1 : 0) + (a.cap2 != 0.0f ? 2 : 0);
}
int64_t blocks_of(int64_t rows) { return (rows + kBlock - 1) / kBlock; }

}  // namespace

int64_t scored_blocks(int64_t b, int64_t heads, int64_t rows) { return b * heads * blocks_of(rows); }

// Chunks of a walk of `steps`, and their length: none until the walk is `most` times as long as `target`.
static void cut(int64_t steps, int64_t target, double most, int* n, int* length) {
  const int64_t want = steps > most * target ? (steps + target - 1) / target : 1;
  *length = static_cast<int>(std::max<int64_t>(1, (steps + want - 1) / want));
  *n = static_cast<int>(std::max<int64_t>(1, (steps + *length - 1) / *length));
}
// The part of sq x sk pairs that a causal mask leaves (documents and prefixes are on the device).
static double seen_part(int64_t sq, int64_t sk, int causal) {
  return causal ? 1.0 - 0.5 * static_cast<double>(sq) / static_cast<double>(sk) : 1.0;
}

ScoredPlan scored_plan(int64_t b, int64_t h, int64_t sq, int64_t sk, int64_t d) {
  ScoredPlan p{};
  p.nc = 1;
  if (b == 0 || sq == 0 || sk == 0) return p;
  const int64_t steps = (sk + kRows - 1) / kRows, blocks = scored_blocks(b, h, sq);
  const int64_t slots = 256 * (d == 32 ? 4 : d == 64 ? 3 : 2);
  // Chunks of the keys, as many as run at once (one more is a second round: 2 x 32 heads 512 x 4097 d 128 two
  // chunks 297 us, three 320; 1 x 32 heads four 158, five 193; 5 x 12 heads of 1000 d 64 whole 79, two 92), of 2
  // tiles or more, where that saves the 3 tiles that a join takes as long as (6 heads 240 x 240 d 64: whole 17.4,
  // in four 12.5). The join reads them four at a time: more than sqrt(8 steps) take longer there than they save (a
  // tile is some eight chunks of a join: one query to 131072 keys, 683 chunks 230 us, 179 96).
  const int64_t most = std::max<int64_t>(1, static_cast<int64_t>(sqrt(8.0 * static_cast<double>(steps))));
  const int64_t fit = std::min(most, blocks <= slots ? slots / blocks : 1);
  const int64_t longest = std::max<int64_t>(2, (steps + fit - 1) / fit);
  if (fit > 1 && steps - longest >= 3) {
    p.chunk = static_cast<int>(longest);
    p.nc = static_cast<int>((steps + longest - 1) / longest);
  }
  if (p.nc > 1) {
    const size_t parts = static_cast<size_t>(p.nc) * b * h * sq;
    p.l_part = parts * d * sizeof(float);
    p.bytes = p.l_part + parts * sizeof(double);
  }
  return p;
}

ScoredBackwardPlan scored_backward_plan(int64_t b, int64_t h, int64_t hk, int64_t sq, int64_t sk, int64_t d,
                                        int causal) {
  ScoredBackwardPlan p{1, 1, 1, 1, 0, 0};
  if (sq == 0 || sk == 0) return p;
  const int64_t slots = 256 * (d == 32 ? 3 : d == 64 ? 2 : 1), g = h / hk;
  const int64_t tq = (sq + kRows - 1) / kRows, tk = (sk + kRows - 1) / kRows;
  // A step of a key block takes four products, of a query block three. Chunks of 24 products or more.
  const double all = (static_cast<double>(scored_blocks(b, hk, sk)) * g * tq * 4 +
                      static_cast<double>(scored_blocks(b, h, sq)) * tk * 3) * seen_part(sq, sk, causal);
  const int64_t target = std::max<int64_t>(24, static_cast<int64_t>(all / slots) + 1);
  // (Whole walks of up to 2.5 targets end beside the others': 2 x 16 heads s 1024 d 64 causal 91, cut at 1.5 98.)
  cut(g * tq, (target + 3) / 4, 2.5, &p.nck, &p.chk);
  cut(tk, (target + 2) / 3, 2.5, &p.ncq, &p.chq);
  const size_t q = static_cast<size_t>(b) * h * sq * d * sizeof(float);
  const size_t k = static_cast<size_t>(b) * hk * sk * d * 2 * sizeof(float);
  p.k_part = p.ncq > 1 ? p.ncq * q : 0;
  p.bytes = p.k_part + (p.nck > 1 ? p.nck * k : 0);
  return p;
}

int launch_scored_forward(ScoredArgs a, int d, const ScoredPlan& plan, void* workspace, void* stream) {
  a.nqb = static_cast<int>(blocks_of(a.SQ));
  a.nc = plan.nc, a.chunk = plan.chunk;
  a.o_part = static_cast<float*>(workspace);
  a.l_part = reinterpret_cast<double*>(static_cast<char*>(workspace) + plan.l_part);
  void* args[] = {&a};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(int64_t{a.B} * a.H * a.nqb * a.nc);
  const int m = mods(a);
  const void* fn = m == 7   ? fwd_fn<7>(d)
                   : m == 3 ? fwd_fn<3>(d)
                   : m == 2 ? fwd_fn<2>(d)
                   : m == 1 ? fwd_fn<1>(d)
                            : fwd_fn<0>(d);
  const hipError_t err = hipLaunchKernel(fn, dim3(grid), dim3(64 * kW), args, 0, s);
  if (err != hipSuccess || a.nc == 1) return static_cast<int>(err);
  const void* join = d == 32    ? reinterpret_cast<const void*>(join_scored_kernel<32>)
                     : d == 128 ? reinterpret_cast<const void*>(join_scored_kernel<128>)
                                : reinterpret_cast<const void*>(join_scored_kernel<64>);
  const int64_t rows = int64_t{a.B} * a.H * a.SQ, per = 1024 / d;
  return static_cast<int>(hipLaunchKernel(join, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), args,
                                          0, s));
}

int launch_scored_backward(ScoredArgs a, int d, const ScoredBackwardPlan& plan, void* workspace, void* stream) {
  a.nqb = static_cast<int>(blocks_of(a.SQ)), a.nkb = static_cast<int>(blocks_of(a.SK));
  a.nc = 1;
  a.nck = plan.nck, a.chk = plan.chk, a.ncq = plan.ncq, a.chq = plan.chq;
  if (a.SQ == 0) a.nck = a.ncq = 1;
  float *q_part = static_cast<float*>(workspace), *dq = a.dq, *dkv = a.dkv;
  float* k_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.k_part);
  if (a.ncq > 1) a.dq = q_part;
  if (a.nck > 1) a.dkv = k_part;
  void* args[] = {&a};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int HK = a.H / a.G;
  const int64_t grid = scored_blocks(a.B, HK, a.SK) * a.nck + scored_blocks(a.B, a.H, a.SQ) * a.ncq;
  const int m = mods(a);
  const void* fn = m == 7   ? bwd_fn<7>(d)
                   : m == 3 ? bwd_fn<3>(d)
                   : m == 2 ? bwd_fn<2>(d)
                   : m == 1 ? bwd_fn<1>(d)
                            : bwd_fn<0>(d);
  hipError_t err = hipLaunchKernel(fn, dim3(static_cast<unsigned>(grid)), dim3(64 * kW), args, 0, s);
  auto sum = [&](const float* part, float* out, int64_t n, int nc) {
    void* sargs[] = {&part, &out, &n, &nc};
    return hipLaunchKernel(reinterpret_cast<const void*>(sum_scored_kernel),
                           dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), sargs, 0, s);
  };
  if (err == hipSuccess && a.ncq > 1) err = sum(q_part, dq, int64_t{a.B} * a.SQ * a.H * d / 4, a.ncq);
  if (err == hipSuccess && a.nck > 1) err = sum(k_part, dkv, int64_t{a.B} * a.SK * HK * d / 2, a.nck);
  return static_cast<int>(err);
}

}  // namespace fattn
