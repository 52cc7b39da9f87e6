// Cross attention's launches, on the kernels of fattn_pair_kernels.h (kCross): queries and keys of their
// own lengths, key heads shared by groups of query heads, per-sample numbers of keys.
//
// A key block walks the queries of each head of its group in turn, so that dK and dV of a shared head
// are summed in one workgroup's registers, in a fixed order: no atomics. Rows of keys that a sample does
// not see are written as 0. Where there are too few blocks for the chip their walks are cut into chunks,
// whose outputs are joined in order here: reruns are bit-identical either way.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "fattn_internal.h"
#include "fattn_pair_kernels.h"

namespace fattn {
namespace {

constexpr int kBlockRows = 4 * kRows;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Chunks of a walk of `steps`, and their length: none until the walk is twice as long as `target`.
void chunks(int64_t steps, int64_t target, int* n, int* length) {
  const int64_t want = steps >= 2 * target ? ceil_div(steps, target) : 1;
  *length = static_cast<int>(std::max<int64_t>(1, ceil_div(steps, want)));
  *n = static_cast<int>(std::max<int64_t>(1, ceil_div(steps, *length)));
}

// The chunks of sample b's keys that hold any (of `nc` chunks of `chunk` tiles).
__device__ __forceinline__ int chunks_of(const int32_t* key_lengths, int b, int SK, int nc, int chunk) {
  if (key_lengths == nullptr) return nc;
  const int keys = min(max(key_lengths[b], 0), SK), rows = chunk * kRows;
  return (keys + rows - 1) / rows;
}

// O and L of the chunks' [nc][b, s, h, d] and [nc][b, h, s]: O = sum_c w_c O_c / sum_c w_c, w_c =
// exp(L_c - max), L = max + log sum. D / 4 lanes a row.
template <int D>
__global__ void __launch_bounds__(256) join_forward_kernel(const float* o_part, const double* l_part,
                                                           float* o, float* lse, int B, int H, int S,
                                                           int SK, const int32_t* key_lengths, int nc,
                                                           int chunk) {
  constexpr int kLanes = D / 4;
  const int64_t rows = static_cast<int64_t>(B) * S * H;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (row >= rows) return;
  const int d = threadIdx.x % kLanes * 4;
  const int h = static_cast<int>(row % H), b = static_cast<int>(row / H / S);
  const int i = static_cast<int>(row / H % S);
  const int64_t at = (static_cast<int64_t>(b) * H + h) * S + i;
  const int n = chunks_of(key_lengths, b, SK, nc, chunk);
  double top = -__builtin_inf();
  for (int c = 0; c < n; ++c) {
    const double L = l_part[c * rows + at];
    top = L > top || L != L ? L : top;
  }
  float sum = 0.0f;
  f4 x{};
#pragma unroll 4
  for (int c = 0; c < n; ++c) {
    const float w = expf(static_cast<float>(l_part[c * rows + at] - top));
    sum += w;
    x += ld4(o_part + (c * rows + row) * D + d) * w;
  }
  st4(o + row * D + d, n == 0 ? f4{} : x * (1.0f / sum));
  if (d == 0) lse[at] = n == 0 ? kNegInf : static_cast<float>(top + logf(sum));
}

// out = sum_c part[c], of `per` vectors of four of each sample (blockIdx.y), chunks in order.
__global__ void __launch_bounds__(256) join_sum_kernel(const float* part, float* out, int64_t per, int SK,
                                                       const int32_t* key_lengths, int nc, int chunk) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= per) return;
  const int b = static_cast<int>(blockIdx.y);
  const int n = chunks_of(key_lengths, b, SK, nc, chunk);
  const int64_t at = (b * per + i) * 4, size = gridDim.y * per * 4;
  f4 x{};
#pragma unroll 4
  for (int c = 0; c < n; ++c) x += ld4(part + c * size + at);
  st4(out + at, x);
}

}  // namespace

int64_t cross_blocks(int64_t heads, int64_t s) { return heads * ceil_div(s, kBlockRows); }
int64_t cross_query_blocks(int64_t pairs, int64_t g, int64_t s, int wave_rows) {
  return pairs * ceil_div(g * ceil_div(s, wave_rows), 4);
}

CrossForwardPlan cross_forward_plan(int64_t b, int64_t h, int64_t hk, int64_t sq, int64_t sk, int64_t d) {
  CrossForwardPlan p{};
  p.nc = 1, p.chunk = static_cast<int>(ceil_div(sk, kRows));
  // The split kernel reads the keys once for 16 rows (the group's heads times the queries) and has the
  // fp32 matrix instruction's rate, but no prologue and every key's own workgroup: taken for up to 16
  // rows, where memory bounds both, and for little work (0.35 GFLOP, 8 us of it). Split / blocks, us (with
  // 6 us of a graph's launch): 8 x 8 heads 17 x 600 23.5 / 23.0, 1 head 500 x 500 14.9 / 23.3, d 128
  // 4 x 8 heads in 2 groups 12 x 1000 20.9 / 32.8; past it 16 x 8 heads 20 x 1500 46 / 34, 64 x 8 144 / 82.
  const int64_t rows = h / hk * sq, padded = ceil_div(rows, 16) * 16;
  p.split = rows <= 16 || 4.0 * padded * d * b * hk * sk <= 3.5e8;
  if (p.split) {
    p.bytes = split_plan(b, hk, rows, d, sk).bytes;
    return p;
  }
  // Chunks of the keys where the blocks do not fill the chip, of 8 tiles or more: d 128 2 x 16 heads
  // 100 x 3000 58 us (202 whole), 4 heads 2048 x 4096 60 (164). A grid that fills it loses by them: b 64
  // h 6 240 x 1024 116 in two chunks, 80 whole.
  const int64_t slots = 256 * (d == 32 ? 4 : d == 64 ? 3 : 2), blocks = cross_query_blocks(b * hk, h / hk, sq);
  const int64_t steps = ceil_div(sk, kRows);
  chunks(steps, std::max<int64_t>(8, ceil_div(blocks * steps, slots)), &p.nc, &p.chunk);
  if (p.nc > 1) {
    const size_t parts = static_cast<size_t>(p.nc) * b * h * sq;
    p.l_part = parts * d * sizeof(float);
    p.bytes = p.l_part + parts * sizeof(double);
  }
  return p;
}

CrossBackwardPlan cross_backward_plan(int64_t b, int64_t h, int64_t hk, int64_t sq, int64_t sk, int64_t d) {
  CrossBackwardPlan p{};
  p.ncq = p.nck = 1, p.chq = static_cast<int>(ceil_div(sk, kRows)), p.chk = 1;
  if (sq == 0 || sk == 0) return p;  // (nothing to walk, and nothing to join)
  const int64_t slots = 256 * (d == 32 ? 3 : d == 64 ? 2 : 1);
  const int64_t tq = ceil_div(sq, kRows), tk = ceil_div(sk, kRows), g = h / hk;
  // A step of a key block takes four products, of a query block three. Chunks as in the forward, of 20
  // products or more: forward and backward, us, 4 x 8 heads 1 x 4096 82 (235 whole), d 128 2 x 16 heads
  // 100 x 3000 221 (320), 1 head 500 x 500 45 (63); of 32 57, of 12 42, but d 128 4 x 8 heads in 2
  // groups 12 x 1000 74, 68 and 69.
  const int64_t all = cross_blocks(b * hk, sk) * g * tq * 4 + cross_query_blocks(b * hk, g, sq) * tk * 3;
  const int64_t target = std::max<int64_t>(20, ceil_div(all, slots));
  chunks(g * tq, ceil_div(target, 4), &p.nck, &p.chk);
  chunks(tk, ceil_div(target, 3), &p.ncq, &p.chq);
  const size_t q = static_cast<size_t>(b) * h * sq * d * sizeof(float);
  const size_t k = static_cast<size_t>(b) * hk * sk * d * 2 * sizeof(float);
  p.k_part = p.ncq > 1 ? p.ncq * q : 0;
  p.bytes = p.k_part + (p.nck > 1 ? p.nck * k : 0);
  return p;
}

int launch_cross_forward(View q, View k, View v, float* o, float* lse, int b, int h, int hk, int sq,
                         int sk, int d, const int32_t* key_lengths, float scale,
                         const CrossForwardPlan& plan, void* workspace, void* stream) {
  // 64 queries per wave where self-attention takes them.
  const int64_t pairs = int64_t{b} * hk;
  const bool wide = wide_queries(cross_query_blocks(pairs, h / hk, sq, 2 * kRows),
                                 cross_query_blocks(pairs, h / hk, sq), sq, d);
  const int nqb = static_cast<int>(cross_query_blocks(1, h / hk, sq, wide ? 2 * kRows : kRows));
  float* o_part = static_cast<float*>(workspace);
  double* l_part = reinterpret_cast<double*>(static_cast<char*>(workspace) + plan.l_part);
  const bool cut = plan.nc > 1;
  FwdArgs a{q, k, v, cut ? o_part : o, lse, b, h, sq, nqb, scale, 0, sk, h / hk, key_lengths, plan.nc,
            plan.chunk, cut ? l_part : nullptr};
  void* args[] = {&a};
  const void* fn = wide && d == 32   ? reinterpret_cast<const void*>(fwd_cross_kernel<32, 2, 4, 3>)
                   : wide && d == 64 ? reinterpret_cast<const void*>(fwd_cross_kernel<64, 2, 4, 2>)
                   : d == 32         ? reinterpret_cast<const void*>(fwd_cross_kernel<32, 1, 4, 4>)
                   : d == 128        ? reinterpret_cast<const void*>(fwd_cross_kernel<128, 1, 4, 2>)
                                     : reinterpret_cast<const void*>(fwd_cross_kernel<64, 1, 4, 3>);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(pairs * nqb * plan.nc);
  const hipError_t err = hipLaunchKernel(fn, dim3(grid), dim3(256), args, 0, s);
  if (err != hipSuccess || !cut) return static_cast<int>(err);
  const float* op = o_part;
  const double* lp = l_part;
  int nc = plan.nc, chunk = plan.chunk;
  void* jargs[] = {&op, &lp, &o, &lse, &b, &h, &sq, &sk, &key_lengths, &nc, &chunk};
  const void* join = d == 32    ? reinterpret_cast<const void*>(join_forward_kernel<32>)
                     : d == 128 ? reinterpret_cast<const void*>(join_forward_kernel<128>)
                                : reinterpret_cast<const void*>(join_forward_kernel<64>);
  const unsigned join_grid = static_cast<unsigned>(ceil_div(int64_t{b} * h * sq, 1024 / d));
  return static_cast<int>(hipLaunchKernel(join, dim3(join_grid), dim3(256), jargs, 0, s));
}

int launch_cross_backward(View q, View k, View v, View d_o, const float* o, const float* lse, float* dq,
                          float* dkv, int b, int h, int hk, int sq, int sk, int d,
                          const int32_t* key_lengths, float scale, const CrossBackwardPlan& plan,
                          void* workspace, void* stream) {
  const int nblk = (sk + kBlockRows - 1) / kBlockRows, nblk_q = static_cast<int>(cross_query_blocks(1, h / hk, sq));
  float* q_part = static_cast<float*>(workspace);
  float* k_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.k_part);
  BwdPairArgs a{};
  a.q = q, a.k = k, a.v = v, a.d_o = d_o, a.o = o, a.lse = lse;
  a.dq = plan.ncq > 1 ? q_part : dq, a.dkv = plan.nck > 1 ? k_part : dkv;
  a.B = b, a.H = h, a.S = sq, a.SK = sk, a.G = h / hk, a.key_lengths = key_lengths, a.scale = scale;
  a.nck = plan.nck, a.chk = plan.chk, a.ncq = plan.ncq, a.chq = plan.chq;
  a.nblk = nblk, a.nkv = nblk * b * hk * plan.nck, a.nblk_q = nblk_q;
  a.give_up_bh = -1;
  void* args[] = {&a};
  const void* fn = d == 32    ? reinterpret_cast<const void*>(bwd_cross_kernel<32, 4, 3>)
                   : d == 128 ? reinterpret_cast<const void*>(bwd_cross_kernel<128, 4, 1>)
                              : reinterpret_cast<const void*>(bwd_cross_kernel<64, 4, 2>);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t err = hipLaunchKernel(fn, dim3(static_cast<unsigned>(a.nkv + nblk_q * b * hk * plan.ncq)),
                                   dim3(256), args, 0, s);
  auto sum = [&](const float* part, float* out, int64_t per, const int32_t* lengths, int nc, int chunk) {
    void* jargs[] = {&part, &out, &per, &sk, &lengths, &nc, &chunk};
    return hipLaunchKernel(reinterpret_cast<const void*>(join_sum_kernel),
                           dim3(static_cast<unsigned>(ceil_div(per, 256)), static_cast<unsigned>(b)),
                           dim3(256), jargs, 0, s);
  };
  if (err == hipSuccess && plan.ncq > 1) {
    err = sum(q_part, dq, int64_t{sq} * h * d / 4, key_lengths, plan.ncq, plan.chq);
  }
  if (err == hipSuccess && plan.nck > 1) {
    err = sum(k_part, dkv, int64_t{sk} * hk * d / 2, nullptr, plan.nck, plan.chk);
  }
  return static_cast<int>(err);
}

}  // namespace fattn
