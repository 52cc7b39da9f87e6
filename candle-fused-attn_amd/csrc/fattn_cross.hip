// Cross attention's launches, on the kernels of fattn_pair_kernels.h (kCross): queries and keys of their
// own lengths, key heads shared by groups of query heads, per-sample numbers of keys.
//
// A key block walks the queries of each head of its group in turn, so that dK and dV of a shared head
// are summed in one workgroup's registers, in a fixed order: no partial sums, no atomics. Rows of keys
// that a sample does not see are written as 0.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fattn_internal.h"
#include "fattn_pair_kernels.h"

namespace fattn {

int64_t cross_blocks(int64_t heads, int64_t s) { return heads * ((s + 4 * kRows - 1) / (4 * kRows)); }

bool cross_splits(int64_t, int64_t h, int64_t hk, int64_t sq, int64_t, int64_t) {
  return h / hk * sq <= 32;
}

int launch_cross_forward(View q, View k, View v, float* o, float* lse, int b, int h, int hk, int sq,
                         int sk, int d, const int32_t* key_lengths, float scale, void* stream) {
  const int nqb = (sq + 4 * kRows - 1) / (4 * kRows);
  FwdArgs a{q, k, v, o, lse, b, h, sq, nqb, scale, 0, sk, h / hk, key_lengths};
  void* args[] = {&a};
  const void* fn = d == 32    ? reinterpret_cast<const void*>(fwd_pair_kernel<32, false, 1, 4, 4, true>)
                   : d == 128 ? reinterpret_cast<const void*>(fwd_pair_kernel<128, false, 1, 4, 2, true>)
                              : reinterpret_cast<const void*>(fwd_pair_kernel<64, false, 1, 4, 3, true>);
  return static_cast<int>(hipLaunchKernel(fn, dim3(static_cast<unsigned>(cross_blocks(int64_t{b} * h, sq))), dim3(256), args, 0,
                                          static_cast<hipStream_t>(stream)));
}

int launch_cross_backward(View q, View k, View v, View d_o, const float* o, const float* lse, float* dq,
                          float* dkv, int b, int h, int hk, int sq, int sk, int d,
                          const int32_t* key_lengths, float scale, void* stream) {
  const int rows = 4 * kRows, nblk = (sk + rows - 1) / rows, nblk_q = (sq + rows - 1) / rows;
  BwdPairArgs a{};
  a.q = q, a.k = k, a.v = v, a.d_o = d_o, a.o = o, a.lse = lse, a.dq = dq, a.dkv = dkv;
  a.B = b, a.H = h, a.S = sq, a.SK = sk, a.G = h / hk, a.key_lengths = key_lengths, a.scale = scale;
  a.nblk = nblk, a.nkv = nblk * b * hk, a.nblk_q = nblk_q;
  a.give_up_bh = -1;
  void* args[] = {&a};
  const void* fn = d == 32 ? reinterpret_cast<const void*>(bwd_pair_kernel<32, false, false, 4, 3, true>)
                   : d == 128
                       ? reinterpret_cast<const void*>(bwd_pair_kernel<128, false, false, 4, 1, true>)
                       : reinterpret_cast<const void*>(bwd_pair_kernel<64, false, false, 4, 2, true>);
  return static_cast<int>(hipLaunchKernel(fn, dim3(static_cast<unsigned>(a.nkv + nblk_q * b * h)), dim3(256), args,
                                          0, static_cast<hipStream_t>(stream)));
}

}  // namespace fattn
