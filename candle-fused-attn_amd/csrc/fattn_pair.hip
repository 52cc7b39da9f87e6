// Self-attention's launches: which of the kernels of fattn_pair_kernels.h a shape takes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fattn_internal.h"
#include "fattn_pair_kernels.h"

namespace fattn {
namespace {

template <int D, int WAVES>
const void* fwd_pair_fn(int causal, int waves) {
  auto fn = [&](auto w) {
    constexpr int W = decltype(w)::value;
    constexpr int kOcc = W == 2 && D == 64 ? 2 : WAVES;  // (two waves share two tiles' LDS)
    return causal ? reinterpret_cast<const void*>(fwd_pair_kernel<D, true, 1, W, kOcc>)
                  : reinterpret_cast<const void*>(fwd_pair_kernel<D, false, 1, W, kOcc>);
  };
  if constexpr (D != 128) {
    if (waves == 2) return fn(Const<2>{});
  }
  return waves == 1 ? fn(Const<1>{}) : fn(Const<4>{});
}

// Waves per workgroup, each of 32 rows. Four share the staging of a tile, but over a short sequence
// those past its end only stage and wait, and the tiles ahead of the walk are staged for nothing:
// where there are workgroups enough for every CU without them, one wave takes s <= 32 and two
// s <= 64, with every tile staged before the walk (and, backward, the two kinds of workgroup of one
// (b, h) side by side). Fewer waves against four, us, 1536 (b, h), forward / backward: D 64, s 16
// 9.5 / 18 (16.0 / 41), s 32 11.5 / 22 (17.0 / 47), s 64 22.8 / 47 (24.4 / 66), causal s 64 25.3 / 49
// (25.2 / 72); D 128 s 32 27 / 56 (31 / 148), s 64 backward 122 (209), forward 46 (44: four);
// D 32 s 64 13.4 / 27 (15.9 / 39). With 64 (b, h), where the time is one workgroup's: D 64 s 64
// 8.1 / 11.4 (7.2 / 10.1), D 128 s 32 9.2 / 14.1 (8.1 / 13.4).
int workgroup_waves(int bh, int s, bool two) {
  if (bh <= 256 || s > 64) return 4;
  return s <= 32 ? 1 : two ? 2 : 4;
}

// Causal, s up to kSerialLength and up to kSerialBlocks key blocks: dV summed over the queries one at a
// time, on the fp32 matrix instruction (kSerial). The first keys of a causal row sum hundreds of terms
// of one sign, and there a sum of one rounding per query, as the composed fp32 path makes, and one of
// three per 16 queries drift apart by more than the reference's band around that path (5e-6;
// tests/parity.rs:218): at b 2 h 6 s 240 the composed path's dV is 6.0e-6 from fp64, so a correctly
// rounded one misses the band too. Small grids of the lengths for which the reference states the band
// (up to 240; here two blocks) keep to it, at a few us per call; all others take the faster and more
// accurate sum. With it / without, backward us: s 64 12.3 / 10.7, s 128 19.3 / 16.1, s 240 30.5 / 23.5
// (b 2 h 6: 31.0 / 24.0), and what longer walks would pay: s 512 51.5 / 36.9, s 2048 179 / 119, s 8192
// 689 / 447; D 128 s 1024 180 / 125.
constexpr int kSerialBlocks = 64, kSerialLength = 256;
template <int D, int WAVES>
const void* bwd_pair_fn(int causal, bool serial, int waves) {
  auto fn = [&](auto w) {
    constexpr int W = decltype(w)::value;
    if constexpr (W == 4) {  // (fewer waves: more than 256 (b, h))
      if (serial) return reinterpret_cast<const void*>(bwd_pair_kernel<D, true, true, W, WAVES>);
    }
    return causal ? reinterpret_cast<const void*>(bwd_pair_kernel<D, true, false, W, WAVES>)
                  : reinterpret_cast<const void*>(bwd_pair_kernel<D, false, false, W, WAVES>);
  };
  return waves == 1 ? fn(Const<1>{}) : waves == 2 ? fn(Const<2>{}) : fn(Const<4>{});
}

}  // namespace

bool wide_queries(int64_t wide, int64_t narrow, int s, int d) {
  // 64 queries per wave (256 per workgroup) halve what a query pays for reading, splitting and
  // waiting for the key tiles, but hold 2 waves per SIMD instead of 3 (D 64; 3 instead of 4 at D 32)
  // and halve the workgroups. Taken where every workgroup walks all keys, 1024 of them keep every CU
  // busy for two rounds or more, and no more than an eighth of their queries is padding that 128 per
  // workgroup would not have. Measured, 64 against 32 queries per wave, us: D 64, b h 256 s 1024
  // (1024 workgroups) 224 / 247, 512 x 512 121 / 131, 1024 x 256 77 / 83; too few, 64 x 1280 (320)
  // 119 / 108, 256 x 256 26 / 23; padded, 1024 x 300 140 / 121, 1024 x 640 425 / 419, and below s 128
  // half of it is (1536 x 32: 29 / 17). D 32, 256 x 1024 145 / 150, 512 x 512 81 / 81, but 1024 x 200
  // 46 / 43: from s 257 on. At D 128 their registers do not fit.
  const bool filled = 8 * 2 * wide <= 9 * narrow && (d == 64 || s > 256);
  return d != 128 && wide >= 1024 && filled;
}

int launch_forward(View q, View k, View v, float* o, float* lse, int b, int h, int s, int d,
                   float scale, int causal, void* stream) {
  const int nq = !causal && wide_queries(int64_t{b} * h * ((s + 255) / 256), int64_t{b} * h * ((s + 127) / 128),
                                           s, d)
                     ? 2
                     : 1;
  const int waves = workgroup_waves(b * h, s, d != 128), qb = kRows * waves * nq, nqb = (s + qb - 1) / qb;
  FwdArgs a{q, k, v, o, lse, b, h, s, nqb, scale, causal ? 1 : 0, s, 1, nullptr,
            1, 0, nullptr};
  void* args[] = {&a};
  const void* fn;
  if (nq == 2) {
    fn = d == 32 ? reinterpret_cast<const void*>(fwd_pair_kernel<32, false, 2, 4, 3>)
                 : reinterpret_cast<const void*>(fwd_pair_kernel<64, false, 2, 4, 2>);
  } else {
    fn = d == 32    ? fwd_pair_fn<32, 4>(causal, waves)
         : d == 128 ? fwd_pair_fn<128, 2>(causal, waves)
                    : fwd_pair_fn<64, 3>(causal, waves);
  }
  return static_cast<int>(hipLaunchKernel(fn, dim3(static_cast<unsigned>(nqb) * b * h),
                                          dim3(64u * waves), args, 0,
                                          static_cast<hipStream_t>(stream)));
}

int launch_backward(View q, View k, View v, View d_o, const float* o, const float* lse, float* dqkv,
                    float* part, unsigned long long* done, unsigned long long* epoch_slot,
                    unsigned long long epoch, int* ctrl, int b, int h, int s, int d, float scale,
                    int causal, int defer, int last, int give_up_bh, void* stream) {
  const int waves = workgroup_waves(b * h, s, true), rows = kRows * waves, nblk = (s + rows - 1) / rows;
  BwdPairArgs a{q, k, v, d_o, o, lse, dqkv, part, done, epoch_slot, epoch, ctrl, b, h, s,
                nblk * b * h, nblk, scale, causal ? 1 : 0, defer, last, give_up_bh,
                nullptr, nullptr, s, 1, nullptr, nblk, 1, 0, 1, 0};
  void* args[] = {&a};
  const bool serial = causal && s <= kSerialLength && a.nkv <= kSerialBlocks;
  // Waves per SIMD: what the registers allow without spills to the loop. At d 32 the third fits once
  // the fp32 fallback's loops are not unrolled (they set the register count); with it b64 h6 s240
  // takes 63 us (67 with two), causal b8 h12 s2048 352 (375).
  const void* fn = d == 32    ? bwd_pair_fn<32, 3>(causal, serial, waves)
                   : d == 128 ? bwd_pair_fn<128, 1>(causal, serial, waves)
                              : bwd_pair_fn<64, 2>(causal, serial, waves);
  return static_cast<int>(hipLaunchKernel(fn, dim3(2u * static_cast<unsigned>(a.nkv)),
                                          dim3(64u * waves), args, 0,
                                          static_cast<hipStream_t>(stream)));
}

}  // namespace fattn
