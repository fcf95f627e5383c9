// Products of one to four rows, shared by the dense ones (gdn_linear_act.hip) and the experts' (gdn_experts.hip).
//
// A matrix instruction would multiply 12 to 15 empty rows, and a tile of 16 weight rows would leave most CUs without
// work: a wave takes two or four rows of the weights, each lane eight neighbouring values of every 512, which it
// multiplies as bf16 pairs (v_dot2_f32_bf16: exact products, fp32 sums); the lanes' sums meet at the end.  Bound by
// reading the weights, whole cache lines at a time, with all loads of 2048 values on their way at once.
#pragma once

#include "gdn_product.hpp"

namespace {

constexpr int kLanes8 = 64 * CPL;  // values of a row that a wave's load takes

__device__ __forceinline__ float dot8(const u32x4& a, const u32x4& b, float sum) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = a[j], y = b[j];  // (a bit cast of a vector's element itself takes the first one)
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, y), sum, false);
  }
  return sum;
}

// sums[r][i] = x_r . w_i over K, in every lane: R rows ldx apart, W weight rows at w[i].  What lies past K counts as zero.
template <int R, int W>
__device__ __forceinline__ void dot_rows(const uint16_t* x, int64_t ldx, const uint16_t* const (&w)[W], int K,
                                         float (&sums)[R][W]) {
  constexpr int CH = 4;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < W; ++i) sums[r][i] = 0.0f;
  for (int k0 = 0; k0 < K; k0 += CH * kLanes8) {
    u32x4 wv[CH][W], xv[CH][R];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (c > 0 && k0 + c * kLanes8 >= K) break;
      const int k = k0 + c * kLanes8 + lane * CPL, at = min(k, K - CPL);
#pragma unroll
      for (int i = 0; i < W; ++i) wv[c][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w[i] + at));
#pragma unroll
      for (int r = 0; r < R; ++r) xv[c][r] = *reinterpret_cast<const u32x4*>(x + r * ldx + at);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (c > 0 && k0 + c * kLanes8 >= K) break;
      const bool in = k0 + c * kLanes8 + lane * CPL < K;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const u32x4 wz = row_or_zero(in, wv[c][i]);
#pragma unroll
        for (int r = 0; r < R; ++r) sums[r][i] = dot8(wz, row_or_zero(in, xv[c][r]), sums[r][i]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < W; ++i) sums[r][i] = wave_sum(sums[r][i]);
}

}  // namespace
