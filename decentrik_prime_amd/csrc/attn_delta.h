#pragma once
// The row kernel that both attention backwards launch first.
#include "attn_dev.h"

namespace {

// delta[h][t] = sum_d O[t][h][d] dO[t][h][d] (solution/k_attn.py:84-94): 16 lanes per (token, head), in
// rounds where the launch has fewer
__global__ __launch_bounds__(kAThreads) void attn_delta_kernel(const f16* __restrict__ o,
                                                               const f16* __restrict__ dout,
                                                               float* __restrict__ delta,
                                                               int64_t n_tokens, int nq) {
  for (int64_t pair = (int64_t)blockIdx.x * (kAThreads / 16) + (threadIdx.x >> 4); pair < n_tokens * nq;
       pair += (int64_t)gridDim.x * (kAThreads / 16)) {
    const int64_t t = pair / nq;
    const int hh = (int)(pair % nq), e = (threadIdx.x & 15) * 8;
    const int64_t off = t * nq * kHD + hh * kHD + e;
    const f16x8 ov = *reinterpret_cast<const f16x8*>(o + off);
    const f16x8 gv = *reinterpret_cast<const f16x8*>(dout + off);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __fadd_rn(s, __fmul_rn((float)ov[j], (float)gv[j]));
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) s = __fadd_rn(s, __shfl_xor(s, x));
    if ((threadIdx.x & 15) == 0) delta[(int64_t)hh * n_tokens + t] = s;
  }
}

}  // namespace
