// Projection of fp16 activations with its epilogue (route linear_f16), gfx950.
//
//   out = act(x W^T + bias) + residual       x [M, K], W [N, K], residual, out [M, N], bias [N]
// The products of fp16 values are exact in fp32 and are summed in fp32 on MFMA; bias, activation and
// residual are applied to the fp32 sum and one rounding to the output's type ends it.
#include "common.h"
#include "kernels.h"

#include <math.h>

namespace tessery {
namespace {

__device__ __forceinline__ float activate(float y, int act) {
  switch (act) {
    case kActRelu:
      return y < 0.0f ? 0.0f : y;
    case kActGelu:
      return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    case kActGeluTanh:  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (y + 0.044715 y^3)
      return y / (1.0f + expf(-1.5957691216057308f * fmaf(0.044715f * y * y, y, y)));
    case kActSilu:
      return y / (1.0f + expf(-y));
    default:
      return y;
  }
}

// Four consecutive columns n .. n + 3 of row m.
__device__ __forceinline__ void finish4(const LinearF16Args& a, int m, int n, floatx4 y) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j >= a.N) return;
    float r = activate(y[j] + (a.bias ? a.bias[n + j] : 0.0f), a.act);
    const size_t at = static_cast<size_t>(m) * a.N + n + j;
    if (a.residual) r += static_cast<float>(a.residual[at]);
    if (a.out_f32)
      static_cast<float*>(a.out)[at] = r;
    else
      static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(r);
  }
}

// 64 x 64 outputs a workgroup, 32 x 32 a wavefront (v_mfma_f32_32x32x16_f16: lane (r = l % 32,
// g = l / 32) supplies A[r][8g..8g+7] and B[8g..8g+7][r] and holds D[8a + 4g + c][r] in element
// 4a + c), 32 of K at a time through registers into LDS. A is W and B is x, so that a lane's four
// elements are neighbours in a row of out. Any M, N and K.
__global__ __launch_bounds__(256) void linear_f16_any(LinearF16Args a) {
  constexpr int KT = 32, ROW = KT + 8;
  __shared__ __attribute__((aligned(16))) _Float16 ws[64 * ROW], xs[64 * ROW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n0 = blockIdx.x * 64, m0 = blockIdx.y * 64;
  const int lr = tid >> 2, lc = (tid & 3) * 8;
  const bool whole = a.K % 8 == 0;
  auto fetch = [&](const _Float16* p, int row, int rows, int k) {
    half8 v = {};
    if (row < rows) {
      const _Float16* at = p + static_cast<size_t>(row) * a.K + k;
      if (whole) {
        if (k < a.K) v = *reinterpret_cast<const half8*>(at);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k + j < a.K) v[j] = at[j];
      }
    }
    return v;
  };
  floatx16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
  const int nw = (wave & 1) * 32, mw = (wave >> 1) * 32, r = lane & 31, g = lane >> 5;
  for (int k = 0; k < a.K; k += KT) {
    const half8 wv = fetch(a.w, n0 + lr, a.N, k + lc), xv = fetch(a.x, m0 + lr, a.M, k + lc);
    __syncthreads();
    *reinterpret_cast<half8*>(ws + lr * ROW + lc) = wv;
    *reinterpret_cast<half8*>(xs + lr * ROW + lc) = xv;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KT / 16; ++s) {
      const half8 af = *reinterpret_cast<const half8*>(ws + (nw + r) * ROW + 16 * s + 8 * g);
      const half8 bf = *reinterpret_cast<const half8*>(xs + (mw + r) * ROW + 16 * s + 8 * g);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(af, bf, acc, 0, 0, 0);
    }
  }
  const int m = m0 + mw + r;
  if (m >= a.M) return;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    finish4(a, m, n0 + nw + 8 * q + 4 * g,
            floatx4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]});
}

}  // namespace

hipError_t launch_linear_f16(const LinearF16Args& a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.N + 63) / 64), static_cast<unsigned>((a.M + 63) / 64));
  linear_f16_any<<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace tessery
