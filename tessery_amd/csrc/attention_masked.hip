// Attention with score functions and masks for gfx950 (route attention_masked).
//
//   s_ij = scale q_i . k_j ;  s_ij = cap tanh(s_ij / cap) with a cap
//   s_ij -= slope_h |i - j|, or += table_h[clamp(j - i, -radius, radius) + radius]
//   out_i = sum_j softmax_j(s_ij) v_j over the keys lo_i <= j < hi_i; zeros where there is none
// Every mask here is a range of keys: hi_i is the row's length, i + 1 (causal) or max(i + 1, prefix_b),
// i + window and the end of the token's span, whichever is least; lo_i the most of 0, i - window + 1 and
// the span's start. kv head = h / (H / KV).
#include "common.h"
#include "kernels.h"

#include <math.h>

namespace tessery {
namespace {

struct KeyRange {
  int lo, hi;
};

__device__ __forceinline__ KeyRange key_range(const MaskedArgs& a, int b, int i) {
  const uint32_t S = static_cast<uint32_t>(a.S);
  int hi = static_cast<int>(min(a.lengths[b], S)), lo = 0;
  if (a.mask == kMaskCausal) hi = min(hi, i + 1);
  if (a.mask == kMaskPrefix) hi = min(hi, max(i + 1, static_cast<int>(min(a.prefix[b], S))));
  if (a.window) {
    lo = max(lo, i - a.window + 1);
    hi = min(hi, a.window < a.S - i ? i + a.window : a.S);
  }
  if (a.spans) {
    const uint32_t* span = a.spans + 2 * (static_cast<size_t>(b) * S + i);
    lo = max(lo, static_cast<int>(min(span[0], S)));
    hi = min(hi, static_cast<int>(min(span[1], S)));
  }
  return {lo, hi};
}

// log2(e) times the bias, so that finite values stay finite (a mask of the type's lowest value is no
// infinity: a row that holds nothing else attends its keys alike)
__device__ __forceinline__ float log2_bias(float x) {
  const float y = x * kLog2e;
  return y == -INFINITY && x != -INFINITY ? -3.402823466e38f : y;
}

__device__ __forceinline__ float capped(float s, float cap) { return cap * tanhf(s / cap); }

// One row by one wavefront, lanes across the channels, keys one after the other: online softmax with
// the running maximum and sum in fp32.
template <typename T>
__device__ __forceinline__ void masked_row(const MaskedArgs& a, int b, int i, int h, int lane) {
  const KeyRange keys = key_range(a, b, i);
  const int kvh = h / (a.H / a.KV);
  const size_t token = static_cast<size_t>(b) * a.S;
  const T* q = static_cast<const T*>(a.q) + (token + i) * a.q_row + h * a.D;
  const T* k = static_cast<const T*>(a.k) + token * a.k_row + kvh * a.D;
  const T* v = static_cast<const T*>(a.v) + token * a.v_row + kvh * a.D;
  const float slope = a.bias_kind == kBiasSlopes ? a.bias[h] : 0.0f;
  const float* table = a.bias_kind == kBiasTable ? a.bias + h * (2 * static_cast<size_t>(a.radius) + 1) : nullptr;
  float qv[4], acc[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    qv[c] = lane + 64 * c < a.D ? static_cast<float>(q[lane + 64 * c]) : 0.0f;
    acc[c] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;
  for (int j = keys.lo; j < keys.hi; ++j) {
    const T* kr = k + static_cast<size_t>(j) * a.k_row;
    const T* vr = v + static_cast<size_t>(j) * a.v_row;
    float dot = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 64 * c < a.D) dot = fmaf(qv[c], static_cast<float>(kr[lane + 64 * c]), dot);
    float s = wave_sum(dot) * a.scale;
    if (a.cap > 0.0f) s = capped(s, a.cap);
    s *= kLog2e;
    if (a.bias_kind == kBiasSlopes) s = fmaf(-slope * kLog2e, static_cast<float>(abs(i - j)), s);
    if (table) s += log2_bias(table[min(max(j - i, -a.radius), a.radius) + a.radius]);
    const float next = fmaxf(top, s);
    const float base = next == -INFINITY ? 0.0f : next;
    const float old = exp2f(top - base), p = exp2f(s - base);
    sum = fmaf(sum, old, p);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 64 * c < a.D)
        acc[c] = fmaf(p, static_cast<float>(vr[lane + 64 * c]), acc[c] * old);
    top = next;
  }
  T* out = static_cast<T*>(a.out) + ((token + i) * a.H + h) * a.D;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < a.D) out[lane + 64 * c] = static_cast<T>(acc[c] * inv);
}

template <typename T>
__global__ __launch_bounds__(256) void attn_masked_rows(MaskedArgs a) {
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const uint64_t per = static_cast<uint64_t>(a.S) * a.H;
  if (row >= a.B * per) return;  // wavefront-uniform
  const int b = static_cast<int>(row / per);
  const uint32_t rest = static_cast<uint32_t>(row - b * per);
  masked_row<T>(a, b, static_cast<int>(rest / a.H), static_cast<int>(rest % a.H),
                threadIdx.x & 63);
}

}  // namespace

bool attention_masked_fits(uint64_t B, uint64_t S, uint64_t H, uint64_t D) {
  // a launch's work items stay below 2^32
  return D % 8 == 0 && D <= 256 && B * S * H < (1ull << 26);
}

hipError_t launch_attention_masked(const MaskedArgs& a, hipStream_t st) {
  const uint64_t rows = static_cast<uint64_t>(a.B) * a.S * a.H;
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
  if (a.f16)
    attn_masked_rows<_Float16><<<grid, 256, 0, st>>>(a);
  else
    attn_masked_rows<float><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace tessery
