// Rotation of queries and keys by position, with their per-head RMSNorm in the same pass (gfx950).
//
//   y = x / sqrt(mean(x^2) + eps) * bf16(w)      per head, when norm weights are given
//   (a, b) -> (a cos - b sin, a sin + b cos)     pairs c < rot / 2 of the first rot channels, being
//                                                (c, c + rot / 2) or, interleaved, (2c, 2c + 1)
//   channels from rot on keep y
// cos and sin of pos * frequency[c] (times a factor that long contexts may ask for) come from a table
// that rotary_table fills once in float64, so the angle of a far position is as exact as a near one's.
#include "common.h"
#include "kernels.h"

namespace tessery {
namespace {

// A wavefront per (token, head), any even rot <= D <= 1024. Each lane owns whole pairs, so a row
// may be rotated in place.
template <typename T>
__global__ __launch_bounds__(256) void rotary_any(RotaryArgs a) {
  const int heads = a.H + a.KV;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<uint64_t>(a.tokens) * heads) return;  // wavefront-uniform
  const int lane = threadIdx.x & 63;
  const uint32_t token = static_cast<uint32_t>(row / heads);
  const int head = static_cast<int>(row - static_cast<uint64_t>(token) * heads);
  const bool isq = head < a.H;
  const T* x = isq ? static_cast<const T*>(a.q) + static_cast<size_t>(token) * a.in_q_row + head * a.D
                   : static_cast<const T*>(a.k) + static_cast<size_t>(token) * a.in_k_row +
                         (head - a.H) * a.D;
  T* y = isq ? static_cast<T*>(a.q_out) + static_cast<size_t>(token) * a.out_q_row + head * a.D
             : static_cast<T*>(a.k_out) + static_cast<size_t>(token) * a.out_k_row +
                   (head - a.H) * a.D;
  const uint16_t* w = isq ? a.q_norm : a.k_norm;
  float inv = 1.0f;
  if (w) {
    float squares = 0.0f;
    for (int c = lane; c < a.D; c += 64) {
      const float v = static_cast<float>(x[c]);
      squares = fmaf(v, v, squares);
    }
    inv = 1.0f / sqrtf(wave_sum(squares) / static_cast<float>(a.D) + a.eps);
  }
  auto at = [&](int c) {
    const float v = static_cast<float>(x[c]);
    return w ? v * inv * bf16_to_float(w[c]) : v;
  };
  const uint32_t pos = a.positions ? a.positions[token] : token % a.S;
  const int half = a.rot >> 1;
  const bool known = pos < a.table_rows;
  const float* cs = a.table + static_cast<size_t>(known ? pos : 0) * a.rot;
  for (int p = lane; p < half; p += 64) {
    const int c0 = a.interleaved ? 2 * p : p, c1 = a.interleaved ? 2 * p + 1 : p + half;
    const float u = at(c0), v = at(c1), cv = cs[p], sv = cs[half + p];
    y[c0] = static_cast<T>(known ? fmaf(u, cv, -(v * sv)) : 0.0f);
    y[c1] = static_cast<T>(known ? fmaf(u, sv, v * cv) : 0.0f);
  }
  for (int c = a.rot + lane; c < a.D; c += 64) y[c] = static_cast<T>(known ? at(c) : 0.0f);
}

__global__ __launch_bounds__(256) void rotary_table(const double* __restrict__ frequencies,
                                                    float* __restrict__ table, uint64_t n, int half,
                                                    double factor) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const uint64_t pos = i / half;
  const int c = static_cast<int>(i - pos * half);
  const double angle = static_cast<double>(pos) * frequencies[c];
  float* row = table + pos * 2 * half;
  row[c] = static_cast<float>(cos(angle) * factor);
  row[half + c] = static_cast<float>(sin(angle) * factor);
}

}  // namespace

bool rotary_fits(uint64_t tokens, uint64_t heads, uint64_t dim) {
  // a launch's work items stay below 2^32
  return tokens && heads && dim && dim <= 1024 && tokens * heads < (1ull << 26);
}

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t st) {
  const uint64_t rows = static_cast<uint64_t>(a.tokens) * (a.H + a.KV);
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
  if (a.f16)
    rotary_any<_Float16><<<grid, 256, 0, st>>>(a);
  else
    rotary_any<float><<<grid, 256, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t launch_rotary_table(const double* frequencies, float* table, uint32_t positions, int rot,
                               float factor, hipStream_t st) {
  const uint64_t n = static_cast<uint64_t>(positions) * (rot / 2);
  rotary_table<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(
      frequencies, table, n, rot / 2, static_cast<double>(factor));
  return hipGetLastError();
}

}  // namespace tessery
