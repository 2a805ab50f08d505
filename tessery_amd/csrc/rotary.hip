// Rotation of queries and keys by position, with their per-head RMSNorm in the same pass (gfx950).
//
//   y = x / sqrt(mean(x^2) + eps) * bf16(w)      per head, when norm weights are given
//   (a, b) -> (a cos - b sin, a sin + b cos)     pairs c < rot / 2 of the first rot channels, being
//                                                (c, c + rot / 2) or, interleaved, (2c, 2c + 1)
//   channels from rot on keep y
// cos and sin of pos * frequency[c] (times a factor that long contexts may ask for) come from a table
// that rotary_table fills once in float64, so the angle of a far position is as exact as a near one's.
// Every channel of q and k is read and written once, and its arithmetic is a few operations: the bound is
// HBM. 16384 tokens of 24 fp16 heads of 128 channels with norms, 201 MB, take 47.7 us, 4.2 TB/s (a copy of
// 1 GiB reaches 5.15); one query of 24 tokens takes 4 us, of which nearly all is the launch.
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

template <int CTRL>
__device__ __forceinline__ float plus_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// The sum over each aligned run of N lanes, in all of them: lane pairs, quads, then mirrored halves of 8
// and 16 lanes, then the lane swaps of gfx950 (no trip through LDS).
template <int N>
__device__ __forceinline__ float run_sum(float x) {
  if constexpr (N >= 2) x = plus_dpp<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  if constexpr (N >= 4) x = plus_dpp<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  if constexpr (N >= 8) x = plus_dpp<0x141>(x);  // row_half_mirror
  if constexpr (N >= 16) x = plus_dpp<0x140>(x); // row_mirror
  if constexpr (N >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (N >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return x;
}

// Lanes of pieces: C channels a piece (16 bytes, or 2 channels where the sizes ask for it), two pieces a lane,
// D / 2C lanes a head (TP: up to a power of two, at most a wavefront). Lane j of the rotated channels holds pairs C j .. C j + C - 1 -
// the pieces at C j and rot / 2 + C j, or, interleaved, the two from 2 C j - so the turn stays in the lane
// and only the norm's sum crosses lanes. Blocks (x: tokens, y: parts of HP heads, those of q before those
// of k); a thread reads its table entries and weights once for HP heads of its token.
// Needs D and rot to be multiples of 2C: rows are then whole pieces too.
template <typename T, int C, int TP, int HP, bool INTERLEAVED, bool NORM>
__global__ __launch_bounds__(256) void rotary_pieces(RotaryArgs a, int q_parts) {
  constexpr int F = C < 4 ? C : 4;  // floats a read of the table
  typedef float few __attribute__((ext_vector_type(F)));
  typedef T piece __attribute__((ext_vector_type(C)));
  const int j = threadIdx.x % TP;
  const uint32_t token = blockIdx.x * (256 / TP) + threadIdx.x / TP;
  const bool isq = static_cast<int>(blockIdx.y) < q_parts;
  const int h0 = (static_cast<int>(blockIdx.y) - (isq ? 0 : q_parts)) * HP;
  const int heads = min(HP, (isq ? a.H : a.KV) - h0);
  const uint32_t at = min(token, a.tokens - 1);  // lanes past the end take part in the sums
  const T* const x = static_cast<const T*>(isq ? a.q : a.k) +
                     static_cast<size_t>(at) * (isq ? a.in_q_row : a.in_k_row) + h0 * a.D;
  T* const y = static_cast<T*>(isq ? a.q_out : a.k_out) +
               static_cast<size_t>(at) * (isq ? a.out_q_row : a.out_k_row) + h0 * a.D;
  const bool live = token < a.tokens && j < a.D / (2 * C);
  const bool turns = j < a.rot / (2 * C);
  const int c0 = INTERLEAVED ? 2 * C * j : turns ? C * j : 2 * C * j;
  const int c1 = INTERLEAVED || !turns ? c0 + C : c0 + (a.rot >> 1);
  const uint32_t pos = a.positions ? a.positions[at] : at % a.S;
  const bool known = pos < a.table_rows;

  piece p0[HP], p1[HP];
#pragma unroll
  for (int n = 0; n < HP; ++n) {
    p0[n] = p1[n] = piece{};
    if (live && n < heads) {
      p0[n] = *reinterpret_cast<const piece*>(x + n * a.D + c0);
      p1[n] = *reinterpret_cast<const piece*>(x + n * a.D + c1);
    }
  }
  float cs[C], sn[C];
#pragma unroll
  for (int c = 0; c < C; ++c) cs[c] = sn[c] = 0.0f;
  if (turns && known) {
    const float* const row = a.table + static_cast<size_t>(pos) * a.rot + C * j;
#pragma unroll
    for (int c = 0; c < C; c += F) {
      const few u = *reinterpret_cast<const few*>(row + c);
      const few v = *reinterpret_cast<const few*>(row + (a.rot >> 1) + c);
#pragma unroll
      for (int m = 0; m < F; ++m) {
        cs[c + m] = u[m];
        sn[c + m] = v[m];
      }
    }
  }
  float w0[C], w1[C];
  const float per_channel = 1.0f / static_cast<float>(a.D);
  if constexpr (NORM) {
    const uint16_t* const w = isq ? a.q_norm : a.k_norm;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      w0[c] = live ? bf16_to_float(w[c0 + c]) : 0.0f;
      w1[c] = live ? bf16_to_float(w[c1 + c]) : 0.0f;
    }
  }
#pragma unroll
  for (int n = 0; n < HP; ++n) {
    float u[C], v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      u[c] = static_cast<float>(p0[n][c]);
      v[c] = static_cast<float>(p1[n][c]);
    }
    if constexpr (NORM) {
      float squares = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) squares = fmaf(u[c], u[c], fmaf(v[c], v[c], squares));
      squares = run_sum<TP>(squares);
      const float mean = squares * per_channel + a.eps;
      // one instruction (1 ulp) where the mean of fp16 squares cannot be subnormal
      const float inv = sizeof(T) == 2 ? __builtin_amdgcn_rsqf(mean) : 1.0f / sqrtf(mean);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        u[c] = u[c] * inv * w0[c];
        v[c] = v[c] * inv * w1[c];
      }
    }
    piece r0, r1;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float f = u[c], g = v[c];
      if (turns) {
        // pair c of the lane: interleaved, its channels lie side by side
        const float first = INTERLEAVED ? (2 * c < C ? u[(2 * c) % C] : v[(2 * c) % C]) : u[c];
        const float second = INTERLEAVED ? (2 * c < C ? u[(2 * c + 1) % C] : v[(2 * c + 1) % C]) : v[c];
        f = fmaf(first, cs[c], -(second * sn[c]));
        g = fmaf(first, sn[c], second * cs[c]);
      }
      if constexpr (INTERLEAVED) {
        // unturned lanes keep their channels in place
        const float keep0 = 2 * c < C ? u[(2 * c) % C] : v[(2 * c) % C];
        const float keep1 = 2 * c < C ? u[(2 * c + 1) % C] : v[(2 * c + 1) % C];
        const T t0 = static_cast<T>(known ? (turns ? f : keep0) : 0.0f);
        const T t1 = static_cast<T>(known ? (turns ? g : keep1) : 0.0f);
        if (2 * c < C) {
          r0[(2 * c) % C] = t0;
          r0[(2 * c + 1) % C] = t1;
        } else {
          r1[(2 * c) % C] = t0;
          r1[(2 * c + 1) % C] = t1;
        }
      } else {
        r0[c] = static_cast<T>(known ? f : 0.0f);
        r1[c] = static_cast<T>(known ? g : 0.0f);
      }
    }
    if (live && n < heads) {
      if constexpr (HP > 1) {  // more rows than the caches hold: 5 to 10 % less time
        __builtin_nontemporal_store(r0, reinterpret_cast<piece*>(y + n * a.D + c0));
        __builtin_nontemporal_store(r1, reinterpret_cast<piece*>(y + n * a.D + c1));
      } else {
        *reinterpret_cast<piece*>(y + n * a.D + c0) = r0;
        *reinterpret_cast<piece*>(y + n * a.D + c1) = r1;
      }
    }
  }
}

template <typename T, int C, int TP, int HP>
hipError_t launch_pieces(const RotaryArgs& a, hipStream_t st) {
  const int q_parts = (a.H + HP - 1) / HP, parts = q_parts + (a.KV + HP - 1) / HP;
  const dim3 grid((a.tokens + 256 / TP - 1) / (256 / TP), static_cast<unsigned>(parts));
  if (a.interleaved) {
    if (a.q_norm) rotary_pieces<T, C, TP, HP, true, true><<<grid, 256, 0, st>>>(a, q_parts);
    else rotary_pieces<T, C, TP, HP, true, false><<<grid, 256, 0, st>>>(a, q_parts);
  } else {
    if (a.q_norm) rotary_pieces<T, C, TP, HP, false, true><<<grid, 256, 0, st>>>(a, q_parts);
    else rotary_pieces<T, C, TP, HP, false, false><<<grid, 256, 0, st>>>(a, q_parts);
  }
  return hipGetLastError();
}

template <typename T, int C, int TP>
hipError_t launch_lanes(const RotaryArgs& a, hipStream_t st) {
  // Four heads a thread share its table entries and weights: 16384 tokens of 24 heads of 128 with norms take
  // 49.8 us (a head 66, two 52.4, eight 52; stores past the caches then took it to 47.7). Few rows take a
  // head a thread, so that the chip has work.
  const bool few = static_cast<uint64_t>(a.tokens) * (a.H + a.KV) * TP < (1u << 20);
  return few ? launch_pieces<T, C, TP, 1>(a, st) : launch_pieces<T, C, TP, 4>(a, st);
}

template <typename T>
hipError_t launch_typed(const RotaryArgs& a, hipStream_t st) {
  constexpr int C = 16 / static_cast<int>(sizeof(T));
  const int lanes = a.D / (2 * C);
  if (a.D % (2 * C) == 0 && a.rot % (2 * C) == 0 && lanes <= 64) {
    if (lanes <= 4) return launch_lanes<T, C, 4>(a, st);
    if (lanes <= 8) return launch_lanes<T, C, 8>(a, st);
    if (lanes <= 16) return launch_lanes<T, C, 16>(a, st);
    return lanes <= 32 ? launch_lanes<T, C, 32>(a, st) : launch_lanes<T, C, 64>(a, st);
  }
  // Sizes that 16-byte pieces do not divide: 32 x 714 tokens of 8 heads of 80 channels, 40 of them rotated,
  // in fp16 take 16.1 us in pieces of two channels (52.6 as a wavefront per row).
  if (a.D % 4 == 0 && a.rot % 4 == 0 && a.D <= 256) {
    if (a.D <= 32) return launch_lanes<T, 2, 8>(a, st);
    if (a.D <= 64) return launch_lanes<T, 2, 16>(a, st);
    return a.D <= 128 ? launch_lanes<T, 2, 32>(a, st) : launch_lanes<T, 2, 64>(a, st);
  }
  const uint64_t rows = static_cast<uint64_t>(a.tokens) * (a.H + a.KV);
  rotary_any<T><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

bool rotary_fits(uint64_t tokens, uint64_t heads, uint64_t dim) {
  // a launch's work items stay below 2^32
  return tokens && heads && dim && dim <= 1024 && tokens * heads < (1ull << 26);
}

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t st) {
  return a.f16 ? launch_typed<_Float16>(a, st) : launch_typed<float>(a, st);
}

hipError_t launch_rotary_table(const double* frequencies, float* table, uint32_t positions, int rot,
                               float factor, hipStream_t st) {
  const uint64_t n = static_cast<uint64_t>(positions) * (rot / 2);
  rotary_table<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(
      frequencies, table, n, rot / 2, static_cast<double>(factor));
  return hipGetLastError();
}

}  // namespace tessery
