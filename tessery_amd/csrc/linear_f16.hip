// Projection of fp16 activations with its epilogue (route linear_f16), gfx950.
//
//   out = act(x W^T + bias) + residual       x [M, K], W [N, K], residual, out [M, N], bias [N]
// The products of fp16 values are exact in fp32 and are summed in fp32 on MFMA; bias, activation and
// residual are applied to the fp32 sum and one rounding to the output's type ends it.
//
// Bound by MFMA from a few hundred rows on: 8192^3 runs at 1130 TFLOP/s (a library product at 1355), 4096 x 1024 x
// 4096 takes 44 us (47.8), 16384 x 4096 x 1024 140 (122), or 168 to 174 with gelu, whose arithmetic no product
// hides. Bound by the read of W below: 24 x 4096 x 1024 takes 6 us, mostly one trip to HBM.
#include "common.h"
#include "kernels.h"
#include "lds_dma.h"

#include <math.h>

#include <type_traits>

namespace tessery {
namespace {

// 1 / (1 + 2^-x)
__device__ __forceinline__ float logistic(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x));
}

// y times the normal distribution's integral up to y, y (1 + erf(y / sqrt 2)) / 2, as max(y, 0) - t P(-t)
// with t = |y|. The integral up to -t is exp(-t^2 / 2) times a polynomial in u = 1 / (1 + p t) (the form of
// Abramowitz and Stegun 7.1.26; p and the coefficients are a weighted minimax fit to the function, off by
// less than 1e-8, 2e-7 with fp32 rounding). erff took 56 us of a 16384 x 4096 output, this 32 us.
__device__ __forceinline__ float gelu(float y) {
  const float t = fabsf(y), u = __builtin_amdgcn_rcpf(fmaf(0.28f, t, 1.0f));
  float s = -0.10580878214302342f;
  s = fmaf(s, u, 0.3898762044949095f);
  s = fmaf(s, u, -0.23699701042804464f);
  s = fmaf(s, u, 0.26891299545827674f);
  s = fmaf(s, u, 0.06749562607910956f);
  s = fmaf(s, u, 0.11652095725613074f);
  const float below = s * u * __builtin_amdgcn_exp2f(t * (t * -0.72134752044448170f));
  return fmaf(-fminf(t, 1e18f), below, fmaxf(y, 0.0f));  // an infinite t times 0 would be NaN
}

template <int ACT>
__device__ __forceinline__ float activate(float y) {
  if constexpr (ACT == kActRelu) return y < 0.0f ? 0.0f : y;
  if constexpr (ACT == kActGelu) return gelu(y);
  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (y + 0.044715 y^3)
  if constexpr (ACT == kActGeluTanh)
    return y * logistic(1.5957691216057308f * kLog2e * fmaf(0.044715f * y * y, y, y));
  if constexpr (ACT == kActSilu) return y * logistic(kLog2e * y);
  return y;
}

// Rows of K values begin at any even address where K is odd: 16-byte accesses that promise no more. The
// memory system takes them at any address; a copy straight into LDS (dma16_at) is given aligned ones.
typedef half8 half8_any __attribute__((aligned(2)));
typedef floatx4 floatx4_any __attribute__((aligned(4)));

// The eight values at p, of which the row has `left` (zeros behind them).
__device__ __forceinline__ half8 load8(const _Float16* p, int left) {
  if (left >= 8) return *reinterpret_cast<const half8_any*>(p);
  half8 v = {};
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < left) v[j] = p[j];
  return v;
}

// TM x TN outputs a workgroup of WM x WN wavefronts, K taken BK at a time through a ring of NST stages in
// LDS that global_load_lds_dwordx4 fills NST - 1 stages ahead. A row of a stage is BK halves; its 16-byte
// chunks are XORed with sw(row), so the 16 rows of a read fall on 16 bank groups. Rows past M or N read the
// last row and are not stored; the chunks of a last stage past K are left out as the operands are read.
// Where K is no multiple of 8 the stages pass through registers instead, one ahead (STAGED; NST = 2).
template <int BK>
__device__ __forceinline__ int sw(int row) {
  static_assert(BK == 64 || BK == 128, "rows of a half or a whole line of banks");
  return BK == 128 ? row & 15 : (row >> 1) & 7;
}

template <int TM, int TN, int WM, int WN, int BK, int NST>
struct TileShape {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int MB = TM / WM / 32, NB = TN / WN / 32;  // 32 x 32 blocks of a wavefront
  static constexpr int CPR = BK / 8;                          // chunks of a row
  static constexpr int STAGE = (TM + TN) * BK;                // halves
  static constexpr int LOADS = STAGE / 512 / WAVES;           // 1 KiB blocks a wavefront fills
  static constexpr int ROWS = 64 / CPR;                       // rows of a block
  static constexpr int OUT = TN / WN + 4;                     // floats of a row staged for the stores
  static constexpr int BYTES = NST * STAGE * 2 > WAVES * 32 * OUT * 4 ? NST * STAGE * 2 : WAVES * 32 * OUT * 4;
  static_assert(STAGE % (512 * WAVES) == 0 && TM * BK % 512 == 0, "whole blocks");
};

// Eight columns n .. n + 7 of row m from fp32 sums that bias and activation have been applied to.
__device__ __forceinline__ void store8(const LinearF16Args& a, int m, int n, const float* y) {
  const size_t at = static_cast<size_t>(m) * a.N + n;
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = y[j];
  if (n + 8 <= a.N) {
    if (a.residual) {
      const half8 v = *reinterpret_cast<const half8_any*>(a.residual + at);
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] += static_cast<float>(v[j]);
    }
    if (a.out_f32) {
      floatx4_any* const o = reinterpret_cast<floatx4_any*>(static_cast<float*>(a.out) + at);
      o[0] = floatx4{r[0], r[1], r[2], r[3]};
      o[1] = floatx4{r[4], r[5], r[6], r[7]};
    } else {
      half8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = static_cast<_Float16>(r[j]);
      *reinterpret_cast<half8_any*>(static_cast<_Float16*>(a.out) + at) = v;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (n + j >= a.N) return;
    if (a.residual) r[j] += static_cast<float>(a.residual[at + j]);
    if (a.out_f32) static_cast<float*>(a.out)[at + j] = r[j];
    else static_cast<_Float16*>(a.out)[at + j] = static_cast<_Float16>(r[j]);
  }
}

// How a workgroup's stages are filled and read: by copies into LDS, the same with its wavefronts in two
// groups that take turns, or through registers.
enum class Feed { kCopies, kTurns, kStaged };

// A product whose K is shared out: part p takes the k_each of K from p k_each and leaves its fp32 sums in
// sums + p M N, for linear_f16_sum. One part: all of K, no sums.
struct Split {
  int parts, k_each;
  float* sums;
};

// Workgroups go round the eight XCDs, each with an L2 of its own: an XCD takes a run of tiles, walked in
// bands of kBand tiles of M, so that the tiles that run on it together share rows of x and of W.
constexpr int kBand = 8;
struct TilePlace {
  int m, n, part;
  __device__ __forceinline__ TilePlace(int tiles_m, int tiles_n, const Split& split) {
    const int tiles = tiles_m * tiles_n;
    part = static_cast<int>(blockIdx.x) / tiles;
    const int id = static_cast<int>(blockIdx.x) - part * tiles;
    const int xcd = id & 7, each = tiles >> 3, over = tiles & 7;
    const int tile = xcd * each + min(xcd, over) + (id >> 3);
    const int band = tile / (kBand * tiles_n), in = tile - band * kBand * tiles_n;
    const int high = min(kBand, tiles_m - band * kBand);  // tiles of M in this band
    n = in / high;
    m = band * kBand + in - n * high;
  }
};

template <int TM, int TN, int WM, int WN, int BK, int NST, Feed FEED, int ACT>
__global__ __launch_bounds__(64 * WM * WN) void linear_f16_tiles(LinearF16Args a, int tiles_m, int tiles_n,
                                                                  Split split) {
  using S = TileShape<TM, TN, WM, WN, BK, NST>;
  constexpr int MB = S::MB, NB = S::NB;
  __shared__ __attribute__((aligned(1024))) char lds[S::BYTES];
  _Float16* const ring = reinterpret_cast<_Float16*>(lds);
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TilePlace place(tiles_m, tiles_n, split);
  const int m0 = place.m * TM, n0 = place.n * TN;
  const int row_k = a.K, k0 = place.part * split.k_each;  // values of a row, the first of this part
  if (split.parts > 1) {
    a.K = min(a.K - k0, split.k_each);  // from here on the part's
    a.bias = nullptr;
    a.residual = nullptr;
    a.out = split.sums + static_cast<size_t>(place.part) * a.M * a.N;
    a.out_f32 = 1;
  }
  const int wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);

  // Load i of a wavefront fills block i * WAVES + wave of a stage, rows of W (the first TN) or of x: the bytes
  // from the tile's first row to this lane's row and chunk of K.
  constexpr int WLOADS = TN / S::ROWS / S::WAVES;  // loads of W, before those of x
  static_assert(TN % (S::ROWS * S::WAVES) == 0, "a load takes rows of one operand");
  const char* const wbase = reinterpret_cast<const char*>(a.w + static_cast<size_t>(n0) * row_k + k0);
  const char* const xbase = reinterpret_cast<const char*>(a.x + static_cast<size_t>(m0) * row_k + k0);
  uint32_t off[S::LOADS];
#pragma unroll
  for (int i = 0; i < S::LOADS; ++i) {
    const int row = (i * S::WAVES + wave) * S::ROWS + lane / S::CPR - (i < WLOADS ? 0 : TN);
    const int chunk = (lane % S::CPR) ^ sw<BK>(row);
    off[i] = static_cast<uint32_t>(min(row, (i < WLOADS ? a.N - n0 : a.M - m0) - 1)) *
                 static_cast<uint32_t>(2 * row_k) + 16 * chunk;
  }
  const int steps = (a.K + BK - 1) / BK;
  auto issue = [&](int step) {
    _Float16* const to = ring + step % NST * S::STAGE + wave * 512;
    const int left = 2 * (a.K - step * BK);  // bytes of a row from here
    if (left >= 2 * BK) {
#pragma unroll
      for (int i = 0; i < S::LOADS; ++i)
        dma16_at((i < WLOADS ? wbase : xbase) + 2 * step * BK, off[i], to + i * S::WAVES * 512);
    } else {
#pragma unroll
      for (int i = 0; i < S::LOADS; ++i) {
        // chunks past K: the first of the tile (any; left out below)
        const int row = (i * S::WAVES + wave) * S::ROWS + lane / S::CPR;
        const int chunk = (lane % S::CPR) ^ sw<BK>(row);
        dma16_at(i < WLOADS ? wbase : xbase, 16 * chunk < left ? off[i] + 2 * step * BK : 0u,
                 to + i * S::WAVES * 512);
      }
    }
  };

  floatx16 acc[MB][NB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[mb][nb][e] = 0.0f;

  const int whole = a.K / BK;
  if constexpr (FEED == Feed::kTurns) {
    // Two groups of wavefronts, one of each on a SIMD, half a turn apart: while one reads its operands from
    // LDS the other has the matrix pipe. Between two barriers a group either reads (2 k-steps of 16) and
    // starts the copies of the stage after, or multiplies. Group 1 runs one barrier behind, so when group 0
    // starts on a stage, group 1 has just read the last of the stage before: the copies into that one may
    // start, and both have waited for their copies into this one.
    constexpr int TURNS = BK / 32;
    const int group = wave / (S::WAVES / 2);
    // this wavefront's copies into the stage after `step` have landed
    auto next_ready = [&](int step) {
      if (step + NST - 1 < steps) wait_vmcnt<(NST - 2) * S::LOADS>();
      else wait_vmcnt<0>();
    };
    auto turn = [&](int step, int c, auto tail) {
      constexpr bool TAIL = decltype(tail)::value;
      const _Float16* const ws = ring + step % NST * S::STAGE + (wn + r) * BK;
      const _Float16* const xs = ring + step % NST * S::STAGE + (TN + wm + r) * BK;
      half8 wf[2][NB], xf[2][MB];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = 2 * c + i, at = 8 * ((2 * k + h) ^ sw<BK>(r));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) wf[i][nb] = *reinterpret_cast<const half8*>(ws + 32 * nb * BK + at);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) xf[i][mb] = *reinterpret_cast<const half8*>(xs + 32 * mb * BK + at);
        if (TAIL && step * BK + 16 * k + 8 * h >= a.K) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) wf[i][nb] = half8{};
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) xf[i][mb] = half8{};
        }
      }
      if (c == 0 && step > 0 && step + NST - 1 < steps) issue(step + NST - 1);
      wait_lgkmcnt<0>();
      if (c == TURNS - 1 && group == 1) next_ready(step);
      __builtin_amdgcn_sched_barrier(0);
      stage_barrier();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            acc[mb][nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[i][nb], xf[i][mb], acc[mb][nb], 0, 0, 0);
      __builtin_amdgcn_s_setprio(0);
      if (c == TURNS - 1 && group == 0) next_ready(step);
      __builtin_amdgcn_sched_barrier(0);
      stage_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < NST; ++i)
      if (i < steps) issue(i);
    if (steps >= NST) wait_vmcnt<(NST - 1) * S::LOADS>();
    else wait_vmcnt<0>();
    stage_barrier();
    if (group == 1) stage_barrier();
    for (int step = 0; step < whole; ++step) {
#pragma unroll
      for (int c = 0; c < TURNS; ++c) turn(step, c, std::false_type{});
    }
    if (whole < steps) {
#pragma unroll
      for (int c = 0; c < TURNS; ++c) turn(whole, c, std::true_type{});
    }
    if (group == 0) stage_barrier();
  } else {
    // the products of one stage; TAIL: the last one, with less than BK of K left
    auto multiply = [&](int step, auto tail) {
      constexpr bool TAIL = decltype(tail)::value;
      const _Float16* const ws = ring + step % NST * S::STAGE + (wn + r) * BK;
      const _Float16* const xs = ring + step % NST * S::STAGE + (TN + wm + r) * BK;
      half8 wf[2][NB], xf[2][MB];
      auto read = [&](int s) {
        const int at = 8 * ((2 * s + h) ^ sw<BK>(r));  // rows 32 apart share it
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) wf[s & 1][nb] = *reinterpret_cast<const half8*>(ws + 32 * nb * BK + at);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) xf[s & 1][mb] = *reinterpret_cast<const half8*>(xs + 32 * mb * BK + at);
        if (TAIL && step * BK + 16 * s + 8 * h >= a.K) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) wf[s & 1][nb] = half8{};
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) xf[s & 1][mb] = half8{};
        }
      };
      read(0);
#pragma unroll
      for (int s = 0; s < BK / 16; ++s) {
        if (s + 1 < BK / 16) read(s + 1);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            acc[mb][nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[s & 1][nb], xf[s & 1][mb], acc[mb][nb], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
      }
    };
    if constexpr (FEED == Feed::kCopies) {
      auto take = [&](int step, auto tail) {
        if (step + NST - 2 < steps) wait_vmcnt<(NST - 2) * S::LOADS>();
        else wait_vmcnt<0>();
        wait_lgkmcnt<0>();  // this wavefront's reads of the stage that is filled next
        stage_barrier();
        if (step + NST - 1 < steps) issue(step + NST - 1);
        multiply(step, tail);
      };
#pragma unroll
      for (int i = 0; i < NST - 1; ++i)
        if (i < steps) issue(i);
      for (int step = 0; step < whole; ++step) take(step, std::false_type{});
      if (whole < steps) take(whole, std::true_type{});
    } else {
      static_assert(NST == 2, "one stage ahead");
      half8 held[S::LOADS];
      auto fetch = [&](int step) {
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) {
          const int row = (i * S::WAVES + wave) * S::ROWS + lane / S::CPR;
          const int at = step * BK + 8 * ((lane % S::CPR) ^ sw<BK>(row));
          held[i] = load8(reinterpret_cast<const _Float16*>((i < WLOADS ? wbase : xbase) + off[i]) + step * BK,
                          a.K - at);
        }
      };
      auto store = [&](int step) {
        _Float16* const to = ring + step % NST * S::STAGE + wave * 512 + lane * 8;
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) *reinterpret_cast<half8*>(to + i * S::WAVES * 512) = held[i];
      };
      fetch(0);
      store(0);
      for (int step = 0; step < steps; ++step) {
        __syncthreads();
        if (step + 1 < steps) fetch(step + 1);
        multiply(step, std::false_type{});  // what lies past K is zeros
        if (step + 1 < steps) store(step + 1);
      }
    }
  }
  wait_lgkmcnt<0>();
  stage_barrier();  // the ring is read out: it takes the rows to be stored, 32 a wavefront at a time

  // LDS serves a wavefront's accesses in order: its own rows need no barrier
  float* const box = reinterpret_cast<float*>(lds) + wave * 32 * S::OUT;
  constexpr int PER = TN / WN / 8;  // lanes of a row, eight columns each
  const int c = lane % PER * 8, n = n0 + wn + c;
  float bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = a.bias && n + j < a.N ? a.bias[n + j] : 0.0f;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<floatx4*>(box + r * S::OUT + 32 * nb + 8 * q + 4 * h) =
            floatx4{acc[mb][nb][4 * q], acc[mb][nb][4 * q + 1], acc[mb][nb][4 * q + 2],
                    acc[mb][nb][4 * q + 3]};
#pragma unroll 1
    for (int row = lane / PER; row < 32; row += 64 / PER) {
      const floatx4 lo = *reinterpret_cast<const floatx4*>(box + row * S::OUT + c);
      const floatx4 hi = *reinterpret_cast<const floatx4*>(box + row * S::OUT + c + 4);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = activate<ACT>((j < 4 ? lo[j & 3] : hi[j & 3]) + bias[j]);
      const int m = m0 + wm + 32 * mb + row;
      if (m < a.M && n < a.N) store8(a, m, n, y);
    }
  }
}

// f(ACT) as a compile-time value
template <typename F>
void for_activation(int act, F&& f) {
  switch (act) {
    case kActRelu: return f(std::integral_constant<int, kActRelu>{});
    case kActGelu: return f(std::integral_constant<int, kActGelu>{});
    case kActGeluTanh: return f(std::integral_constant<int, kActGeluTanh>{});
    case kActSilu: return f(std::integral_constant<int, kActSilu>{});
    default: return f(std::integral_constant<int, kActNone>{});
  }
}

// out = act(sums of all parts + bias) + residual, eight outputs a thread, the parts in order.
template <int ACT>
__global__ __launch_bounds__(256) void linear_f16_sum(LinearF16Args a, Split split) {
  const size_t n = static_cast<size_t>(a.M) * a.N, at = (blockIdx.x * size_t{256} + threadIdx.x) * 8;
  if (at >= n) return;
  float y[8] = {};
  const bool whole = at + 8 <= n;
  for (int p = 0; p < split.parts; ++p) {
    const float* const from = split.sums + p * n + at;
    if (whole) {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const floatx4 v = *reinterpret_cast<const floatx4_any*>(from + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[j + i] += v[i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j < n) y[j] += from[j];
    }
  }
  int c = static_cast<int>(at % a.N);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (a.bias) y[j] += a.bias[c];
    y[j] = activate<ACT>(y[j]);
    c = c + 1 == a.N ? 0 : c + 1;
  }
  a.N = static_cast<int>(n < 0x7fffffff ? n : 0x7fffffff);  // one row of all outputs
  store8(a, 0, static_cast<int>(at), y);
}

template <int TM, int TN, int WM, int WN, int BK, int NST, Feed FEED>
hipError_t launch_tiles(const LinearF16Args& a, hipStream_t st, Split split = {1, 0, nullptr}) {
  const int tm = (a.M + TM - 1) / TM, tn = (a.N + TN - 1) / TN;
  const unsigned grid = static_cast<unsigned>(tm) * static_cast<unsigned>(tn) * static_cast<unsigned>(split.parts);
  if (split.parts > 1) {
    linear_f16_tiles<TM, TN, WM, WN, BK, NST, FEED, kActNone><<<grid, 64 * WM * WN, 0, st>>>(a, tm, tn, split);
    const size_t pieces = (static_cast<size_t>(a.M) * a.N + 7) / 8;
    for_activation(a.act, [&](auto act) {
      linear_f16_sum<decltype(act)::value>
          <<<static_cast<unsigned>((pieces + 255) / 256), 256, 0, st>>>(a, split);
    });
    return hipGetLastError();
  }
  for_activation(a.act, [&](auto act) {
    linear_f16_tiles<TM, TN, WM, WN, BK, NST, FEED, decltype(act)::value>
        <<<grid, 64 * WM * WN, 0, st>>>(a, tm, tn, split);
  });
  return hipGetLastError();
}

// Up to 32 rows of x: the weights are what is read, once, straight into registers. A workgroup
// has 32 columns of out; its wavefronts take every WAVES-th 64 of K each, and their sums meet in LDS and
// are added in that order.
template <int WAVES, int ACT>
__global__ __launch_bounds__(64 * WAVES) void linear_f16_rows(LinearF16Args a) {
  constexpr int ROW = 36;  // floats of a staged row of 32 columns
  __shared__ __attribute__((aligned(16))) float box[WAVES][32 * ROW];
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.x * 32;
  const _Float16* const w = a.w + static_cast<size_t>(min(n0 + r, a.N - 1)) * a.K + 8 * h;
  const _Float16* const x = a.x + static_cast<size_t>(min(r, a.M - 1)) * a.K + 8 * h;
  floatx16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
#pragma unroll 2
  for (int k = 64 * wave; k < a.K; k += 64 * WAVES) {
    half8 wf[4], xf[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int left = a.K - (k + 16 * s + 8 * h);
      wf[s] = load8(w + k + 16 * s, left);
      xf[s] = load8(x + k + 16 * s, left);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[s], xf[s], acc, 0, 0, 0);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<floatx4*>(&box[wave][r * ROW + 8 * q + 4 * h]) =
        floatx4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * 32; i += 64 * WAVES) {
    const int m = i >> 5, n = n0 + (i & 31);
    if (m >= a.M || n >= a.N) continue;
    float y = box[0][m * ROW + (i & 31)];
#pragma unroll
    for (int g = 1; g < WAVES; ++g) y += box[g][m * ROW + (i & 31)];
    y = activate<ACT>(y + (a.bias ? a.bias[n] : 0.0f));
    const size_t at = static_cast<size_t>(m) * a.N + n;
    if (a.residual) y += static_cast<float>(a.residual[at]);
    if (a.out_f32) static_cast<float*>(a.out)[at] = y;
    else static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(y);
  }
}

template <int WAVES>
hipError_t launch_rows(const LinearF16Args& a, hipStream_t st) {
  for_activation(a.act, [&](auto act) {
    linear_f16_rows<WAVES, decltype(act)::value>
        <<<static_cast<unsigned>((a.N + 31) / 32), 64 * WAVES, 0, st>>>(a);
  });
  return hipGetLastError();
}

// The kernels and how long they take, in us, by the tiles that one round of the chip holds and the K of a
// round, measured over M 8 .. 16384, N and K 384 .. 4096 (the fit holds within a tenth from one round on):
//   rows    32 x 32, M <= 32        24 x 4096 x 1024 5.9 against 6.8 on 64 x 64; 64 rows 9.0 against 6.8
//   64      512 a round             3.7 + 6.2 K / 1024    2048 x 1024 x 1024 10.0 (128: 12.4, 256: 26.9)
//     its K in parts                + 4.5, and 3 us a MB of sums   363 x 68 x 6479 20.3 between events (60.1)
//   128     256 a round             4.3 + 9.4 K / 1024    4096 x 1024 x 4096 42.1 (64: 55.6, 256: 87.3)
//   128 x 2 512 a round, 2 a CU     5.2 + 15.5 K / 1024   2048 x 4096 x 1024 22.9 (128: 26.2, 256: 31.6)
//   256     256 a round             7.0 + 28.5 K / 1024   16384 x 4096 x 1024 139.9 (128 x 2: 156.5)
// Where K is no multiple of 8: 64 and 128, through registers.
enum class Kind { kRows, k64, k128, k128x2, k256 };
struct Choice {
  Kind kind;
  int parts;
};

float rounds(int64_t m, int64_t n, int64_t tile, int64_t parts, int64_t slots) {
  return static_cast<float>(((m + tile - 1) / tile * ((n + tile - 1) / tile) * parts + slots - 1) / slots);
}

Choice choose(int M, int N, int K, size_t scratch_floats) {
  if (M <= 32) return {Kind::kRows, 1};
  const float k = static_cast<float>(K) / 1024.0f;
  Choice best = {Kind::k64, 1};
  float least = rounds(M, N, 64, 1, 512) * (3.7f + 6.2f * k);
  auto offer = [&](Kind kind, int parts, float us) {
    if (us < least) {
      least = us;
      best = {kind, parts};
    }
  };
  offer(Kind::k128, 1, rounds(M, N, 128, 1, 256) * (4.3f + 9.4f * k));
  if (K % 8 == 0) {
    offer(Kind::k128x2, 1, rounds(M, N, 128, 1, 512) * (5.2f + 15.5f * k));
    offer(Kind::k256, 1, rounds(M, N, 256, 1, 256) * (7.0f + 28.5f * k));
  }
  const size_t sums = static_cast<size_t>(M) * N;
  for (int parts = 2; parts <= 32 && parts * sums <= scratch_floats && parts * 128 <= K; ++parts)
    offer(Kind::k64, parts, rounds(M, N, 64, parts, 512) * (3.7f + 6.2f * k / parts) + 4.5f +
                                3.0f * static_cast<float>(parts * sums) * 4e-6f);
  return best;
}

}  // namespace

bool linear_f16_in_parts(int M, int N, int K, size_t scratch_floats) {
  return choose(M, N, K, scratch_floats).parts > 1;
}

hipError_t launch_linear_f16(const LinearF16Args& a, hipStream_t st) {
  const Choice c = choose(a.M, a.N, a.K, a.scratch ? a.scratch_floats : 0);
  const bool staged = a.K % 8 != 0;
  Split split = {c.parts, 0, a.scratch};
  split.k_each = ((a.K + c.parts - 1) / c.parts + 127) / 128 * 128;
  split.parts = (a.K + split.k_each - 1) / split.k_each;
  switch (c.kind) {
    case Kind::kRows:
      return launch_rows<8>(a, st);
    case Kind::k64:
      return staged ? launch_tiles<64, 64, 2, 2, 128, 2, Feed::kStaged>(a, st, split)
                    : launch_tiles<64, 64, 2, 2, 128, 2, Feed::kCopies>(a, st, split);
    case Kind::k128:
      return staged ? launch_tiles<128, 128, 2, 4, 64, 2, Feed::kStaged>(a, st)
                    : launch_tiles<128, 128, 2, 4, 128, 2, Feed::kCopies>(a, st);
    case Kind::k128x2:
      return launch_tiles<128, 128, 2, 2, 64, 2, Feed::kCopies>(a, st);
    default:
      return launch_tiles<256, 256, 2, 4, 64, 2, Feed::kTurns>(a, st);
  }
}

}  // namespace tessery
