// Attention with score functions and masks for gfx950 (route attention_masked).
//
//   s_ij = scale q_i . k_j ;  s_ij = cap tanh(s_ij / cap) with a cap
//   s_ij -= slope_h |i - j|, or += table_h[clamp(j - i, -radius, radius) + radius]
//   out_i = sum_j softmax_j(s_ij) v_j over the keys lo_i <= j < hi_i; zeros where there is none
// Every mask here is a range of keys: hi_i is the row's length, i + 1 (causal) or max(i + 1, prefix_b),
// i + window and the end of the token's span, whichever is least; lo_i the most of 0, i - window + 1 and
// the span's start. kv head = h / (H / KV).
//
// A workgroup of four wavefronts keeps the queries and their outputs in registers and walks tiles of keys that LDS
// copies bring (Tile), with one pass of a softmax in fp32 (Softmax). Two products of 2 D operations a pair go to
// MFMA, one exponential a pair (with a cap three transcendentals, at a quarter of the rate) to the vector units,
// which bound it beside them: uniform rows of 8192, 16 fp16 heads of 128, run at about 800 TFLOP/s, of 2048, 48
// heads of 64, at 670, in fp32 32 heads of 64 at 104 (a product of 8192^3 reaches 1355 and 153). 2 x 4096 with a cap
// and a window of 1024 takes 116 us, of which the cap's two transcendentals are about a third; a row of 8192 in documents,
// 12 heads of 64, 80, two rounds of workgroups of unlike length; 8 x 512 with slopes in fp32 58; 24 tokens 6.
#include "common.h"
#include "kernels.h"
#include "lds_dma.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

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

// Batch rows of a few tokens: a wavefront for each token and head, instead of a tile that is mostly masked.
template <typename T>
__global__ __launch_bounds__(256) void attn_masked_rows(MaskedArgs a) {
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<uint32_t>(a.B) * a.S * a.H) return;  // wavefront-uniform
  const uint32_t token = row / a.H;
  masked_row<T>(a, static_cast<int>(token / a.S), static_cast<int>(token % a.S), static_cast<int>(row % a.H),
                threadIdx.x & 63);
}

// 8 bytes of a row-major fp16 V tile a lane, transposed across each group of 16 lanes: lane r of a group
// names row r / 4, channels 4 (r % 4) .. + 3 and receives channel r of the four rows.
typedef __fp16 fp16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ half4 read_transposed(const _Float16* p) {
  const fp16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
      (__attribute__((address_space(3))) fp16x4_t*)(p));
  return __builtin_bit_cast(half4, v);
}

// The hardware does not hold back a VALU read of an MFMA result and the compiler pads such reads only
// inside a basic block: 20 wait states (a 32x32x16 product needs 19) before a branch may follow.
__device__ __forceinline__ void product_done(floatx16& acc) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(acc));
}

__device__ __forceinline__ float other_half(float x, bool take_max) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float a = __uint_as_float(p[0]), b = __uint_as_float(p[1]);
  return take_max ? fmaxf(a, b) : a + b;
}

// Least and most over the 32 lanes of each half (both halves hold the same queries), by lane exchanges
// in quads, in mirrored halves of 8 and 16 lanes, and between rows of 16.
template <int CTRL>
__device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_mov_dpp(x, CTRL, 0xf, 0xf, true);
}
template <bool MOST>
__device__ __forceinline__ int of_two(int a, int b) {
  return MOST ? max(a, b) : min(a, b);
}
template <bool MOST>
__device__ __forceinline__ int half_wave(int x) {
  x = of_two<MOST>(x, dpp<0xB1>(x));   // quad_perm [1, 0, 3, 2]
  x = of_two<MOST>(x, dpp<0x4E>(x));   // quad_perm [2, 3, 0, 1]
  x = of_two<MOST>(x, dpp<0x141>(x));  // row_half_mirror
  x = of_two<MOST>(x, dpp<0x140>(x));  // row_mirror
  const auto p = __builtin_amdgcn_permlane16_swap(static_cast<unsigned>(x), static_cast<unsigned>(x), false, false);
  return __builtin_amdgcn_readfirstlane(of_two<MOST>(static_cast<int>(p[0]), static_cast<int>(p[1])));
}

// Keys that some row of a wavefront attends (lo, hi) and keys that all its rows attend (all_lo, all_hi).
struct WaveKeys {
  int lo, hi, all_lo, all_hi;
};

__device__ __forceinline__ WaveKeys wave_keys(KeyRange r, bool row) {
  const bool some = row && r.lo < r.hi;
  WaveKeys w;
  w.lo = half_wave<false>(some ? r.lo : 0x7fffffff);
  w.hi = half_wave<true>(some ? r.hi : 0);
  w.all_lo = half_wave<true>(!row ? 0 : some ? r.lo : 0x7fffffff);
  w.all_hi = half_wave<false>(!row ? 0x7fffffff : some ? r.hi : 0);
  return w;
}

// The running maximum of a row moves when a tile exceeds it by more than kSlack (log2 units), and
// probabilities carry 2^kLift: at most 2^14 in fp16, and full fp16 precision down to 2^-20 of the
// largest. The softmax does not depend on either.
constexpr float kSlack = 8.0f, kLift = 6.0f;

// Up to this cap fp16 scores may be off by 2^-22 of it: at most 2^-14, and a probability by an eighth of its
// rounding to fp16.
constexpr float kCoarseCap = 256.0f;

// Blocks of queries of a batch row, up to which those of long documents come first. It takes about 1 us, and so is
// left out where all workgroups run at once: 1 x 8192 in documents, 12 heads of 64 (1536 workgroups), 90 -> 78 us, fp32
// 8 x 2002, 12 heads of 40, 462 -> 393; 4 x 246, 36 heads of 128, 64 -> 67.
constexpr int kRanked = 256;

// Rows of up to so many tokens go to attn_masked_rows, of twice as many where a tile's work is largest (256
// channels, fp32 above 64). 512 x S, 16 heads on 8, as rows and in tiles, us: 128 fp16, S = 1 8.2 and 58.9, S = 4 29.6
// and 59.5, S = 8 116 and 60; 256 fp32, S = 1 9.4 and 479, S = 8 179 and 484, S = 16 820 and 504; one of them: 128 fp16,
// S = 4 8.0 and 7.9; 256 fp32, S = 8 13.7 and 18.5.
constexpr int kFewTokens = 4;

// What the kernels on tiles take beside the arguments: signs and factors of the scores in log2 units.
struct ScoreArgs {
  float q_sign;  // -1 for a negative scale, 0 for none
  float scale2;  // |scale| log2 e; with a cap the factor in front of tanh's exponent, 2 |scale| log2 e / cap
  float cap2;    // cap log2 e
};

// tanh of half of x ln 2, to about 4 units of 2^-24 relative: t / (t + 2) of t = 2^x - 1 = 2^n (2^f - 1) + 2^n - 1 with
// n the integer next to x, where 2^f - 1 is a polynomial (minimax of the relative error on [-1/2, 1/2], 2^-25).
// NaN for NaN and infinities, whose rows are then made by masked_row.
__device__ __forceinline__ float tanh_of_log2(float x) {
  const float n = rintf(x), f = x - n;
  float p = 0x1.39f2eap-13f;
  p = fmaf(p, f, 0x1.5e8ac4p-10f);
  p = fmaf(p, f, 0x1.3b34a0p-7f);
  p = fmaf(p, f, 0x1.c6b084p-5f);
  p = fmaf(p, f, 0x1.ebfbe0p-3f);
  p = fmaf(p, f, 0x1.62e430p-1f) * f;
  // from 2^64 on t / (t + 2) is 1, and -1 from 2^-64 - 1
  const float two = __builtin_amdgcn_ldexpf(1.0f, static_cast<int>(__builtin_amdgcn_fmed3f(n, -64.0f, 64.0f)));
  const float t = fmaf(two, p, two - 1.0f);
  return t * __builtin_amdgcn_rcpf(t + 2.0f);
}

// What is done to the products before the softmax: nothing (they are scaled as exponents are taken), the cap
// alone, or a cap or none and then a bias, told apart as the kernel runs. (With the cap alone told apart there
// too, 2 x 4096 with 16 heads of 128, a cap and a window took 143 us instead of 119.)
// fp16 takes kCapped and kAny where the tanh may be coarse, else kAnyFine (within kAny it cost a third wavefront a
// SIMD at 96 channels: 8 x 1024, 16 heads, with slopes 93 -> 102 us).
enum class Scores { kPlain, kCapped, kAny, kAnyFine };
constexpr bool any(Scores how) { return how == Scores::kAny || how == Scores::kAnyFine; }

// Scores of one 32-key block, from products to log2 units, still to be masked: element e of lane (query, h)
// is the key 8 (e / 4) + 4 h + e % 4 of the block. rel: the key of element 0 less the query's position.
template <bool F16, Scores HOW>
__device__ __forceinline__ void score_block(floatx16& v, const MaskedArgs& a, const ScoreArgs& s,
                                            float slope2, float rel, const float* biases) {
  // tanh(u) = 1 - 2 / (exp(2 u) + 1): exact at both ends, off by at most 2^-23 around 0. Under fp16 probabilities
  // (2^-11) that is nothing for caps up to kCoarseCap; fp32 takes the tanh that is exact there too.
  auto turned = [&](float x) {
    return -__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * s.scale2) + 1.0f);
  };
  if constexpr (HOW == Scores::kCapped) {
    // without the 1, which no softmax sees, and the factor 2 cap (fp32: cap), which the exponents take
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = F16 ? turned(v[e]) : tanh_of_log2(v[e] * s.scale2);
    return;
  }
  if (a.cap > 0.0f) {
    if constexpr (F16 && HOW == Scores::kAny) {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = fmaf(2.0f * s.cap2, turned(v[e]), s.cap2);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = s.cap2 * tanh_of_log2(v[e] * s.scale2);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] *= s.scale2;
  }
  if (a.bias_kind == kBiasSlopes) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      v[e] = fmaf(-slope2, fabsf(rel + static_cast<float>(8 * (e >> 2) + (e & 3))), v[e]);
  }
  if (a.bias_kind == kBiasTable) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] += biases[8 * (e >> 2) + (e & 3)];
  }
}

// The batch row of a rank by falling length (equal ones in order); of up to 64 rows.
__device__ __forceinline__ int row_of_rank(const MaskedArgs& a, int rank) {
  if (a.B == 1 || a.B > 64) return rank;
  const int lane = threadIdx.x & 63;
  const uint32_t mine = lane < a.B ? min(a.lengths[lane], static_cast<uint32_t>(a.S)) : 0;
  int before = 0;
  for (int n = 0; n < a.B; ++n) {
    const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), n));
    before += other > mine || (other == mine && n < lane);
  }
  return __ffsll(__ballot(lane < a.B && before == rank)) - 1;
}

// The block of QB queries of batch row b that comes `place`-th by the span of keys from its first token's to its
// last one's (powers of two from 128 keys on; equal ones from the last).
template <int QB>
__device__ __forceinline__ int block_by_span(const MaskedArgs& a, int b, int blocks, int place) {
  const int lane = threadIdx.x & 63;
  const uint32_t* const spans = a.spans + 2 * static_cast<size_t>(b) * a.S;
  int size[kRanked / 64];
#pragma unroll
  for (int m = 0; m < kRanked / 64; ++m) {
    const int n = lane + 64 * m;
    size[m] = -1;
    if (n < blocks) {
      const uint32_t lo = min(spans[2 * n * QB], static_cast<uint32_t>(a.S));
      const uint32_t hi = min(spans[2 * min(n * QB + QB - 1, a.S - 1) + 1], static_cast<uint32_t>(a.S));
      const uint32_t keys = hi > lo ? hi - lo : 0;
      size[m] = keys < 128 ? 0 : min(24 - __clz(static_cast<int>(keys)) + 1, 7);
    }
  }
  for (int k = 7; k >= 0; --k)
#pragma unroll
    for (int m = kRanked / 64 - 1; m >= 0; --m) {
      const unsigned long long mask = __ballot(size[m] == k);
      const int count = __popcll(mask);
      if (place < count) {
        const int above = count - 1 - static_cast<int>(__popcll(mask & ((1ull << lane) - 1)));
        return __ffsll(__ballot(size[m] == k && above == place)) - 1 + 64 * m;
      }
      place -= count;
    }
  return 0;
}

// Where a workgroup of four wavefronts works: 4 / KS wavefronts of 32 queries of one head each, in KS
// groups that share the keys out. Lane l holds query r = l % 32, as its half h = l / 32.
template <int KS>
struct Place {
  static constexpr int QW = 4 / KS, QB = 32 * QW;
  int lane, r, h, wave, qw, group, head, kvh, b, i0, i, L;
  size_t token;
  bool row;        // i is a query
  KeyRange mine;   // the keys of query i
  WaveKeys keys;

  __device__ __forceinline__ explicit Place(const MaskedArgs& a) {
    lane = threadIdx.x & 63;
    r = lane & 31;
    h = lane >> 5;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    qw = wave % QW;
    group = wave / QW;
    // Long work first: batch rows by falling length, blocks of queries from the last (under a causal mask the
    // longest, and outermost there), or by the documents they meet. Within that, key heads change fastest, so that neighbours, which start
    // on different compute units, are alike, and where they are a multiple of eight the query heads of one
    // meet on one XCD.
    const int blocks = (a.S + QB - 1) / QB, share = a.H / a.KV;
    int at = static_cast<int>(blockIdx.x);
    kvh = at % a.KV;
    at /= a.KV;
    head = kvh * share + at % share;
    at /= share;
    int block, rank;
    if (a.mask == kMaskBidirectional) {
      block = at % blocks;
      rank = at / blocks;
    } else {
      rank = at % a.B;
      block = at / a.B;
    }
    b = row_of_rank(a, rank);
    const bool ranked = a.spans && blocks >= 16 && blocks <= kRanked && gridDim.x >= 768;
    const int qb = ranked ? __builtin_amdgcn_readfirstlane(block_by_span<QB>(a, b, blocks, block))
                          : blocks - 1 - block;
    i0 = qb * QB;
    i = i0 + qw * 32 + r;
    row = i < a.S;
    token = static_cast<size_t>(b) * a.S;
  }

  // The keys of this lane's query and of the wavefront. (Loads, like the lengths that the order of rows
  // takes: after those of Q, whose way is as long.)
  __device__ __forceinline__ void look(const MaskedArgs& a) {
    mine = key_range(a, b, min(i, a.S - 1));
    keys = wave_keys(mine, row);
    L = static_cast<int>(min(a.lengths[b], static_cast<uint32_t>(a.S)));
  }

  // the tiles of `size` keys that the workgroup walks, from the wavefronts' `ends`; none where nothing is
  // attended
  __device__ __forceinline__ void tiles(const int (*ends)[2], int size, int* first, int* last) const {
    __syncthreads();
    int lo = ends[0][0], hi = ends[0][1];
#pragma unroll
    for (int n = 1; n < QW; ++n) {
      lo = min(lo, ends[n][0]);
      hi = max(hi, ends[n][1]);
    }
    *first = lo / size;
    *last = (hi + size - 1) / size;
  }

  // whether no row of this wavefront attends a key of j0 .. j0 + n - 1, and whether some row does not attend
  // them all
  __device__ __forceinline__ bool skips(int j0, int n) const { return j0 >= keys.hi || j0 + n <= keys.lo; }
  __device__ __forceinline__ bool partial(int j0, int n) const {
    return j0 < keys.all_lo || j0 + n > keys.all_hi;
  }
  __device__ __forceinline__ void mask(floatx16& s, int j0) const {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int j = j0 + 8 * (e >> 2) + 4 * h + (e & 3);
      if (j < mine.lo || j >= mine.hi) s[e] = -INFINITY;
    }
  }
};

// The online softmax of one query: the running maximum (in log2 units), what exponents are taken less
// of, and this lane's share of the sum.
template <int NDT>
struct Softmax {
  float top = -INFINITY, base = 0.0f, sum = 0.0f;
  floatx16 o[NDT];

  __device__ __forceinline__ Softmax() {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
  }

  // takes in the blocks' largest score, `factor` times that of s
  template <int N>
  __device__ __forceinline__ void raise(const floatx16 (&s)[N], float factor, float lift) {
    float most = s[0][0];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) most = fmaxf(most, s[n][e]);
    most = other_half(most, true) * factor;
    const bool grow = most > top + kSlack;
    if (__any(grow)) {
      const float old = grow ? __builtin_amdgcn_exp2f(top - most) : 1.0f;
      top = grow ? most : top;
      base = grow ? most - lift : base;
      sum *= old;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] *= old;
    }
  }

  // After the last tile: the lanes' shares of the sum meet, then the groups' results: groups
  // 1 .. KS - 1 hand theirs over in `box` and group 0 adds them in that order. False: not group 0.
  static constexpr int BOX = NDT * 16 + 2;
  template <int KS>
  __device__ __forceinline__ bool join(const Place<KS>& w, float* box) {
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) product_done(o[dt]);
    sum = other_half(sum, false);
    if constexpr (KS > 1) {
      if (w.group > 0) {
        float* const to = box + ((w.group - 1) * w.QW + w.qw) * BOX * 64 + w.lane;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) to[(16 * dt + e) * 64] = o[dt][e];
        to[(BOX - 2) * 64] = top;
        to[(BOX - 1) * 64] = sum;
      }
      __syncthreads();
      if (w.group > 0) return false;
#pragma unroll
      for (int g = 1; g < KS; ++g) {
        const float* const from = box + ((g - 1) * w.QW + w.qw) * BOX * 64 + w.lane;
        const float top1 = from[(BOX - 2) * 64], both = fmaxf(top, top1);
        const float c0 = top == both ? 1.0f : __builtin_amdgcn_exp2f(top - both);
        const float c1 = top1 == both ? 1.0f : __builtin_amdgcn_exp2f(top1 - both);
        sum = sum * c0 + from[(BOX - 1) * 64] * c1;
        top = both;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * c0 + from[(16 * dt + e) * 64] * c1;
        }
      }
    }
    return true;
  }

  // Stores the wavefront's rows. A product of a probability of zero with a value that is not finite
  // leaves NaN in a row that does not attend that value: rows that are not finite are computed again,
  // each on its own.
  template <typename T, int KS>
  __device__ __forceinline__ void store(const MaskedArgs& a, const Place<KS>& w) const {
    typedef T out4 __attribute__((ext_vector_type(4)));
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float odd = sum * 0.0f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) odd += o[dt][e] * 0.0f;
    const unsigned long long found = __ballot(w.row && !(odd == 0.0f));
    uint32_t again = static_cast<uint32_t>(found) | static_cast<uint32_t>(found >> 32);
    if (w.row && !((again >> w.r) & 1)) {
      T* const out = static_cast<T*>(a.out) + ((w.token + w.i) * a.H + w.head) * a.D;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int ch = 32 * dt + 8 * c + 4 * w.h;
          if (ch < a.D)
            *reinterpret_cast<out4*>(out + ch) =
                out4{static_cast<T>(o[dt][4 * c] * inv), static_cast<T>(o[dt][4 * c + 1] * inv),
                     static_cast<T>(o[dt][4 * c + 2] * inv), static_cast<T>(o[dt][4 * c + 3] * inv)};
        }
    }
    while (again) {
      const int n = __ffs(again) - 1;
      again &= again - 1;
      masked_row<T>(a, w.b, w.i0 + w.qw * 32 + n, w.head, w.lane);
    }
  }
};

// The tiles of one kernel: KT keys of K and V pass through a ring of NST stages in LDS, which
// global_load_lds_dwordx4 fills in blocks of 1 KiB, NST - 1 tiles ahead; one barrier a tile (two of a ring of
// one: fp32 tiles so wide that LDS holds one, whose products take far longer than the copy). Rows lie as in
// memory, DP channels long (the head size up to 32, 64, 96, 128 or 256), their 16-byte chunks permuted so that
// what an instruction reads falls on different banks: place_k and place_v. Keys past the length repeat the
// last one and are masked; chunks past the head size repeat its last one, against zeros of Q or into channels
// that are not stored. (What of that is not finite is put right with the rows that are not: Softmax::store.)
template <bool F16, int DP, int KS>
struct Tile {
  typedef typename std::conditional<F16, _Float16, float>::type T;
  static constexpr int SIZE = F16 ? 2 : 4;
  static constexpr int NB = F16 && (KS == 1 ? DP <= 96 : KS == 2 && DP <= 64) ? 2 : 1;  // blocks of 32 keys a group takes of a tile
  static constexpr int KT = 32 * KS * NB;
  static constexpr int CPR = DP * SIZE / 16;           // chunks of a row
  static constexpr int BYTES = KT * DP * SIZE;         // of K, and of V
  static constexpr int BLOCKS = BYTES / 1024;
  static constexpr int LOADS = BLOCKS / 2;             // copies a wavefront makes for a tile
  static constexpr int NST = BYTES > 32768 ? 1 : !F16 ? 2 : BYTES <= 4096 ? 4 : BYTES <= 8192 ? 3 : 2;
  static constexpr int BIASES = KT + 128;              // distances of one tile, KT + QB - 1
  static constexpr int RING = NST * 2 * BYTES;
  static_assert(BLOCKS % 4 == 0, "a copy takes rows of one operand");

  // chunk c of key row r lies at this chunk of its row
  __device__ static __forceinline__ int place_k(int r, int c) {
    if (CPR == 4) return c ^ ((r >> 1) & 3);
    if (CPR == 8) return c ^ ((r >> 1) & 7);
    if (CPR == 12) return c ^ ((r >> 2) & 3);
    if (CPR == 24) return c ^ ((r >> 1) & 7);
    return c ^ (r & 15);
  }
  // fp16: the 64-byte units of four rows that a transposed read takes; fp32: the 128-byte units of two rows
  // four apart that a step takes
  __device__ static __forceinline__ int place_v(int r, int c) {
    if (F16) return DP == 64 ? c ^ (4 * ((r >> 1) & 1)) : DP >= 128 ? c ^ (4 * (r & 3)) : c;
    return DP == 32 || DP == 96 ? c : c ^ (8 * ((r >> 2) & 1));
  }
  // fp32 rows of 32 or 96 channels: neighbours change places instead
  __device__ static __forceinline__ int row_v(int r) {
    return !F16 && (DP == 32 || DP == 96) ? r ^ ((r >> 2) & 1) : r;
  }
};

// fp16 on v_mfma_f32_32x32x16_f16: lane (r = l % 32, h = l / 32) supplies A[r][8h .. 8h + 7] and B[8h .. 8h + 7][r]
// and holds D[8a + 4h + c][r] in element 4a + c.
//   S^T = K Q^T for blocks of 32 keys x 32 queries: a query's scores lie in the two lanes r and r + 32.
//   O^T = V^T P^T for 16 keys x 32 channels at a time: a lane's probabilities 8s .. 8s + 7 (keys 16s + 4h .. + 3
//   and 16s + 8 + 4h .. + 3) are the B operand as they lie; the A operand takes the same keys of V by two
//   transposed reads.
// fp32 on v_mfma_f32_32x32x2_f32 (A[r][h], B[h][r], D as above), products and probabilities in fp32:
//   S^T: step s takes channels s and s + DP / 2, so that a lane's values of Q are neighbours.
//   O^T: the two keys of step e are those of the lanes' element e.
template <bool F16, int DP, int KS, Scores HOW>
__global__ __launch_bounds__(256, DP == 256 ? 1 : KS == 1 && (F16 ? !any(HOW) || DP < 128 : DP == 64) ? 3 : 2) void attn_masked_tiles(MaskedArgs a, ScoreArgs sc) {
  using T = Tile<F16, DP, KS>;
  using E = typename T::T;
  constexpr int KT = T::KT, QB = 128 / KS, NDT = DP / 32, NST = T::NST;
  constexpr int JOIN = (KS - 1) * (4 / KS) * Softmax<NDT>::BOX * 256;
  constexpr int BIAS_BYTES = any(HOW) ? 2 * T::BIASES * 4 : 0;
  constexpr int BYTES = T::RING + BIAS_BYTES > JOIN ? T::RING + BIAS_BYTES : JOIN;
  __shared__ __attribute__((aligned(1024))) char lds[BYTES];
  __shared__ int ends[4][2];
  float* const bt0 = reinterpret_cast<float*>(lds + T::RING);

  Place<KS> w(a);
  const int lane = w.lane, r = w.r, h = w.h;
  // Q, in the order its operand takes it: half8 s is channels 16s + 8h .., floatx4 c channels DP / 2 h + 4c ..
  typedef typename std::conditional<F16, half8, floatx4>::type Piece;
  constexpr int PER = 16 / T::SIZE, NQ = F16 ? DP / 16 : DP / 8;
  Piece qf[NQ];
  {
    const E* const q = static_cast<const E*>(a.q) + (w.token + min(w.i, a.S - 1)) * a.q_row + w.head * a.D;
#pragma unroll
    for (int s = 0; s < NQ; ++s) {
      const int ch = F16 ? 16 * s + 8 * h : h * (DP / 2) + 4 * s;
      qf[s] = Piece{};
      if (ch < a.D) qf[s] = *reinterpret_cast<const Piece*>(q + ch);
    }
  }
  // what a score is multiplied by as its exponent is taken
  const float factor = HOW == Scores::kPlain ? sc.scale2 : HOW == Scores::kCapped ? (F16 ? 2.0f : 1.0f) * sc.cap2 : 1.0f;
  const bool tabled = any(HOW) && a.bias_kind == kBiasTable;
  const float slope2 = any(HOW) && a.bias_kind == kBiasSlopes ? a.bias[w.head] * kLog2e : 0.0f;
  const float* const table = a.bias + w.head * (2 * static_cast<size_t>(a.radius) + 1);  // if tabled
  w.look(a);
  if (lane == 0) {
    ends[w.wave][0] = w.keys.lo;
    ends[w.wave][1] = w.keys.hi;
  }
  int first, last;
  w.tiles(ends, KT, &first, &last);

  // copy i of a wavefront fills block 4 i + wave of a stage: K, then V
  const char* const kplane = reinterpret_cast<const char*>(static_cast<const E*>(a.k) + w.token * a.k_row + w.kvh * a.D);
  const char* const vplane = reinterpret_cast<const char*>(static_cast<const E*>(a.v) + w.token * a.v_row + w.kvh * a.D);
  const int krow = a.k_row * T::SIZE, vrow = a.v_row * T::SIZE, chunks = a.D * T::SIZE / 16;
  auto issue = [&](int tile, int stage) {
    const char* const kt = kplane + static_cast<size_t>(tile) * KT * krow;
    const char* const vt = vplane + static_cast<size_t>(tile) * KT * vrow;
    const int most = w.L - 1 - tile * KT;
    int mine = lane;
    // wide fp32 tiles: up to 32 offsets, made again for each tile rather than kept in registers
    if constexpr (!F16 && DP >= 96) asm volatile("" : "+v"(mine));
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) {
      constexpr int HALF = T::LOADS / 2;
      const int at = ((i < HALF ? i : i - HALF) * 4 + w.wave) * 64 + mine;
      const int row = i < HALF ? at / T::CPR : T::row_v(at / T::CPR);
      const int c = min(i < HALF ? T::place_k(row, at % T::CPR) : T::place_v(row, at % T::CPR), chunks - 1);
      dma16_at(i < HALF ? kt : vt,
               __umul24(static_cast<uint32_t>(min(row, most)), static_cast<uint32_t>(i < HALF ? krow : vrow)) +
                   16u * static_cast<uint32_t>(c),
               reinterpret_cast<_Float16*>(lds + stage * 2 * T::BYTES + (i * 4 + w.wave) * 1024));
    }
  };
  float bias = 0.0f;
  auto fetch_bias = [&](int tile) {
    // entry x: distance key - query of tile * KT - i0 + x - (QB - 1)
    if (tabled) {
      const int x = static_cast<int>(threadIdx.x), away = tile * KT - w.i0 + x - (QB - 1);
      if (x < KT + QB - 1) bias = log2_bias(table[min(max(away, -a.radius), a.radius) + a.radius]);
    }
  };
  auto store_bias = [&](int buffer) {
    if (tabled && static_cast<int>(threadIdx.x) < KT + QB - 1)
      bt0[buffer * T::BIASES + threadIdx.x] = bias;
  };

  Softmax<NDT> soft;
#pragma unroll
  for (int s = 0; s < NQ; ++s) {
    if (sc.q_sign != 1.0f) qf[s] *= static_cast<E>(sc.q_sign);
    // Q has come before the first copy goes out: the compiler does not see the copies, and a wait for Q that
    // it placed among them would wait for all
    asm volatile("" : "+v"(qf[s]));
  }
  if (first < last) {
    fetch_bias(first);
    store_bias(0);
  }
#pragma unroll
  for (int n = 0; n < NST - 1; ++n)
    if (first + n < last) issue(first + n, n);
  int stage = 0;
  for (int tile = first; tile < last; ++tile) {
    if constexpr (NST == 1) {
      wait_lgkmcnt<0>();
      stage_barrier();
      issue(tile, 0);
      wait_vmcnt<0>();
      stage_barrier();
    } else {
      if (tile + NST - 2 < last) wait_vmcnt<(NST - 2) * T::LOADS>();
      else wait_vmcnt<0>();
      wait_lgkmcnt<0>();  // this wavefront's reads of the stage that is filled next
      stage_barrier();
      if (tile + NST - 1 < last) issue(tile + NST - 1, stage == 0 ? NST - 1 : stage - 1);
    }
    if (tile + 1 < last) fetch_bias(tile + 1);
    const E* const kt = reinterpret_cast<const E*>(lds + stage * 2 * T::BYTES);
    const E* const vt = reinterpret_cast<const E*>(lds + stage * 2 * T::BYTES + T::BYTES);
    const int kb = w.group * T::NB * 32, j0 = tile * KT + kb;
    if (!w.skips(j0, 32 * T::NB)) {  // wavefront-uniform
      // while these products are issued, before the waves of the SIMD that are at their softmax: 1 x 4096 causal,
      // 16 heads of 128, 111 -> 101 us
      __builtin_amdgcn_s_setprio(1);
      floatx16 s[T::NB];
#pragma unroll
      for (int nb = 0; nb < T::NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[nb][e] = 0.0f;
#pragma unroll
      for (int nb = 0; nb < T::NB; ++nb)
#pragma unroll
        for (int st = 0; st < NQ; ++st) {
          const int c = F16 ? 2 * st + h : h * (T::CPR / 2) + st;
          const Piece kf = *reinterpret_cast<const Piece*>(kt + (kb + 32 * nb + r) * DP + PER * T::place_k(r, c));
          if constexpr (F16) {
            s[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[st], s[nb], 0, 0, 0);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              s[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[st][j], s[nb], 0, 0, 0);
          }
        }
#pragma unroll
      for (int nb = 0; nb < T::NB; ++nb) product_done(s[nb]);
      __builtin_amdgcn_s_setprio(0);
      if constexpr (HOW != Scores::kPlain) {
#pragma unroll
        for (int nb = 0; nb < T::NB; ++nb)
          score_block<F16, HOW>(s[nb], a, sc, slope2, static_cast<float>(j0 + 32 * nb + 4 * h - w.i),
                      bt0 + ((tile - first) & 1) * T::BIASES + kb + 32 * nb + 4 * h + QB - 1 - (w.qw * 32 + r));
      }
      if (w.partial(j0, 32 * T::NB)) {
#pragma unroll
        for (int nb = 0; nb < T::NB; ++nb) w.mask(s[nb], j0 + 32 * nb);
      }
      soft.raise(s, factor, F16 ? kLift : 0.0f);
#pragma unroll
      for (int nb = 0; nb < T::NB; ++nb) {
        auto probability = [&](int e) {
          return __builtin_amdgcn_exp2f(any(HOW) ? s[nb][e] - soft.base : fmaf(s[nb][e], factor, -soft.base));
        };
        const int kn = kb + 32 * nb;
        if constexpr (F16) {
          half8 p[2];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            // fp16 probabilities for the product with V: their rounding, averaged over the keys, is of the size
            // of the output's own. The sum is that of the rounded ones, in fp32.
            const half2v two = __builtin_convertvector((float2v){probability(e), probability(e + 1)}, half2v);
            p[e >> 3][e & 7] = two.x;
            p[e >> 3][(e & 7) + 1] = two.y;
            soft.sum = __builtin_amdgcn_fdot2(two, half2v{1, 1}, soft.sum, false);
          }
          const int at = kn + 4 * h + ((lane & 15) >> 2);  // the row that this lane names
          const int in = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
          for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
              // rows 8 apart share their placing; chunk 4 dt is the block's first
              const int ch = 8 * T::place_v(at + 16 * st, 4 * dt) + in;
              const half4 v0 = read_transposed(vt + (at + 16 * st) * DP + ch);
              const half4 v1 = read_transposed(vt + (at + 16 * st + 8) * DP + ch);
              const half8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
              soft.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[st], soft.o[dt], 0, 0, 0);
            }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[nb][e] = probability(e);
            soft.sum += s[nb][e];
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int at = kn + 8 * (e >> 2) + 4 * h + (e & 3);
            const E* const vr = vt + T::row_v(at) * DP;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
              soft.o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vr[4 * T::place_v(at, 8 * dt) + r], s[nb][e], soft.o[dt], 0, 0, 0);
          }
        }
      }
    }
    if (tile + 1 < last) store_bias((tile + 1 - first) & 1);
    stage = stage + 1 == NST ? 0 : stage + 1;
  }
  wait_lgkmcnt<0>();
  __syncthreads();  // the ring is read out
  if (soft.join(w, reinterpret_cast<float*>(lds))) soft.template store<E>(a, w);
}

template <bool F16, int DP, int KS>
hipError_t launch_tiles(const MaskedArgs& a, const ScoreArgs& s, hipStream_t st) {
  constexpr int QB = 128 / KS;
  const dim3 grid(static_cast<unsigned>(static_cast<uint64_t>(a.B) * a.H * ((a.S + QB - 1) / QB)));
  if constexpr (F16 || DP < 256 || KS == 1)
    if (a.bias_kind != kBiasNone) {
      attn_masked_tiles<F16, DP, KS, Scores::kAny><<<grid, 256, 0, st>>>(a, s);
      return hipGetLastError();
    }
  if (a.cap > 0.0f)
    attn_masked_tiles<F16, DP, KS, Scores::kCapped><<<grid, 256, 0, st>>>(a, s);
  else
    attn_masked_tiles<F16, DP, KS, Scores::kPlain><<<grid, 256, 0, st>>>(a, s);
  return hipGetLastError();
}

// How the keys of a block of queries are shared out: KS groups of wavefronts, 128 / KS queries a workgroup.
// More groups shorten the walk over the keys and fill a chip that few workgroups would leave idle, and read
// K and V oftener. W: workgroups at KS = 1; in us, KS = 1, 2 and 4 (up to 128 channels):
//   one block of keys at most             17 x 5, 36 heads of 128, fp32            23.3  35.4  41.6
//   W <= 72, from 128 keys on             fp16 1 x 5720, 1 head of 32, documents   56.7  32.9  23.8
//                                         fp32 3 x 1210, 2 heads of 64, causal    107.4  64.1  41.5
//   W <= 512                              fp16 1 x 4096, 16 heads of 128, causal  131   110      -
//                                         fp32 8 x 1589, 4 heads of 32, causal     95.8  71.3  77.8
//     beyond                              fp16 5 x 1971, 8 heads of 64, W 640      64.1  76.0  94.2
//   twice that with spans, up to 64 channels or from 96 in fp32 (a block's documents may lie far apart)
//                                         fp16 1 x 8192, 12 heads of 64           103    80     -
//   W <= 256 where one workgroup's tiles fill a compute unit (fp32 from 96 channels, 256 channels)
//                                         fp32 10 x 1518, 4 heads of 128          208   120     -
//     beyond                              fp16 26 x 402, 4 heads of 256, W 416     49.1  59.4   -
template <bool F16, int DP>
hipError_t launch_split(const MaskedArgs& a, const ScoreArgs& s, hipStream_t st) {
  if constexpr (F16)
    if (a.cap > kCoarseCap) {
      attn_masked_tiles<F16, DP, 1, Scores::kAnyFine>
          <<<dim3(static_cast<unsigned>(static_cast<uint64_t>(a.B) * a.H * ((a.S + 127) / 128))), 256, 0, st>>>(a, s);
      return hipGetLastError();
    }
  constexpr bool FILLS = DP == 256 || (!F16 && DP >= 96);
  const int64_t w = int64_t{a.B} * a.H * ((a.S + 127) / 128);
  const int64_t reach = a.window ? std::min<int64_t>(a.S, 2 * int64_t{a.window} + 128) : a.S;
  if constexpr (DP <= 128)
    if (w <= 72 && reach >= 128) return launch_tiles<F16, DP, 4>(a, s, st);
  // (with a bias, two groups of fp32 of 256 channels would not fit their registers: launch_tiles has none)
  const bool two = F16 || DP < 256 || a.bias_kind == kBiasNone;
  if (two && reach > 32 && w <= (FILLS ? 256 : 512) * (a.spans && (FILLS || DP <= 64) ? 2 : 1))
    return launch_tiles<F16, DP, 2>(a, s, st);
  return launch_tiles<F16, DP, 1>(a, s, st);
}

template <bool F16>
hipError_t launch_sized(const MaskedArgs& a, const ScoreArgs& s, hipStream_t st) {
  if (a.D <= 32) return launch_split<F16, 32>(a, s, st);
  if (a.D <= 64) return launch_split<F16, 64>(a, s, st);
  if (a.D <= 96) return launch_split<F16, 96>(a, s, st);
  if (a.D <= 128) return launch_split<F16, 128>(a, s, st);
  return launch_split<F16, 256>(a, s, st);
}

}  // namespace

bool attention_masked_fits(uint64_t B, uint64_t S, uint64_t H, uint64_t D) {
  // a launch's work items stay below 2^32: attn_masked_rows has 64 for a row; with more tokens than it takes, a
  // block of queries has 256
  static_assert(kFewTokens >= 4, "2^26 / 5 blocks of 256 work items");
  return D % 8 == 0 && D <= 256 && B * S * H < (1ull << 26);
}

hipError_t launch_attention_masked(const MaskedArgs& a, hipStream_t st) {
  if (a.S <= (a.D > 128 || (!a.f16 && a.D > 64) ? 2 * kFewTokens : kFewTokens)) {
    const dim3 grid(static_cast<unsigned>((static_cast<uint64_t>(a.B) * a.S * a.H + 3) / 4));
    if (a.f16) attn_masked_rows<_Float16><<<grid, 256, 0, st>>>(a);
    else attn_masked_rows<float><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
  }
  const float size = fabsf(a.scale) * kLog2e;
  ScoreArgs s{};
  s.q_sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
  s.scale2 = a.cap > 0.0f ? 2.0f * size / a.cap : a.scale == 0.0f ? 1.0f : size;
  s.cap2 = a.cap * kLog2e;
  return a.f16 ? launch_sized<true>(a, s, st) : launch_sized<false>(a, s, st);
}

}  // namespace tessery
