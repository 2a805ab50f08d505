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
#include <stdlib.h>

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

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = min(x, __shfl_xor(x, off));
  return x;
}
__device__ __forceinline__ int wave_max_int(int x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = max(x, __shfl_xor(x, off));
  return x;
}

// Keys that some row of a wavefront attends (lo, hi) and keys that all its rows attend (all_lo, all_hi).
struct WaveKeys {
  int lo, hi, all_lo, all_hi;
};

__device__ __forceinline__ WaveKeys wave_keys(KeyRange r, bool row) {
  const bool some = row && r.lo < r.hi;
  WaveKeys w;
  w.lo = wave_min(some ? r.lo : 0x7fffffff);
  w.hi = wave_max_int(some ? r.hi : 0);
  w.all_lo = wave_max_int(!row ? 0 : some ? r.lo : 0x7fffffff);
  w.all_hi = wave_min(!row ? 0x7fffffff : some ? r.hi : 0);
  return w;
}

// The running maximum of a row moves when a tile exceeds it by more than kSlack (log2 units), and
// probabilities carry 2^kLift: at most 2^14 in fp16, and full fp16 precision down to 2^-20 of the
// largest. The softmax does not depend on either.
constexpr float kSlack = 8.0f, kLift = 6.0f;

// What the kernels on tiles take beside the arguments: signs and factors of the scores in log2 units.
struct ScoreArgs {
  float q_sign;  // -1 for a negative scale, 0 for none
  float scale2;  // |scale| log2 e; with a cap the factor in front of tanh's exponent, 2 |scale| log2 e / cap
  float cap2;    // cap log2 e
};

// Scores of one 32-key block as v (log2 units), still to be masked: element e of lane (query, h) is the
// key 8 (e / 4) + 4 h + e % 4 of the block. rel: the key of element 0 less the query's position.
template <bool CAP, int BIAS>
__device__ __forceinline__ void score_block(floatx16& v, const ScoreArgs& s, float slope2, float rel,
                                            const float* biases) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int c = 8 * (e >> 2) + (e & 3);
    float x = v[e];
    if constexpr (CAP) {
      // tanh(u) = 1 - 2 / (exp(2 u) + 1): exact at both ends, off by at most 2^-23 around 0
      const float t = __builtin_amdgcn_exp2f(x * s.scale2);
      x = fmaf(-2.0f * s.cap2, __builtin_amdgcn_rcpf(t + 1.0f), s.cap2);
    } else if constexpr (BIAS != kBiasNone) {
      x *= s.scale2;
    }
    if constexpr (BIAS == kBiasSlopes) x = fmaf(-slope2, fabsf(rel + static_cast<float>(c)), x);
    if constexpr (BIAS == kBiasTable) x += biases[c];
    v[e] = x;
  }
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

  __device__ __forceinline__ Place(const MaskedArgs& a, int (*ends)[2]) {
    lane = threadIdx.x & 63;
    r = lane & 31;
    h = lane >> 5;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    qw = wave % QW;
    group = wave / QW;
    const int blocks = (a.S + QB - 1) / QB;
    int at = static_cast<int>(blockIdx.x);
    const int qb = blocks - 1 - at % blocks;  // the last (causally longest) blocks of a head first
    at /= blocks;
    head = at % a.H;
    b = at / a.H;
    kvh = head / (a.H / a.KV);
    i0 = qb * QB;
    i = i0 + qw * 32 + r;
    row = i < a.S;
    mine = key_range(a, b, min(i, a.S - 1));
    keys = wave_keys(mine, row);
    if (lane == 0) {
      ends[wave][0] = keys.lo;
      ends[wave][1] = keys.hi;
    }
    L = static_cast<int>(min(a.lengths[b], static_cast<uint32_t>(a.S)));
    token = static_cast<size_t>(b) * a.S;
  }

  // the tiles of `size` keys that the workgroup walks; none where nothing is attended
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

  // whether no row of this wavefront attends a key of the block of 32 from j0, and whether some row does
  // not attend them all
  __device__ __forceinline__ bool skips(int j0) const { return j0 >= keys.hi || j0 + 32 <= keys.lo; }
  __device__ __forceinline__ bool partial(int j0) const {
    return j0 < keys.all_lo || j0 + 32 > keys.all_hi;
  }
  __device__ __forceinline__ void mask(floatx16& s, int j0) const {
    if (!partial(j0)) return;
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

  // takes in the block's largest score, `factor` times that of s
  __device__ __forceinline__ void raise(const floatx16& s, float factor, float lift) {
    float most = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) most = fmaxf(most, s[e]);
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
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[dt][e] = o[dt][e] * c0 + from[(16 * dt + e) * 64] * c1;
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

// Tiles of fp16 operands on v_mfma_f32_32x32x16_f16: lane (r = l % 32, h = l / 32) supplies A[r][8h ..
// 8h + 7] and B[8h .. 8h + 7][r] and holds D[8a + 4h + c][r] in element 4a + c.
//   S^T = K Q^T for blocks of 32 keys x 32 queries: a query's scores lie in the two lanes r and r + 32.
//   O^T = V^T P^T for 16 keys x 32 channels at a time: a lane's probabilities 8s .. 8s + 7 (keys 16s + 4h
//   .. + 3 and 16s + 8 + 4h .. + 3) are the B operand as they lie; the A operand takes the same keys of V
//   by two transposed reads.
// Four wavefronts: 4 / KS of them take 32 queries each and the KS groups every KS-th block of keys; the
// groups' sums meet in LDS at the end. K and V tiles of KT keys pass through registers into two LDS
// buffers, the next tile's loads in flight during the products; keys past the length become zeros.
// DP: the head size up to a power of two, zeros behind D.
template <int DP>
struct F16Tile {
  static constexpr int KT = DP == 256 ? 32 : 64;
  static constexpr int KROW = DP + 8;             // halves: 16 rows' chunks fall on 16 bank groups
  static constexpr int K = KT * KROW, V = KT * DP;
  static constexpr int CHUNKS = KT * DP / 8 / 256;  // 16-byte pieces a thread stages of K (and of V)
  static constexpr int BIASES = 192;              // distances of one tile, KT + 128 - 1
  static constexpr int BYTES = 2 * (K + V) * 2 + 2 * BIASES * 4;
};
// 64-byte units of a V row, so that the four rows of a transposed read fall on different banks
template <int DP>
__device__ __forceinline__ int v_unit(int row) {
  return DP >= 128 ? (row & 3) : DP == 64 ? ((row >> 1) & 1) : 0;
}

template <int DP, int KS, bool CAP, int BIAS>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_masked_f16(MaskedArgs a, ScoreArgs sc) {
  using T = F16Tile<DP>;
  constexpr int KT = T::KT, QB = 128 / KS, NS = DP / 16, NDT = DP / 32;
  constexpr int NB = KT / 32 / KS;  // key blocks of a tile that one wavefront takes
  static_assert(NB >= 1, "a block of keys for every group");
  __shared__ __attribute__((aligned(16))) char lds[T::BYTES];
  __shared__ int ends[4][2];
  _Float16* const kt0 = reinterpret_cast<_Float16*>(lds);
  _Float16* const vt0 = kt0 + 2 * T::K;
  float* const bt0 = reinterpret_cast<float*>(vt0 + 2 * T::V);

  const Place<KS> w(a, ends);
  const int tid = threadIdx.x, lane = w.lane, r = w.r, h = w.h, i = w.i;
  const int b = w.b, head = w.head, kvh = w.kvh, L = w.L;
  const size_t token = w.token;
  const int ic = min(i, a.S - 1);
  const _Float16* const q = static_cast<const _Float16*>(a.q) + (token + ic) * a.q_row + head * a.D;
  const _Float16* const k = static_cast<const _Float16*>(a.k) + token * a.k_row + kvh * a.D;
  const _Float16* const v = static_cast<const _Float16*>(a.v) + token * a.v_row + kvh * a.D;

  half8 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = half8{};
    if (16 * s + 8 * h < a.D) {
      qf[s] = *reinterpret_cast<const half8*>(q + 16 * s + 8 * h);
      if (sc.q_sign != 1.0f) qf[s] *= static_cast<_Float16>(sc.q_sign);
    }
  }
  const float slope2 = BIAS == kBiasSlopes ? a.bias[head] * kLog2e : 0.0f;
  const float* const table =
      BIAS == kBiasTable ? a.bias + head * (2 * static_cast<size_t>(a.radius) + 1) : nullptr;
  int first, last;
  w.tiles(ends, KT, &first, &last);

  // staging: thread t takes 16-byte pieces t, t + 256, ... of the tile
  half8 kreg[T::CHUNKS], vreg[T::CHUNKS];
  float breg = 0.0f;
  auto fetch = [&](int tile) {
#pragma unroll
    for (int c = 0; c < T::CHUNKS; ++c) {
      const int piece = tid + 256 * c, key = tile * KT + piece / (DP / 8), ch = piece % (DP / 8) * 8;
      kreg[c] = vreg[c] = half8{};
      if (key < L && ch < a.D) {
        kreg[c] = *reinterpret_cast<const half8*>(k + static_cast<size_t>(key) * a.k_row + ch);
        vreg[c] = *reinterpret_cast<const half8*>(v + static_cast<size_t>(key) * a.v_row + ch);
      }
    }
    if constexpr (BIAS == kBiasTable) {
      // entry x: distance key - query of tile * KT - i0 + x - (QB - 1)
      const int away = tile * KT - w.i0 + tid - (QB - 1);
      if (tid < KT + QB - 1) breg = log2_bias(table[min(max(away, -a.radius), a.radius) + a.radius]);
    }
  };
  auto stage = [&](int buffer) {
    _Float16* const kt = kt0 + buffer * T::K;
    _Float16* const vt = vt0 + buffer * T::V;
#pragma unroll
    for (int c = 0; c < T::CHUNKS; ++c) {
      const int piece = tid + 256 * c, key = piece / (DP / 8), ch = piece % (DP / 8);
      *reinterpret_cast<half8*>(kt + key * T::KROW + 8 * ch) = kreg[c];
      *reinterpret_cast<half8*>(vt + key * DP + 8 * (ch ^ (4 * v_unit<DP>(key)))) = vreg[c];
    }
    if constexpr (BIAS == kBiasTable)
      if (tid < KT + QB - 1) bt0[buffer * T::BIASES + tid] = breg;
  };

  Softmax<NDT> soft;
  if (first < last) {
    fetch(first);
    stage(0);
  }
  __syncthreads();
  for (int tile = first; tile < last; ++tile) {
    const int buffer = (tile - first) & 1;
    if (tile + 1 < last) fetch(tile + 1);
    const _Float16* const kt = kt0 + buffer * T::K;
    const _Float16* const vt = vt0 + buffer * T::V;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int kb = (KS == 1 ? nb : w.group) * 32, j0 = tile * KT + kb;
      if (w.skips(j0)) continue;  // wavefront-uniform
      floatx16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const half8 kf = *reinterpret_cast<const half8*>(kt + (kb + r) * T::KROW + 16 * st + 8 * h);
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[st], s, 0, 0, 0);
      }
      product_done(s);
      score_block<CAP, BIAS>(s, sc, slope2, static_cast<float>(j0 + 4 * h - i),
                             bt0 + buffer * T::BIASES + kb + 4 * h + QB - 1 - (w.qw * 32 + r));
      w.mask(s, j0);
      constexpr bool RAW = !CAP && BIAS == kBiasNone;  // still to be multiplied by scale2
      soft.raise(s, RAW ? sc.scale2 : 1.0f, kLift);
      half8 p[2];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(RAW ? fmaf(s[e], sc.scale2, -soft.base) : s[e] - soft.base);
        const float p1 =
            __builtin_amdgcn_exp2f(RAW ? fmaf(s[e + 1], sc.scale2, -soft.base) : s[e + 1] - soft.base);
        // fp16 probabilities for the product with V (they add 2^-12 of the output's own rounding,
        // 2^-11, in the mean); the sum is that of the rounded ones, in fp32
        const half2v two = __builtin_convertvector((float2v){p0, p1}, half2v);
        p[e >> 3][e & 7] = two.x;
        p[e >> 3][(e & 7) + 1] = two.y;
        soft.sum = __builtin_amdgcn_fdot2(two, half2v{1, 1}, soft.sum, false);
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const int vrow = kb + 16 * st + 4 * h + ((lane & 15) >> 2);
        const int ch = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          const half4 v0 = read_transposed(vt + vrow * DP + 32 * (dt ^ v_unit<DP>(vrow)) + ch);
          const half4 v1 =
              read_transposed(vt + (vrow + 8) * DP + 32 * (dt ^ v_unit<DP>(vrow + 8)) + ch);
          const half8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
          soft.o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[st], soft.o[dt], 0, 0, 0);
        }
      }
    }
    if (tile + 1 < last) stage(buffer ^ 1);
    __syncthreads();
  }
  static_assert((KS - 1) * (4 / KS) * Softmax<NDT>::BOX * 256 <= T::BYTES, "sums fit the tiles' LDS");
  if (soft.join(w, reinterpret_cast<float*>(lds))) soft.template store<_Float16>(a, w);
}

// Tiles of fp32 operands on v_mfma_f32_32x32x2_f32: lane (r, h) supplies A[r][h] and B[h][r], D as above.
//   S^T = K Q^T: step s takes channels s and s + DP / 2, so that a lane's values of Q are neighbours.
//   O^T = V^T P^T: the two keys of step e are those of the lanes' element e. A row of V lies in LDS with its
//   32-channel blocks interleaved, so one read gives a lane its channel of every block.
// Everything is fp32: products, sums, probabilities.
template <int DP>
struct F32Tile {
  static constexpr int KT = DP >= 128 ? 32 : 64;
  static constexpr int KROW = DP + 4;
  static constexpr int K = KT * KROW, V = KT * DP;
  static constexpr int CHUNKS = KT * DP / 4 / 256;
  static constexpr int BIASES = 192;
  static constexpr int BYTES = (2 * (K + V) + 2 * BIASES) * 4;
};

template <int DP, int KS, bool CAP, int BIAS>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attn_masked_f32(MaskedArgs a, ScoreArgs sc) {
  using T = F32Tile<DP>;
  constexpr int KT = T::KT, QB = 128 / KS, NDT = DP / 32, HALF = DP / 2;
  constexpr int NB = KT / 32 / KS;  // key blocks of a tile that one wavefront takes
  static_assert(NB >= 1, "a block of keys for every group");
  __shared__ __attribute__((aligned(16))) char lds[T::BYTES];
  __shared__ int ends[4][2];
  float* const kt0 = reinterpret_cast<float*>(lds);
  float* const vt0 = kt0 + 2 * T::K;
  float* const bt0 = vt0 + 2 * T::V;

  const Place<KS> w(a, ends);
  const int tid = threadIdx.x, r = w.r, h = w.h;
  const int ic = min(w.i, a.S - 1);
  const float* const q = static_cast<const float*>(a.q) + (w.token + ic) * a.q_row + w.head * a.D;
  const float* const k = static_cast<const float*>(a.k) + w.token * a.k_row + w.kvh * a.D;
  const float* const v = static_cast<const float*>(a.v) + w.token * a.v_row + w.kvh * a.D;
  floatx4 qf[HALF / 4];
#pragma unroll
  for (int c = 0; c < HALF / 4; ++c) {
    const int ch = h * HALF + 4 * c;
    qf[c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    if (ch < a.D) qf[c] = *reinterpret_cast<const floatx4*>(q + ch) * sc.q_sign;
  }
  const float slope2 = BIAS == kBiasSlopes ? a.bias[w.head] * kLog2e : 0.0f;
  const float* const table =
      BIAS == kBiasTable ? a.bias + w.head * (2 * static_cast<size_t>(a.radius) + 1) : nullptr;
  int first, last;
  w.tiles(ends, KT, &first, &last);

  floatx4 kreg[T::CHUNKS], vreg[T::CHUNKS];
  float breg = 0.0f;
  auto fetch = [&](int tile) {
#pragma unroll
    for (int c = 0; c < T::CHUNKS; ++c) {
      const int piece = tid + 256 * c, key = tile * KT + piece / (DP / 4), ch = piece % (DP / 4) * 4;
      kreg[c] = vreg[c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      if (key < w.L && ch < a.D) {
        kreg[c] = *reinterpret_cast<const floatx4*>(k + static_cast<size_t>(key) * a.k_row + ch);
        vreg[c] = *reinterpret_cast<const floatx4*>(v + static_cast<size_t>(key) * a.v_row + ch);
      }
    }
    if constexpr (BIAS == kBiasTable) {
      const int away = tile * KT - w.i0 + tid - (QB - 1);
      if (tid < KT + QB - 1) breg = log2_bias(table[min(max(away, -a.radius), a.radius) + a.radius]);
    }
  };
  auto stage = [&](int buffer) {
    float* const kt = kt0 + buffer * T::K;
    float* const vt = vt0 + buffer * T::V;
#pragma unroll
    for (int c = 0; c < T::CHUNKS; ++c) {
      const int piece = tid + 256 * c, key = piece / (DP / 4), ch = piece % (DP / 4) * 4;
      *reinterpret_cast<floatx4*>(kt + key * T::KROW + ch) = kreg[c];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        vt[key * DP + ((ch + j) & 31) * NDT + ((ch + j) >> 5)] = vreg[c][j];
    }
    if constexpr (BIAS == kBiasTable)
      if (tid < KT + QB - 1) bt0[buffer * T::BIASES + tid] = breg;
  };

  Softmax<NDT> soft;
  if (first < last) {
    fetch(first);
    stage(0);
  }
  __syncthreads();
  for (int tile = first; tile < last; ++tile) {
    const int buffer = (tile - first) & 1;
    if (tile + 1 < last) fetch(tile + 1);
    const float* const kt = kt0 + buffer * T::K;
    const float* const vt = vt0 + buffer * T::V;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int kb = (KS == 1 ? nb : w.group) * 32, j0 = tile * KT + kb;
      if (w.skips(j0)) continue;  // wavefront-uniform
      floatx16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int c = 0; c < HALF / 4; ++c) {
        const floatx4 kf = *reinterpret_cast<const floatx4*>(kt + (kb + r) * T::KROW + h * HALF + 4 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[c][j], s, 0, 0, 0);
      }
      product_done(s);
      score_block<CAP, BIAS>(s, sc, slope2, static_cast<float>(j0 + 4 * h - w.i),
                             bt0 + buffer * T::BIASES + kb + 4 * h + QB - 1 - (w.qw * 32 + r));
      w.mask(s, j0);
      constexpr bool RAW = !CAP && BIAS == kBiasNone;
      soft.raise(s, RAW ? sc.scale2 : 1.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(RAW ? fmaf(s[e], sc.scale2, -soft.base) : s[e] - soft.base);
        soft.sum += s[e];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float* const vr = vt + (kb + 8 * (e >> 2) + 4 * h + (e & 3)) * DP + r * NDT;
        float vf[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) vf[dt] = vr[dt];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
          soft.o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[dt], s[e], soft.o[dt], 0, 0, 0);
      }
    }
    if (tile + 1 < last) stage(buffer ^ 1);
    __syncthreads();
  }
  static_assert((KS - 1) * (4 / KS) * Softmax<NDT>::BOX * 256 <= T::BYTES, "sums fit the tiles' LDS");
  if (soft.join(w, reinterpret_cast<float*>(lds))) soft.template store<float>(a, w);
}

// f(CAP, BIAS) as compile-time values
template <typename F>
void for_scores(const MaskedArgs& a, F&& f) {
  using None = std::integral_constant<int, kBiasNone>;
  using Slopes = std::integral_constant<int, kBiasSlopes>;
  using Table = std::integral_constant<int, kBiasTable>;
  auto with = [&](auto cap) {
    if (a.bias_kind == kBiasNone) f(cap, None{});
    else if (a.bias_kind == kBiasSlopes) f(cap, Slopes{});
    else f(cap, Table{});
  };
  if (a.cap > 0.0f) with(std::true_type{});
  else with(std::false_type{});
}

template <bool F16, int DP, int KS>
hipError_t launch_tiles(const MaskedArgs& a, const ScoreArgs& s, hipStream_t st) {
  constexpr int QB = 128 / KS;
  const dim3 grid(static_cast<unsigned>(static_cast<uint64_t>(a.B) * a.H * ((a.S + QB - 1) / QB)));
  for_scores(a, [&](auto cap, auto bias) {
    if constexpr (F16)
      attn_masked_f16<DP, KS, decltype(cap)::value, decltype(bias)::value><<<grid, 256, 0, st>>>(a, s);
    else
      attn_masked_f32<DP, KS, decltype(cap)::value, decltype(bias)::value><<<grid, 256, 0, st>>>(a, s);
  });
  return hipGetLastError();
}

template <bool F16, int DP>
hipError_t launch_split(const MaskedArgs& a, const ScoreArgs& s, hipStream_t st) {
  static const int ks = getenv("TESSERY_KS") ? atoi(getenv("TESSERY_KS")) : 1;
  if constexpr (DP <= (F16 ? 128 : 64))
    if (ks == 2) return launch_tiles<F16, DP, 2>(a, s, st);
  return launch_tiles<F16, DP, 1>(a, s, st);
}

template <bool F16>
hipError_t launch_sized(const MaskedArgs& a, const ScoreArgs& s, hipStream_t st) {
  if (a.D <= 32) return launch_split<F16, 32>(a, s, st);
  if (a.D <= 64) return launch_split<F16, 64>(a, s, st);
  if (a.D <= 128) return launch_split<F16, 128>(a, s, st);
  return launch_split<F16, 256>(a, s, st);
}

}  // namespace

bool attention_masked_fits(uint64_t B, uint64_t S, uint64_t H, uint64_t D) {
  // a launch's work items stay below 2^32
  return D % 8 == 0 && D <= 256 && B * S * H < (1ull << 26);
}

hipError_t launch_attention_masked(const MaskedArgs& a, hipStream_t st) {
  const float size = fabsf(a.scale) * kLog2e;
  ScoreArgs s{};
  s.q_sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
  s.scale2 = a.cap > 0.0f ? 2.0f * size / a.cap : a.scale == 0.0f ? 1.0f : size;
  s.cap2 = a.cap * kLog2e;
  return a.f16 ? launch_sized<true>(a, s, st) : launch_sized<false>(a, s, st);
}

}  // namespace tessery
