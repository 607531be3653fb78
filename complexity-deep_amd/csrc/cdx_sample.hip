// Choosing the next token from logits and given random numbers, for gfx950.
//
//   w_i = exp((x_i - max x) / T)                    temperature (T == 0: the first maximum)
//   top-k   keeps x_i >= the k-th largest logit     (all that tie with it)
//   top-p   keeps, in descending order and by index among equals, the tokens before which the
//           kept weights sum to no more than p times their total
//   min-p   keeps w_i >= min_p                      (the largest weight is 1)
//   token   the first i whose running sum of kept weights exceeds u times their total
//
// A token is right or wrong, so the sums must not depend on the order in which threads add:
// weights are integers, round(w 2^s) with s = 62 - ceil(log2 V) (at most 51), which 64 bits sum
// exactly in any order.  The exponential is taken in 64 bits, to about 2^-47: with a hundred
// thousand tokens a border lies within the rounding of u with a probability around 1e-8.
//
// One block per row, no sort.  Each of its 16 waves walks a contiguous part of the row, a span
// of 64 pieces of 16 bytes at a time, so that a wave's order is the order of the indices.
//   * The first pass takes the maximum, and each thread's own.  The k-th largest of those 1024
//     is a lower bound of the k-th largest logit; min-p gives a bound as well (where no top-p
//     needs the sum over the tokens below it).
//   * Few tokens pass a bound: a second pass lists them, in order, in LDS, and everything else
//     (the exact k-th, top-p, the draw) happens among at most 256 a wave, four to a lane.
//   * Without a bound, or with more than the lists hold, thresholds come from a histogram, and the
//     draw sums the kept weights by span.  bf16 logits take few values: those within reach of the
//     top are counted one by one, and a table in LDS holds their weights, one exponential each.
//     fp32 logits are summed in 8192 bins of x (of counts for top-k, of weights for top-p), whose
//     border bin is then resolved by a radix descent over its few tokens; their passes are paced
//     by the exponentials, about 20 instructions in 64 bits a token.
//
// Measured (us of the kernel): 1 x 100000 bf16, top-k 50 and top-p 0.9, 16.3, of which 2.2 is the pass
// over the row by one CU, 3.4 the bound, 3.8 the list, 4.7 the wave's choice; 256 x 100000 bf16, top-p by
// row, 46 (a block with a cut: maximum 3, counts 10, table and border 6, sums 14, draw 3, 36 in all; the
// rest is the launch and the slowest rows); one row of those, 36; 64 x 32000 fp32, min-p, 10.5; fp32 with
// top-p, 1 x 100000 78, 256 x 100000 105; the first maximum (T == 0) of 1 x 100000 bf16 7.5, of 256 12.9.
// With radix passes over the row in place of bounds, lists and counts the first three
// took 310, 456 and 46.  A row held in registers for the counts and sums too spilled (256 rows 113), as
// did eight loads ahead instead of four (64 x 32000 17); a bound by waves instead of by the block (the
// least of the waves' own) listed too many (42).
#include <float.h>

#include <algorithm>

#include "cdx_common.h"
#include "cdx_wave.h"

namespace cdx {
namespace {

constexpr int kThreads = 1024;
constexpr int kSampleWaves = kThreads / 64;
constexpr int64_t kMaxVocab = 1 << 20;
constexpr int kListWave = 256;                // tokens that a wave can list
constexpr int kLane = kListWave / 64;
constexpr int kList = kListWave * kSampleWaves;
// Pieces of a row that a lane can hold.  bf16 rows gain by more of them, and the fp32 kernel spills them: 9
// of its registers with 8 pieces, 56 with 13, 112 with 16 (us with 8, 13 and 16: top-k, 1 x 100000 bf16 17.3,
// 16.4, 16.6, 1 x 131072 16.6, 16.5, 16.2; min-p at T = 1, 64 x 32000 fp32 12.5, 13.2, 17.2, 64 x 65536 17.3,
// 17.6, 21.7).
constexpr int kHeld = 13;
constexpr int kBins = 8192;

struct SampleParams {
  const void* logits;  // [B] rows of V at stride ld
  int64_t ld;
  int32_t V, shift;
  const float* uniforms;     // [B]
  const float* temperature;  // [B] or nullptr: the scalar
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature1, top_p1, min_p1;
  int32_t top_k1;
  int64_t* tokens;  // [B]
};

// Order of logits as unsigned integers: -0 = +0; NaN counts as -inf.
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x);
  if (u == 0x80000000u) return 0x80000000u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// One row, in pieces of 16 bytes at 16-byte addresses: piece c holds tokens c * VEC - head ..
// + VEC - 1, those outside 0 .. V - 1 as -inf.
template <typename TIn>
struct Row {
  static constexpr int VEC = 16 / sizeof(TIn);
  typedef __attribute__((ext_vector_type(4))) unsigned int piece_t;
  const TIn* x;  // of token -head (not read before token 0)
  int V, head, pieces;
  int lo, hi;  // the pieces that lie inside the row

  __device__ __forceinline__ Row(const TIn* row, int V_) : V(V_) {
    head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(TIn));
    x = row - head;
    pieces = (head + V + VEC - 1) / VEC;
    lo = head > 0 ? 1 : 0;
    hi = (head + V) / VEC - 1;
  }
  static __device__ __forceinline__ void unpack(const piece_t& v, float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(v[e]);
  }
  static __device__ __forceinline__ void unpack(const piece_t& v, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(v[e] << 16);
      f[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
    }
  }
  // A piece that does not lie inside the row, token by token.
  __device__ __forceinline__ piece_t edge(int c) const {
    piece_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sizeof(TIn) == 2 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int i = c * VEC + e - head;
      if (i < 0 || i >= V) continue;
      if constexpr (sizeof(TIn) == 2)
        v[e / 2] = e & 1 ? (v[e / 2] & 0xffffu) | (uint32_t)x[c * VEC + e] << 16
                         : (v[e / 2] & 0xffff0000u) | (uint32_t)x[c * VEC + e];
      else
        v[e] = __float_as_uint(x[c * VEC + e]);
    }
    return v;
  }
  // f(span, first token, piece) over the spans s0 <= span < s1.  AHEAD loads are on their way
  // together (a piece that does not lie inside the row loads one that does, in its place).
  template <typename F>
  __device__ __forceinline__ void each_piece(int s0, int s1, int lane, F f) const {
    constexpr int AHEAD = 4;
    for (int s = s0; s < s1; s += AHEAD) {
      piece_t raw[AHEAD];
      if (lo <= hi) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int c = max(lo, min(hi, (s + a) * 64 + lane));
          raw[a] = *reinterpret_cast<const piece_t*>(x + (int64_t)c * VEC);
        }
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        if (s + a >= s1) break;
        const int c = (s + a) * 64 + lane;
        if (c < lo || c > hi) raw[a] = edge(c);
        f(s + a, c * VEC - head, raw[a]);
      }
    }
  }
  // All pieces of the spans s0 <= span < s1 <= s0 + HELD, on their way together.
  template <int HELD>
  __device__ __forceinline__ void hold(int s0, int s1, int lane, piece_t (&held)[HELD]) const {
    if (lo <= hi) {
#pragma unroll
      for (int a = 0; a < HELD; ++a) {
        const int c = max(lo, min(hi, (s0 + a) * 64 + lane));
        if (s0 + a < s1) held[a] = *reinterpret_cast<const piece_t*>(x + (int64_t)c * VEC);
      }
    }
#pragma unroll
    for (int a = 0; a < HELD; ++a) {
      const int c = (s0 + a) * 64 + lane;
      if (s0 + a < s1 && (c < lo || c > hi)) held[a] = edge(c);
    }
  }
  // As values.
  template <typename F>
  __device__ __forceinline__ void spans(int s0, int s1, int lane, F f) const {
    each_piece(s0, s1, lane, [&](int s, int i0, const piece_t& raw) {
      float v[VEC];
      unpack(raw, v);
      f(s, i0, v);
    });
  }
};

// exp((x - top) / T) and its integer, in about 20 instructions.
struct Weights {
  double top, per_t, unit;  // per_t: log2(e) / T; unit: 2^shift

  __device__ __forceinline__ Weights(float top_x, float T, int shift)
      : top((double)fminf(top_x, FLT_MAX)), per_t(1.4426950408889634 / (double)T), unit((double)(1ull << shift)) {}

  // 2^t = p 2^n, n the nearest integer to t (the low bits of t + 1.5 2^52), p = 1 + r q(r) with q
  // the interpolation of (2^r - 1) / r at the nine Chebyshev nodes of |r| <= 1/2: 2^r to 3.7e-14 of it.
  // A logit of -inf (whatever the temperature) and one far below the top weigh less than half a
  // unit: the exponent stops at -100.  Beside a top of +inf only +inf itself is asked for.
  __device__ __forceinline__ double fraction(float x) const {
    const double t = fmax(((double)fminf(x, FLT_MAX) - top) * per_t, -100.0);
    const double k = t + 6755399441055744.0, r = t - (k - 6755399441055744.0);
    double p = 1.0203121294744093e-07;
    p = __builtin_fma(p, r, 1.3255224885642954e-06);
    p = __builtin_fma(p, r, 1.5252686845242518e-05);
    p = __builtin_fma(p, r, 0.00015403455852420133);
    p = __builtin_fma(p, r, 0.0013333558179044413);
    p = __builtin_fma(p, r, 0.009618129159402609);
    p = __builtin_fma(p, r, 0.05550410866476042);
    p = __builtin_fma(p, r, 0.2402265069581299);
    p = __builtin_fma(p, r, 0.6931471805599453);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_bit_cast(double, __builtin_bit_cast(u64, p) + ((u64)(uint32_t)__builtin_bit_cast(u64, k) << 52));
  }
  // The bits of w 2^shift + 2^52 (below 2^53): kRaw and, in the low bits, the integer.  Sums of them
  // wrap, and are right after as many kRaw are taken off.
  static constexpr u64 kRaw = 0x4330000000000000ull;
  __device__ __forceinline__ u64 raw(double w) const {
    return __builtin_bit_cast(u64, __builtin_fma(w, unit, 4503599627370496.0));
  }
  __device__ __forceinline__ u64 units(double w) const { return raw(w) - kRaw; }
  __device__ __forceinline__ u64 units(float x) const { return units(fraction(x)); }
};

// Whether exp((x - top) / T) is above 0 at all in 64 bits, for the key of x (rare: u == 0).
__device__ __forceinline__ bool any_weight(uint32_t key, float top, float T) {
  const float x = key_logit(key);
  return x > -INFINITY && top < INFINITY && exp(((double)x - (double)top) / (double)T) > 0.0;
}

constexpr int kTable = kBins;  // values of bf16 logits

// bf16 values in order: from 2^-24 in magnitude on 128 steps a binade, positive and negative; those
// nearer to 0 share step 0.
constexpr int kLeastBits = 0x3380;  // 2^-24
__device__ __forceinline__ int value_step(float x) {
  const int u = (int)__float_as_uint(x), m = max((u >> 16) & 0x7fff, kLeastBits - 1) - (kLeastBits - 1);
  return u < 0 ? -m : m;
}
__device__ __forceinline__ float step_value(int s) {
  const uint32_t m = s == 0 ? 0u : (uint32_t)(abs(s) + kLeastBits - 1) << 16;
  return __uint_as_float(s < 0 ? m | 0x80000000u : m);
}
// For each of a piece's values: how many steps below the top it lies, at most `most` (also a NaN
// and -inf; one of step 0 gives any number up to that).
struct StepsBelow {
  int plus, minus;
  uint32_t most;
  __device__ __forceinline__ StepsBelow(int top_step, int most_)
      : plus(top_step + kLeastBits - 1), minus(top_step - kLeastBits + 1 + 32768), most((uint32_t)most_) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t word, bool high) const {
    const int t = high ? (int)word >> 16 : (int)(word << 16) >> 16;  // negative: its magnitude - 2^15
    return min((uint32_t)(t < 0 ? minus + t : plus - t), most);
  }
};
// Whether a piece holds a value of step 0.
template <typename P>
__device__ __forceinline__ bool has_tiny(const P& v) {
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  u16x2 least = __builtin_bit_cast(u16x2, v[0] & 0x7fff7fffu);
#pragma unroll
  for (int e = 1; e < 4; ++e) least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, v[e] & 0x7fff7fffu));
  return min(least[0], least[1]) < kLeastBits;
}

template <typename TIn>
struct Shared {
  static constexpr int kSpans = (int)(kMaxVocab * sizeof(TIn) / 1024) + 1;
  union {
    u64 bins[kBins];
    u64 table[kTable];
  };
  u64 sums[kSpans];
  int ties[kSpans];
  union {
    struct {
      uint32_t list_key[kList];
      int list_index[kList];
    };
    uint32_t counts[kTable];
  };
  u64 red[kSampleWaves];
  u64 pick[3];
  uint32_t range[2];
  int count[kSampleWaves];
  int total;
};

// Sum over the threads before this one, and over the block.
template <typename T, typename Sh>
__device__ __forceinline__ T block_exclusive(T v, Sh& sh, T& total) {
  const int wave = threadIdx.x >> 6;
  const T run = wave_inclusive(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh.red[wave] = (u64)run;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    before += w < wave ? (T)sh.red[w] : 0;
    total += (T)sh.red[w];
  }
  return before + run - v;
}

// Sum over the block, returned to every thread.
template <typename Sh>
__device__ __forceinline__ u64 block_sum(u64 v, Sh& sh) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) t += sh.red[w];
  return t;
}

// By wave 0: the last of 256 bins, from the highest down, that holds something and before which the
// sum is within the limit: (bin, that sum) into pick.
template <typename Sh>
__device__ __forceinline__ void pick_digit(Sh& sh, u64 above, u64 limit) {
  const int lane = threadIdx.x;
  u64 v[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) mine += v[i] = sh.bins[255 - 4 * lane - i];
  u64 before = above + wave_inclusive(mine) - mine, at = 0;
  int last = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (v[i] != 0 && before <= limit) {
      last = 255 - 4 * lane - i;
      at = before;
    }
    before += v[i];
  }
  const u64 lanes = __ballot(last >= 0);
  if (lanes != 0 && lane == 63 - __builtin_clzll(lanes)) {
    sh.pick[0] = (u64)last;
    sh.pick[1] = at;
  }
}

// The smallest key before which the items of larger keys weigh no more than the limit, and that
// weight.  each(f) calls f(key, weight) for the thread's items.  A byte at a time.
template <typename Sh, typename Each>
__device__ uint32_t descend(Sh& sh, u64& above, u64 limit, Each each) {
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) sh.bins[threadIdx.x] = 0;
    __syncthreads();
    each([&](uint32_t key, u64 w) {
      if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&sh.bins[(key >> shift) & 255], w);
    });
    __syncthreads();
    if (threadIdx.x < 64) pick_digit(sh, above, limit);
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)sh.pick[0];
    above = sh.pick[1];
  }
  return prefix;
}

template <typename TIn>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams p) {
  __shared__ Shared<TIn> sh;
  constexpr int VEC = Row<TIn>::VEC;
  typedef typename Row<TIn>::piece_t piece_t;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t b = blockIdx.x;
  const Row<TIn> row(static_cast<const TIn*>(p.logits) + b * p.ld, p.V);
  const int n_spans = (row.pieces + 63) / 64;
  const int per_wave = (n_spans + kSampleWaves - 1) / kSampleWaves;
  const int s0 = min(n_spans, wave * per_wave), s1 = min(n_spans, s0 + per_wave);
  const float T = p.temperature ? p.temperature[b] : p.temperature1;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p1, u = p.uniforms[b];
  float top_p = p.top_p ? p.top_p[b] : p.top_p1;
  int top_k = p.top_k ? p.top_k[b] : p.top_k1;

  // A row of up to 16 x 13 spans (106496 bf16 logits) stays in registers.
  piece_t held[kHeld];
  const bool holds = per_wave <= kHeld;
  auto each_span = [&](auto f) {
    if (holds) {
#pragma unroll
      for (int a = 0; a < kHeld; ++a) {
        if (s0 + a >= s1) break;
        float v[VEC];
        row.unpack(held[a], v);
        f(s0 + a, ((s0 + a) * 64 + lane) * VEC - row.head, v);
      }
    } else {
      row.spans(s0, s1, lane, f);
    }
  };
  if (holds) row.hold(s0, s1, lane, held);

  // The largest logit (fmaxf passes over NaN), of the thread and of the row.
  float mine = -INFINITY;
  each_span([&](int, int, const float(&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) mine = fmaxf(mine, v[e]);
  });
  float top = mine;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
  if (lane == 0) sh.red[wave] = __float_as_uint(top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) top = fmaxf(top, __uint_as_float((uint32_t)sh.red[w]));
  if (top == -INFINITY) {
    if (tid == 0) p.tokens[b] = -1;
    return;
  }
  if (!(T > 0.f)) {
    int first = p.V;
    if (mine == top)
      row.spans(s0, s1, lane, [&](int, int i0, const float(&v)[VEC]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (v[e] == top) first = min(first, i0 + e);
      });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) first = min(first, __shfl_xor(first, d, 64));
    __syncthreads();
    if (lane == 0) sh.red[wave] = (u64)first;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) first = min(first, (int)sh.red[w]);
    if (tid == 0) p.tokens[b] = first;
    return;
  }
  const Weights wt(top, T, p.shift);
  if (top_k >= p.V) top_k = 0;
  if (!(top_p < 1.f)) top_p = 1.f;
  if (top_p < 0.f) top_p = 0.f;
  const bool cut_p = top_p < 1.f;

  // A logit below `bound` is not kept, whatever the others are.  (Beside +inf nothing else weighs.)
  float bound = top == INFINITY ? INFINITY : -FLT_MAX;
  if (top_k > 0 && top_k <= min(row.pieces, kThreads)) {
    // The high half of the k-th largest key among the threads' maxima, by the first wave, which
    // halves the range between the least and the largest.  (A thread without tokens has -inf.)
    sh.list_key[tid] = logit_key(mine) >> 16;
    __syncthreads();
    if (wave == 0) {
      uint32_t key[kThreads / 64], lo = ~0u, hi = logit_key(top) >> 16;
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i) {
        key[i] = sh.list_key[i * 64 + lane];
        lo = min(lo, key[i]);
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) lo = min(lo, (uint32_t)__shfl_xor((int)lo, d, 64));
      while (lo < hi) {  // at least k keys reach lo, fewer hi + 1
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 64; ++i) n += key[i] >= mid ? 1 : 0;
        if (wave_sum(n) >= top_k)
          lo = mid;
        else
          hi = mid - 1;
      }
      if (lane == 0) sh.range[0] = lo << 16;
    }
    __syncthreads();
    if (sh.range[0] > logit_key(-FLT_MAX)) bound = fmaxf(bound, key_logit(sh.range[0]));
  }
  if (min_p > 0.f && !cut_p) {
    // x >= top + T ln(min_p), less what the rounding of a weight (far below 1e-9 of it), and here of
    // the bound to 32 bits, could make of it.
    const double low = (double)top + (double)T * (log((double)(min_p < 1.f ? min_p : 1.f)) - 1e-9);
    bound = fmaxf(bound, (float)(low - 1e-6 * (fabs((double)top) + fabs(low))));
  }
  const bool bounded = bound > -FLT_MAX || row.pieces * VEC <= kList;

  // The tokens that pass, in order, by wave; more than the list holds: count only.
  int listed = kListWave + 1;
  if (bounded) {
    listed = 0;
    each_span([&](int, int i0, const float(&v)[VEC]) {
      float most = v[0];
#pragma unroll
      for (int e = 1; e < VEC; ++e) most = fmaxf(most, v[e]);
      if (__ballot(most >= bound) == 0) return;
      int n = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) n += v[e] >= bound ? 1 : 0;
      const int incl = wave_inclusive(n);
      int at = listed + incl - n;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v[e] >= bound) {
          if (at < kListWave) {
            sh.list_key[wave * kListWave + at] = logit_key(v[e]);
            sh.list_index[wave * kListWave + at] = i0 + e;
          }
          ++at;
        }
      listed += read_lane(incl, 63);
    });
  }
  __syncthreads();
  if (lane == 0) sh.count[wave] = listed;
  __syncthreads();
  bool fits = true;
  int listed_all = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    fits = fits && sh.count[w] <= kListWave;
    listed_all += sh.count[w];
  }

  if (fits && listed_all <= kListWave) {
    // Few tokens: all that follows by one wave, without barriers.
    if (wave != 0) return;
    constexpr int SHIFT = sizeof(TIn) == 2 ? 16 : 0;  // (the other bits of a bf16 logit's key follow from these)
    uint32_t key[kLane];
    int index[kLane];
    u64 w[kLane];
    double wf[kLane];
    bool on[kLane];
    // Item i of all lies in the list of the last wave that begins at or before it.
    const int through = wave_inclusive(lane < kSampleWaves ? sh.count[lane] : 0);
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      const int i = r * 64 + lane;
      int from = 0, begin = 0;
#pragma unroll
      for (int v = 0; v < kSampleWaves - 1; ++v) {
        const int end = read_lane(through, v);
        from += i >= end ? 1 : 0;
        begin = i >= end ? end : begin;
      }
      on[r] = i < listed_all;
      const int at = on[r] ? from * kListWave + i - begin : 0;
      key[r] = on[r] ? sh.list_key[at] >> SHIFT : 0u;
      index[r] = sh.list_index[at];
      wf[r] = on[r] ? wt.fraction(key_logit(sh.list_key[at])) : 0.0;
      w[r] = on[r] ? wt.units(wf[r]) : 0;
    }
    uint32_t least = ~0u;
#pragma unroll
    for (int r = 0; r < kLane; ++r) least = on[r] ? min(least, key[r]) : least;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
    const uint32_t most = logit_key(top) >> SHIFT;
    if (top_k > 0) {
      // The smallest key that fewer than k keys exceed.
      uint32_t lo = least, hi = most;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int n = 0;
#pragma unroll
        for (int r = 0; r < kLane; ++r) n += __popcll(__ballot(on[r] && key[r] > mid));
        if (n < top_k)
          hi = mid;
        else
          lo = mid + 1;
      }
      least = lo;
#pragma unroll
      for (int r = 0; r < kLane; ++r) on[r] = on[r] && key[r] >= lo;
    }
    if (cut_p) {
      // The smallest key whose larger ones weigh no more than p of the sum; ties by index.
      u64 s = 0;
#pragma unroll
      for (int r = 0; r < kLane; ++r) s += on[r] ? w[r] : 0;
      const u64 limit = (u64)((double)top_p * (double)wave_sum(s));
      uint32_t lo = least, hi = most;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        u64 above = 0;
#pragma unroll
        for (int r = 0; r < kLane; ++r) above += on[r] && key[r] > mid ? w[r] : 0;
        if (wave_sum(above) <= limit)
          hi = mid;
        else
          lo = mid + 1;
      }
      u64 above = 0, each = 0;
#pragma unroll
      for (int r = 0; r < kLane; ++r) {
        above += on[r] && key[r] > lo ? w[r] : 0;
        const u64 tie = __ballot(on[r] && key[r] == lo);
        if (tie != 0) each = read_lane(w[r], __builtin_ctzll(tie));
      }
      const u64 keep = each != 0 ? (limit - wave_sum(above)) / each + 1 : ~0ull;
      u64 before = 0;
#pragma unroll
      for (int r = 0; r < kLane; ++r) {
        const u64 tie = __ballot(on[r] && key[r] == lo);
        on[r] = on[r] && (key[r] > lo || (key[r] == lo && before + __popcll(tie & ((1ull << lane) - 1)) < keep));
        before += __popcll(tie);
      }
    }
    u64 s = 0;
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      const bool is_top = key[r] == most;
      on[r] = on[r] && (!(min_p > 0.f) || is_top || wf[r] >= (double)min_p);
      // u == 0: the first kept token of any weight, also of one that rounds to no unit.
      if (!(u > 0.f)) {
        const uint32_t low_bits = SHIFT != 0 && key[r] < 0x8000u ? 0xffffu : 0u;  // (of a negative logit's key)
        w[r] = is_top || any_weight(key[r] << SHIFT | low_bits, top, T) ? 1 : 0;
      }
      w[r] = on[r] ? w[r] : 0;
      s += w[r];
    }
    const u64 total = wave_sum(s);
    u64 target = u > 0.f ? (u64)((double)(u < 1.f ? u : 1.f) * (double)total) : 0;
    if (target >= total) target = total - 1;
    u64 before = 0;
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      const u64 run = before + wave_inclusive(w[r]);
      const u64 hit = __ballot(run > target);
      if (hit != 0) {
        if (lane == __builtin_ctzll(hit)) p.tokens[b] = index[r];
        return;
      }
      before = read_lane(run, 63);
    }
    return;
  }

  if (fits) {
    uint32_t key[kLane];
    int index[kLane];
    u64 w[kLane];
    double wf[kLane];
    bool on[kLane];
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      const int i = r * 64 + lane;
      on[r] = i < listed;
      key[r] = on[r] ? sh.list_key[wave * kListWave + i] : 0u;
      index[r] = on[r] ? sh.list_index[wave * kListWave + i] : 0;
    }
    if (top_k > 0) {
      u64 above = 0;
      const uint32_t low = descend(sh, above, (u64)top_k - 1, [&](auto f) {
#pragma unroll
        for (int r = 0; r < kLane; ++r)
          if (on[r]) f(key[r], 1);
      });
#pragma unroll
      for (int r = 0; r < kLane; ++r) on[r] = on[r] && key[r] >= low;
    }
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      wf[r] = on[r] ? wt.fraction(key_logit(key[r])) : 0.0;
      w[r] = on[r] ? wt.units(wf[r]) : 0;
    }
    if (cut_p) {
      u64 s = 0;
#pragma unroll
      for (int r = 0; r < kLane; ++r) s += w[r];
      const u64 total = block_sum(s, sh);
      const u64 limit = (u64)((double)top_p * (double)total);
      u64 above = 0;
      const uint32_t border = descend(sh, above, limit, [&](auto f) {
#pragma unroll
        for (int r = 0; r < kLane; ++r)
          if (w[r] != 0) f(key[r], w[r]);
      });
      const u64 keep = (limit - above) / wt.units(key_logit(border)) + 1;
      // Ties at the border by index: those of the waves before, then of this wave's items before.
      int ties = 0;
#pragma unroll
      for (int r = 0; r < kLane; ++r) ties += __popcll(__ballot(on[r] && key[r] == border));
      __syncthreads();
      if (lane == 0) sh.count[wave] = ties;
      __syncthreads();
      u64 before = 0;
      for (int v = 0; v < wave; ++v) before += sh.count[v];
#pragma unroll
      for (int r = 0; r < kLane; ++r) {
        const u64 tie = __ballot(on[r] && key[r] == border);
        const u64 rank = before + __popcll(tie & ((1ull << lane) - 1));
        on[r] = on[r] && (key[r] > border || (key[r] == border && rank < keep));
        before += __popcll(tie);
      }
    }
    u64 s = 0;
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      const bool is_top = key_logit(key[r]) == top;
      on[r] = on[r] && (!(min_p > 0.f) || is_top || wf[r] >= (double)min_p);
      // u == 0: the first kept token of any weight, also of one that rounds to no unit.
      if (!(u > 0.f)) w[r] = is_top || any_weight(key[r], top, T) ? 1 : 0;
      w[r] = on[r] ? w[r] : 0;
      s += w[r];
    }
    const u64 total = block_sum(s, sh);
    u64 target = u > 0.f ? (u64)((double)(u < 1.f ? u : 1.f) * (double)total) : 0;
    if (target >= total) target = total - 1;
    u64 before = 0;
    for (int v = 0; v < wave; ++v) before += sh.red[v];
    if (target < before || target >= before + sh.red[wave]) return;  // another wave's
#pragma unroll
    for (int r = 0; r < kLane; ++r) {
      const u64 run = before + wave_inclusive(w[r]);
      const u64 hit = __ballot(run > target);
      if (hit != 0) {
        if (lane == __builtin_ctzll(hit)) p.tokens[b] = index[r];
        return;
      }
      before = read_lane(run, 63);
    }
    return;
  }

  // Whole rows.  The border of a sum over the row (of counts or of weights), from the highest logit
  // down: by bins of equal width, then among the tokens of the border bin.
  auto border_of = [&](float per_x, auto limit_of, auto weight) -> uint32_t {
    // Bins count down from the top; those past the last one are the last one.
    auto bin = [&](float x) -> int {
      const float d = (top - x) * per_x;
      return d < (float)(kBins - 1) ? (int)d : kBins - 1;
    };
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    row.spans(s0, s1, lane, [&](int, int, const float(&v)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) atomicAdd(&sh.bins[bin(v[e])], weight(v[e]));
    });
    __syncthreads();
    constexpr int PER = kBins / kThreads;
    u64 w[PER], mass = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) mass += w[i] = sh.bins[tid * PER + i];
    u64 above = block_exclusive(mass, sh, total);
    const u64 limit = limit_of(total);
    if (above <= limit && above + mass > limit)  // (one thread)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (above <= limit && above + w[i] > limit) {
          sh.pick[0] = (u64)(tid * PER + i);
          sh.pick[1] = above;
        }
        above += w[i];
      }
    if (tid == 0) sh.total = 0;
    __syncthreads();
    const int chosen = (int)sh.pick[0];
    above = sh.pick[1];
    // The logits of that bin are an interval: its ends by halving the range of keys.
    if (tid < 2) {
      uint32_t lo = logit_key(-FLT_MAX), hi = logit_key(top);
      while (lo < hi) {  // lane 0: the first key at or below the bin; lane 1: the last at or above it
        const uint32_t mid = lo + (hi - lo + tid) / 2;
        const int at = bin(key_logit(mid));
        if (tid == 0) {
          if (at <= chosen)
            hi = mid;
          else
            lo = mid + 1;
        } else {
          if (at >= chosen)
            lo = mid;
          else
            hi = mid - 1;
        }
      }
      sh.range[tid] = lo;
    }
    __syncthreads();
    const float from = key_logit(sh.range[0]), to = key_logit(sh.range[1]);
    row.spans(s0, s1, lane, [&](int, int, const float(&v)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v[e] >= from && v[e] <= to) {
          const int at = atomicAdd(&sh.total, 1);
          if (at < kList) sh.list_key[at] = logit_key(v[e]);
        }
    });
    __syncthreads();
    const int n = sh.total;
    const uint32_t key = descend(sh, above, limit, [&](auto f) {
      if (n <= kList) {
        for (int i = tid; i < n; i += kThreads) {
          f(sh.list_key[i], weight(key_logit(sh.list_key[i])));
        }
      } else {
        row.spans(s0, s1, lane, [&](int, int, const float(&v)[VEC]) {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (v[e] >= from && v[e] <= to) f(logit_key(v[e]), weight(v[e]));
        });
      }
    });
    if (tid == 0) {
      sh.pick[1] = above;
      sh.pick[2] = limit;
    }
    __syncthreads();
    return key;
  };

  const bool any = !(u > 0.f);
  float border = -FLT_MAX;   // the least logit kept
  u64 keep = ~0ull;          // of those that equal it: so many by index, or all
  bool tabled = false;       // whether the weights of the values lie in the table
  int top_step = 0;
  const float cutoff = top - 45.f * T;  // logits below it weigh less than 2^-64
  if constexpr (sizeof(TIn) == 2) {
    top_step = value_step(top);
    const int steps = top_step - value_step(cutoff) + 2;  // (cutoff, cut to 16 bits, may round up a step)
    const bool stepped = fabsf(top) >= 0x1p-24f;
    tabled = stepped && !any && top < INFINITY && cutoff > -FLT_MAX && steps < kTable;
    if (tabled && (top_k > 0 || cut_p)) {
      __syncthreads();
      for (int i = tid; i < kTable; i += kThreads) sh.counts[i] = 0;
      if (tid == 0) {
        sh.total = 0;
        sh.pick[2] = 0;
      }
      __syncthreads();
      const StepsBelow below(top_step, steps);
      row.each_piece(s0, s1, lane, [&](int, int, const piece_t& v) {
        // (What lies below the cutoff goes to a count of its own.)
        if (__ballot(has_tiny(v)) == 0) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) atomicAdd(&sh.counts[below(v[e / 2], e & 1)], 1u);
          return;
        }
        // Step 0: counted together, weighed one by one.
        float f[VEC];
        row.unpack(v, f);
        u64 mass = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const bool tiny = fabsf(f[e]) < 0x1p-24f;
          if (!tiny) {
            atomicAdd(&sh.counts[below(v[e / 2], e & 1)], 1u);
          } else if (f[e] >= cutoff) {
            atomicAdd(&sh.counts[top_step], 1u);
            mass += wt.units(f[e]);
            if (f[e] != 0.f) sh.total = 1;  // (other values among them)
          }
        }
        mass = wave_sum(mass);
        if (lane == 0) atomicAdd(&sh.pick[2], mass);
      });
      __syncthreads();
    }
    if (tabled) {
      constexpr int PER = kTable / kThreads;
      const int i0 = tid * PER;
      const bool counted = top_k > 0 || cut_p;
      uint32_t n[PER];
      u64 w[PER];
      const u64 step0_mass = sh.pick[2];
      const int mixed = counted && sh.total != 0 ? top_step : -1;  // where different values are counted as one
      int last = steps;  // the step (from the top) of the k-th largest logit
#pragma unroll
      for (int i = 0; i < PER; ++i) n[i] = counted && i0 + i < steps ? sh.counts[i0 + i] : 0;
      if (top_k > 0) {
        int mine_n = 0, all_n;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine_n += (int)n[i];
        int before = block_exclusive(mine_n, sh, all_n);
        if (tid == 0) sh.range[0] = (uint32_t)steps;
        __syncthreads();
        if (before < top_k && before + mine_n >= top_k)  // (one thread, or none: fewer lie above the cutoff)
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            if (before < top_k && before + (int)n[i] >= top_k) sh.range[0] = (uint32_t)(i0 + i);
            before += (int)n[i];
          }
        __syncthreads();
        last = (int)sh.range[0];
      }
      // A k-th largest logit among different values counted as one: which of them stay is told by
      // the bins, and what top-p's total holds of them too.
      const bool split = last == mixed;
      border = last < steps ? step_value(top_step - last) : cutoff;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float x = step_value(top_step - i0 - i);
        const bool in = i0 + i <= last && i0 + i < steps && x >= cutoff;
        const double f = in ? wt.fraction(x) : 0.0;
        w[i] = in ? wt.units(f) : 0;
        sh.table[i0 + i] = i0 + i == 0 || !(min_p > 0.f) || f >= (double)min_p ? w[i] : 0;
      }
      if (cut_p && !split) {
        u64 mass = 0, total;
#pragma unroll
        for (int i = 0; i < PER; ++i) mass += i0 + i == mixed && mixed <= last ? step0_mass : n[i] * w[i];
        u64 before = block_exclusive(mass, sh, total);
        const u64 limit = (u64)((double)top_p * (double)total);
        if (before <= limit && before + mass > limit)  // (one thread)
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const u64 m = i0 + i == mixed && mixed <= last ? step0_mass : n[i] * w[i];
            if (before <= limit && before + m > limit) {
              sh.pick[0] = (u64)(i0 + i);
              sh.pick[1] = (limit - before) / w[i] + 1;
            }
            before += m;
          }
        __syncthreads();
        last = (int)sh.pick[0];
        border = step_value(top_step - last);
        keep = sh.pick[1];
      }
      tabled = !split && last != mixed;  // (a border among different values: by bins)
    }
  }
  if (!tabled) {
    float low = top == INFINITY ? INFINITY : -FLT_MAX;  // the least logit that top-k keeps
    if (top_k > 0) {
      // Bins over four times the spread of the threads' maxima.
      float least = mine > -INFINITY ? mine : top;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) least = fminf(least, __shfl_xor(least, d, 64));
      __syncthreads();
      if (lane == 0) sh.red[wave] = __float_as_uint(least);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kSampleWaves; ++w) least = fminf(least, __uint_as_float((uint32_t)sh.red[w]));
      const float spread = top - least;
      const float per_x = spread > 0.f && spread < INFINITY ? (float)(kBins / 4) / spread : 0.f;
      auto limit = [&](u64 n) { return (u64)top_k - 1 < n ? (u64)top_k - 1 : n - 1; };
      auto one = [](float x) -> u64 { return x >= -FLT_MAX ? 1 : 0; };
      low = fmaxf(low, key_logit(border_of(per_x, limit, one)));
    }
    border = low;
    if (cut_p) {
      // A weight below 2^-64 is no unit: bins over that many times T ln 2.
      const float range = 44.4f * T, per_x = range < 1e30f && range > 1e-30f ? (float)kBins / range : 0.f;
      border = key_logit(border_of(per_x, [&](u64 n) { return (u64)((double)top_p * (double)n); },
                                   [&](float x) -> u64 { return wt.units(x >= low ? x : -INFINITY); }));
      keep = (sh.pick[2] - sh.pick[1]) / wt.units(border) + 1;
    }
  }
  // Kept weights by span, the ties at the border counted apart.
  const bool by_ties = keep != ~0ull;
  auto kept = [&](float x) -> u64 {
    if (x == top) return any ? 1 : wt.units(x);
    const double w = wt.fraction(x);
    if (min_p > 0.f && !(w >= (double)min_p)) return 0;
    return any ? (any_weight(logit_key(x), top, T) ? 1 : 0) : wt.units(w);
  };
  // What is summed as it is: the logits above the border, or without ties from it on.
  const float least = by_ties ? key_logit(logit_key(border) + 1) : border;
  const u64 tie_w = by_ties ? kept(border) : 0;
  __syncthreads();
  if (tabled) {
    if constexpr (sizeof(TIn) == 2) {
      // Entries past the border are not looked at, its own counts the ties instead (in the high bits).
      constexpr int TIE = 56;
      const int last = top_step - value_step(border) + (by_ties || border != cutoff ? 0 : 1);
      if (tid == 0) {
        if (by_ties) sh.table[last] = 1ull << TIE;
        sh.table[last + 1] = 0;
      }
      __syncthreads();
      const StepsBelow below(top_step, last + 1);
      row.each_piece(s0, s1, lane, [&](int s, int, const piece_t& raw) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += sh.table[below(raw[e / 2], e & 1)];
        int ties = (int)(sum >> TIE);
        sum &= (1ull << TIE) - 1;
        if (__ballot(has_tiny(raw)) != 0) {  // one by one
          float v[VEC];
          row.unpack(raw, v);
          sum = 0;
          ties = 0;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            sum += v[e] >= least ? kept(v[e]) : 0;
            ties += by_ties && v[e] == border ? 1 : 0;
          }
        }
        sum = wave_sum(sum);
        if (by_ties) ties = wave_sum(ties);
        if (lane == 0) {
          sh.sums[s] = sum;
          sh.ties[s] = ties;
        }
      });
    }
  } else if (any || min_p > 0.f) {
    row.spans(s0, s1, lane, [&](int s, int, const float(&v)[VEC]) {
      u64 sum = 0;
      int ties = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (v[e] >= least) sum += kept(v[e]);
        ties += by_ties && v[e] == border ? 1 : 0;
      }
      sum = wave_sum(sum);
      ties = wave_sum(ties);
      if (lane == 0) {
        sh.sums[s] = sum;
        sh.ties[s] = ties;
      }
    });
  } else {
    row.spans(s0, s1, lane, [&](int s, int, const float(&v)[VEC]) {
      u64 sum = 0;
      int ties = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        sum += wt.raw(wt.fraction(v[e] >= least ? v[e] : -INFINITY));
        ties += v[e] == border ? 1 : 0;
      }
      sum = wave_sum(sum - VEC * Weights::kRaw);
      ties = wave_sum(ties);
      if (lane == 0) {
        sh.sums[s] = sum;
        sh.ties[s] = ties;
      }
    });
  }
  __syncthreads();
  if (wave != 0) return;
  // By the first wave: the spans' sums with their kept ties, then the span that the draw falls in.
  u64 total = 0, ties_before = 0;
  for (int base = 0; base < n_spans; base += 64) {
    const int s = base + lane;
    const u64 ties = by_ties && s < n_spans ? sh.ties[s] : 0;
    const u64 tie_at = ties_before + wave_inclusive(ties) - ties;
    const u64 mine_kept = tie_at >= keep ? 0 : (keep - tie_at < ties ? keep - tie_at : ties);
    const u64 sum = s < n_spans ? sh.sums[s] + mine_kept * tie_w : 0;
    if (s < n_spans) sh.sums[s] = sum;
    total += wave_sum(sum);
    ties_before += wave_sum(ties);
  }
  u64 target = any ? 0 : (u64)((double)(u < 1.f ? u : 1.f) * (double)total);
  if (target >= total) target = total - 1;
  u64 before = 0, rank = 0;
  int span = -1;
  for (int base = 0; base < n_spans && span < 0; base += 64) {
    const int s = base + lane;
    const u64 sum = s < n_spans ? sh.sums[s] : 0, ties = by_ties && s < n_spans ? sh.ties[s] : 0;
    const u64 run = wave_inclusive(sum), tie_run = wave_inclusive(ties);
    const u64 hit = __ballot(before + run > target);
    const int at = hit != 0 ? __builtin_ctzll(hit) : 63;
    // (Up to the span, or past all 64.)
    before += read_lane(run, at) - (hit != 0 ? read_lane(sum, at) : 0);
    rank += read_lane(tie_run, at) - (hit != 0 ? read_lane(ties, at) : 0);
    if (hit != 0) span = base + at;
  }
  row.spans(span, span + 1, lane, [&](int, int i0, const float(&v)[VEC]) {
    u64 w[VEC], sum = 0;
    int ties = 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) ties += by_ties && v[e] == border ? 1 : 0;
    u64 r = rank + wave_inclusive(ties) - ties;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const bool tie = by_ties && v[e] == border;
      const bool in = v[e] >= least || (tie && r < keep);
      r += tie ? 1 : 0;
      w[e] = in ? kept(v[e]) : 0;
      sum += w[e];
    }
    u64 run = before + wave_inclusive(sum) - sum;
    const u64 hit = __ballot(run + sum > target);
    if (hit == 0 || lane != __builtin_ctzll(hit)) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (run <= target && run + w[e] > target) p.tokens[b] = i0 + e;
      run += w[e];
    }
  });
}

}  // namespace
}  // namespace cdx

extern "C" int cdx_sample_tokens(const void* logits, int32_t logits_fp32, int64_t ld, int64_t B, int64_t V,
                                 const float* uniforms, const float* temperature, float temperature1,
                                 const int32_t* top_k, int32_t top_k1, const float* top_p, float top_p1,
                                 const float* min_p, float min_p1, int64_t* tokens, void* stream) {
  using namespace cdx;
  const char* name = "cdx_sample_tokens";
  clear_error();
  if (B < 0 || V <= 0) return fail(CDX_EINVAL, "%s: bad shape B=%lld V=%lld", name, (long long)B, (long long)V);
  if (V > kMaxVocab) return fail(CDX_EUNSUPPORTED, "%s: V=%lld exceeds %lld", name, (long long)V, (long long)kMaxVocab);
  if (B > INT32_MAX) return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (ld < V && B > 1) return fail(CDX_EINVAL, "%s: leading dimension too small", name);
  if ((!temperature && !(temperature1 >= 0.f)) || (!top_k && top_k1 < 0) ||
      (!top_p && !(top_p1 >= 0.f && top_p1 <= 1.f)) || (!min_p && !(min_p1 >= 0.f && min_p1 <= 1.f)))
    return fail(CDX_EINVAL, "%s: temperature and top_k must be >= 0, top_p and min_p in [0, 1]", name);
  if (B == 0) return CDX_OK;
  if (!logits || !uniforms || !tokens) return fail(CDX_EINVAL, "%s: null pointer", name);
  int bits = 0;
  while ((1ll << bits) < V) ++bits;
  SampleParams p{};
  p.ld = ld;
  p.V = (int32_t)V;
  p.shift = 62 - bits < 51 ? 62 - bits : 51;
  p.temperature1 = temperature1;
  p.top_p1 = top_p1;
  p.min_p1 = min_p1;
  p.top_k1 = top_k1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  for (int64_t b0 = 0; b0 < B; b0 += max_blocks(kThreads)) {
    p.logits = static_cast<const char*>(logits) + b0 * ld * (logits_fp32 ? 4 : 2);
    p.uniforms = uniforms + b0;
    p.temperature = temperature ? temperature + b0 : nullptr;
    p.top_k = top_k ? top_k + b0 : nullptr;
    p.top_p = top_p ? top_p + b0 : nullptr;
    p.min_p = min_p ? min_p + b0 : nullptr;
    p.tokens = tokens + b0;
    const dim3 grid((unsigned)std::min<int64_t>(B - b0, max_blocks(kThreads)));
    if (logits_fp32)
      sample_kernel<float><<<grid, dim3(kThreads), 0, s>>>(p);
    else
      sample_kernel<uint16_t><<<grid, dim3(kThreads), 0, s>>>(p);
    if (int rc = check_launch(name)) return rc;
  }
  return CDX_OK;
}
