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
// weights are integers, round(w 2^s) with s = 62 - ceil(log2 V), which 64 bits sum exactly in any
// order.  The exponential is taken in 64 bits: with 2^-44 of the largest weight as the step
// and a hundred thousand tokens, a border lies within rounding of u with probability 1e-8.
//
// One block per row.  Thresholds come from radix descents over the logits' bits, a byte at a
// time: of counts for top-k, of weights for top-p.
#include "cdx_common.h"

namespace cdx {
namespace {

constexpr int kThreads = 1024;
constexpr int kSampleWaves = kThreads / 64;
constexpr int kVec = 8;                       // tokens that a lane takes at a time
constexpr int kSpan = 64 * kVec;              // tokens that a wave takes at a time
constexpr int64_t kMaxVocab = 1 << 20;
constexpr int kMaxSpans = (int)(kMaxVocab / kSpan);

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

__device__ __forceinline__ float load_logit(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float load_logit(const uint16_t* p, int64_t i) { return bf16_bits_to_f32(p[i]); }

typedef unsigned long long u64;

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

template <typename TIn>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams p) {
  __shared__ u64 hist[256];
  __shared__ u64 spans[kMaxSpans];
  __shared__ u64 red[kSampleWaves];
  __shared__ u64 pick[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const TIn* x = static_cast<const TIn*>(p.logits) + row * p.ld;
  const int V = p.V;
  const float T = p.temperature ? p.temperature[row] : p.temperature1;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p1, min_p = p.min_p ? p.min_p[row] : p.min_p1;
  const int top_k = p.top_k ? p.top_k[row] : p.top_k1;

  // The largest logit and the first index that has it.
  u64 best = 0;
  for (int i = tid; i < V; i += kThreads) {
    const u64 c = (u64)logit_key(load_logit(x, i)) << 32 | (uint32_t)~i;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const u64 o = __shfl_xor(best, d, 64);
    best = o > best ? o : best;
  }
  if (lane == 0) red[wave] = best;
  __syncthreads();
  for (int w = 0; w < kSampleWaves; ++w) best = red[w] > best ? red[w] : best;
  const uint32_t top = (uint32_t)(best >> 32);
  const float top_x = key_logit(top);
  if (top_x == -INFINITY || !(T > 0.f)) {
    if (tid == 0) p.tokens[row] = top_x == -INFINITY ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
    return;
  }

  const double one = (double)(1ull << p.shift);
  // Weights as a fraction of the largest, and as integers.
  auto weight = [&](uint32_t key) -> double {
    if (key == top) return 1.0;
    const float v = key_logit(key);
    if (top_x == INFINITY || v == -INFINITY) return 0.0;  // (also at a temperature without bounds)
    return exp(((double)v - (double)top_x) / (double)T);
  };
  auto units = [&](double w) -> u64 { return (u64)(w * one + 0.5); };

  // top-k: the key of the k-th largest logit.
  uint32_t low = 0;
  if (top_k > 0 && top_k < V) {
    uint32_t prefix = 0;
    u64 need = top_k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t key = logit_key(load_logit(x, i));
        if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        u64 above = 0;
        int d = 255;
        while (d > 0 && above + hist[d] < need) above += hist[d--];
        pick[0] = d;
        pick[1] = above;
      }
      __syncthreads();
      prefix = prefix << 8 | (uint32_t)pick[0];
      need -= pick[1];
    }
    low = prefix;
  }

  // top-p: the smallest kept key, and how many of the tokens that have it are kept.
  uint32_t border = low;
  u64 border_count = ~0ull;
  if (top_p < 1.f) {
    u64 limit = 0, above = 0;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const uint32_t key = logit_key(load_logit(x, i));
        if (key >= low && (shift == 24 || key >> (shift + 8) == prefix))
          atomicAdd(&hist[(key >> shift) & 255], units(weight(key)));
      }
      __syncthreads();
      if (tid == 0) {
        if (shift == 24) {
          u64 total = 0;
          for (int d = 0; d < 256; ++d) total += hist[d];
          limit = (u64)((double)(top_p > 0.f ? top_p : 0.f) * (double)total);
        }
        // The last digit, from above, with weight before which the sum is within the limit.
        u64 sum = above;
        int last = 0;
        for (int d = 255; d >= 0 && sum <= limit; --d) {
          if (hist[d] == 0) continue;
          last = d;
          above = sum;
          sum += hist[d];
        }
        pick[0] = last;
        pick[1] = above;
        pick[2] = limit;
      }
      __syncthreads();
      prefix = prefix << 8 | (uint32_t)pick[0];
      above = pick[1];
      limit = pick[2];
    }
    border = prefix;
    border_count = (limit - above) / units(weight(border)) + 1;
  }

  // First index whose running sum of f exceeds a target, from the sums of spans of 512 tokens.
  const int n_spans = (V + kSpan - 1) / kSpan;
  auto span_sums = [&](auto f) {
    __syncthreads();
    for (int s = wave; s < n_spans; s += kSampleWaves) {
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int i = s * kSpan + e * 64 + lane;
        if (i < V) sum += f(i, logit_key(load_logit(x, i)));
      }
      sum = wave_sum(sum);
      if (lane == 0) spans[s] = sum;
    }
    __syncthreads();
  };
  // (Every thread returns the index; target < the sum over the row.)
  auto find = [&](auto f, u64 target) -> int {
    if (wave == 0) {
      int s = 0;
      u64 before = 0;
      while (s < n_spans - 1 && before + spans[s] <= target) before += spans[s++];
      int at = -1;
      for (int e = 0; e < kVec && at < 0; ++e) {
        const int i = s * kSpan + e * 64 + lane;
        u64 run = i < V ? f(i, logit_key(load_logit(x, i))) : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const u64 up = __shfl_up(run, d, 64);
          if (lane >= d) run += up;
        }
        const u64 hit = __ballot(before + run > target);
        if (hit != 0) at = s * kSpan + e * 64 + __builtin_ctzll(hit);
        before += __shfl(run, 63, 64);
      }
      if (lane == 0) pick[0] = (u64)(at < 0 ? V - 1 : at);
    }
    __syncthreads();
    return (int)pick[0];
  };

  // Ties at the border are kept in the order of their indices.
  int last_tie = V;
  if (border_count != ~0ull) {
    auto tie = [&](int, uint32_t key) -> u64 { return key == border ? 1 : 0; };
    span_sums(tie);
    u64 count = 0;
    for (int s = lane; s < n_spans; s += 64) count += spans[s];
    count = wave_sum(count);
    if (count > border_count) last_tie = find(tie, border_count - 1);
  }
  auto allowed = [&](int i, uint32_t key) {
    if (key < border || (key == border && i > last_tie)) return false;
    return !(min_p > 0.f) || key == top || weight(key) >= (double)min_p;
  };
  auto kept = [&](int i, uint32_t key) -> u64 { return allowed(i, key) ? units(weight(key)) : 0; };
  const float u = p.uniforms[row];
  if (!(u > 0.f)) {
    // The first kept token of any weight, also of one that rounds to no unit.
    auto any = [&](int i, uint32_t key) -> u64 { return allowed(i, key) && weight(key) > 0.0 ? 1 : 0; };
    span_sums(any);
    const int token = find(any, 0);
    if (tid == 0) p.tokens[row] = token;
    return;
  }
  span_sums(kept);
  u64 total = 0;
  for (int s = lane; s < n_spans; s += 64) total += spans[s];
  total = wave_sum(total);
  u64 target = (u64)((double)(u < 1.f ? u : 1.f) * (double)total);
  if (target >= total) target = total - 1;
  const int token = find(kept, target);
  if (tid == 0) p.tokens[row] = token;
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
  p.logits = logits;
  p.ld = ld;
  p.V = (int32_t)V;
  p.shift = 62 - bits;
  p.uniforms = uniforms;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature1 = temperature1;
  p.top_p1 = top_p1;
  p.min_p1 = min_p1;
  p.top_k1 = top_k1;
  p.tokens = tokens;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (logits_fp32)
    sample_kernel<float><<<dim3((unsigned)B), dim3(kThreads), 0, s>>>(p);
  else
    sample_kernel<uint16_t><<<dim3((unsigned)B), dim3(kThreads), 0, s>>>(p);
  return check_launch(name);
}
