// Attention of any number of new tokens per sequence over a paged KV cache, for gfx950.
//
//   o[r, h] = sum_t p_t v_t,  p = softmax_t(scale q[r, h] . k_t),  t <= t(r),
//
// t(r) = length[b] - count[b] + i being the slot of row r, the i-th new token of sequence b: it attends to
// everything before it and to itself.  Sequences bring different numbers of rows, which only the
// device knows.  The (row, query head) pairs of one (sequence, KV head) are its queries, row by
// row, so that a tile of queries shares K and V over the heads of the group as well as over rows.
//
//   paged_chunk_tile_kernel  tiles of 128 queries, four waves of 32.  K and V tiles of 64 slots by DMA from the
//     pages into LDS, a descriptor per 16 rows (which lie in one page); page numbers are looked up for 64
//     tiles at a time.  S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16_bf16: a lane holds 32 scores of
//     one query, P goes from the scores' registers straight into the second product, and V is
//     transposed as it is read from LDS (ds_read_b64_tr_b16).  While tile t's scores become weights, the
//     QK products of tile t + 1 run between them.  The matrix cores and the exponentials bound it:
//     1.07 to 1.1 PFLOP/s on long sequences, where a large library product reaches 1.27.
//   paged_chunk_few_kernel   for calls of at most 16 queries a sequence and KV head, which wait for memory or
//     latency: paged_attn_kernel's walk of the pages, the slots over eight waves and over splits, with the
//     columns of the matrix instruction taken by queries of several rows.
//
// Measured (us a call, issued back to back, and what of it bounds the call), 16/8 heads of 128 unless said:
// 2048 new tokens over 65536 slots 990 (1090 TFLOP/s), 8 x 1024 over 2048 113 to 117 (915), 8 prompts of 2048 158
// (871); 4 chunks of 512 among 60 single tokens, up to 2048 slots, 50 to 57 (227 MB: 4.0 to 4.5 TB/s); 16 of
// 1 .. 777 over up to 4099, 16/4 of 80, 82 to 85 (590); 4 x 512 over 4096, 12/4 of 64, 50 (481); 64 single tokens
// over 2049 94 (537 MB: 5.7 TB/s); 8 over 32768 31; 5 over 505, 8/4 of 40, 5.8.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "cdx_gemm.h"
#include "cdx_paged_attn.h"
#include "cdx_wave.h"

namespace cdx {
namespace {

struct ChunkParams {
  const uint16_t* q;  // [rows][nq][D]
  const uint16_t* k_pages;
  const uint16_t* v_pages;
  PagedTable t;
  const int32_t* starts;   // [B], ascending
  const int32_t* counts;   // [B]
  const int32_t* lengths;  // [B], the new tokens counted
  int32_t B, rows, nq, nkv, D, group;
  int32_t splits;   // of a tile's slots, at most
  int32_t piece;    // of the tile kernel: tiles of keys of a split
  uint32_t tiles;   // of the tile kernel: numbers that a tile may have
  float scale_log2;
  uint16_t* out;    // [rows][nq][D]
  // Partial sums by split, row and head.
  float* part_o;    // [splits][rows][nq][D], unnormalised
  float2* part_ml;  // maximum (log2 units) and sum; a sum of -1: no key at all
};

constexpr int kFew = 16;  // queries of a block: the columns of a matrix instruction

// A tile of queries of one sequence: rows begin .. of the call, row r being token r - first of the sequence.
struct ChunkTile {
  int b;
  int32_t begin, first, count, before;  // before: slots in use ahead of the new tokens
  int32_t m0, queries;                  // the tile's first query, and how many the rows have

  __device__ __forceinline__ bool any() const { return m0 < queries; }
  // The token that query m belongs to; outside 0 .. count - 1: none.
  __device__ __forceinline__ int32_t token(int32_t m, int group) const { return begin + m / group - first; }
  __device__ __forceinline__ int32_t slots_of(int32_t token, int32_t cap) const {
    return (int32_t)min(max((int64_t)before + token + 1, (int64_t)0), (int64_t)cap);
  }
  // Slots that query m sees; 0: a row without a token, or a token without slots.
  __device__ __forceinline__ int32_t seen(int32_t m, int group, int32_t cap) const {
    if (m >= queries) return 0;
    const int32_t i = token(m, group);
    return (uint32_t)i < (uint32_t)count ? slots_of(i, cap) : 0;
  }
  // Slots that any of queries m .. to - 1 sees.
  __device__ __forceinline__ int32_t most_seen(int32_t m, int32_t to, int group, int32_t cap) const {
    const int32_t from = max(token(m, group), 0), last = min(token(to - 1, group), count - 1);
    return m < to && from <= last ? slots_of(last, cap) : 0;
  }
};

// The few kernel's tiles take the rows behind a sequence's, up to the next one's, along.  Sequence b's begin at
// number first_row * group / kFew + b: ascending, and at least as far apart as the tiles of the rows
// between.  The whole wave looks at 64 sequences at a time.
__device__ __forceinline__ ChunkTile few_tile(const ChunkParams& p, uint32_t tile, int lane) {
  auto number = [&](int b) { return (int64_t)p.starts[b] * p.group / kFew + b; };
  int lo = 0, n = p.B;
  while (n > 1) {
    const int step = (n + 63) >> 6, b = lo + lane * step;
    const bool upto = lane == 0 || (b < lo + n && number(b) <= tile);
    const int at = (__popcll(__ballot(upto)) - 1) * step;
    lo += at;
    n = min(step, n - at);
  }
  const int b = __builtin_amdgcn_readfirstlane(lo);
  ChunkTile t;
  t.b = b;
  t.first = p.starts[b];
  t.count = max(p.counts[b], 0);
  t.before = (int32_t)max((int64_t)p.lengths[b] - t.count, (int64_t)INT32_MIN);
  t.begin = b == 0 ? 0 : min(max(t.first, 0), p.rows);
  const int32_t end = b + 1 < p.B ? min(max(p.starts[b + 1], t.begin), p.rows) : p.rows;
  t.queries = (end - t.begin) * p.group;  // (rows * nq fits 31 bits)
  const int64_t at = b == 0 ? tile : tile - number(b);
  t.m0 = at < 0 || at * kFew >= t.queries ? t.queries : (int32_t)at * kFew;
  return t;
}

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
// Both bf16 of a word, Inf and NaN as 0.
__device__ __forceinline__ uint32_t without_special(uint32_t x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0xffffu;
  return x;
}

// NC: pieces of 32 dims in a head; DPL: columns of V that a lane holds (16 DPL >= D); FULL: D == 32 NC ==
// 16 DPL, so that every lane holds dims of the head.
template <int NC, int DPL, bool FULL>
__global__ __launch_bounds__(64 * kPagedWaves, NC == 4 && !FULL ? 2 : 4) void paged_chunk_few_kernel(
    const ChunkParams p) {
  typedef typename Piece<DPL>::type vpiece_t;
  constexpr int W = kPagedWaves, PITCH = 16 * DPL + 4;
  __shared__ float lds_o[W][kFew][PITCH];
  __shared__ float lds_m[W][kFew], lds_l[W][kFew];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // Splits run fastest, so that the blocks of one tile and head lie together.
  const uint32_t split = blockIdx.x % p.splits;
  const uint32_t rest = blockIdx.x / p.splits;
  const int h = rest % p.nkv;
  const ChunkTile ct = few_tile(p, rest / p.nkv, lane);
  if (!ct.any()) return;
  const int queries = min(kFew, ct.queries - ct.m0);
  const int32_t cap = p.t.capacity();
  // Column n is query m0 + n.  It sees `seen` slots, the block's queries min_seen to max_seen (those that see any).
  const int32_t seen = ct.seen(ct.m0 + n, p.group, cap);
  int32_t max_seen = seen, min_seen = seen > 0 ? seen : INT32_MAX;
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) {
    max_seen = max(max_seen, __shfl_xor(max_seen, d, 64));
    min_seen = min(min_seen, __shfl_xor(min_seen, d, 64));
  }
  max_seen = __builtin_amdgcn_readfirstlane(max_seen);
  min_seen = __builtin_amdgcn_readfirstlane(min_seen);
  const int32_t tiles = (max_seen + kPagedTile - 1) / kPagedTile;
  const int32_t per = (tiles + p.splits - 1) / p.splits;
  const int32_t t_end = min(tiles, (int32_t)(split + 1) * per);

  // Q^T: 8 dims per lane and piece; dims past the head and columns that see nothing are zero.
  auto query = [&](int i) {
    const int32_t m = ct.m0 + i;
    return (int64_t)(ct.begin + m / p.group) * p.nq + h * p.group + m % p.group;
  };
  bf16x8 qf[NC];
  const uint16_t* q_row = p.q + (seen > 0 ? query(n) : 0) * p.D;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    const int d = c * 32 + g * 8;
    if (seen > 0 && d < p.D) x = *reinterpret_cast<const uint4*>(q_row + d);
    qf[c] = __builtin_bit_cast(bf16x8, x);
  }

  f32x4 acc[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const int32_t* table = p.t.table + (int64_t)ct.b * p.t.ld;
  const int lps = p.t.log2_page;
  // A tile's rows lie at a base that the wave shares; a lane's offsets from it stay.
  const int D = FULL ? 32 * NC : p.D;
  const uint32_t k_at = n * D + g * 8, v_at = 4 * g * D + n * DPL;
  const bool v_on = FULL || n * DPL < D;
  int32_t wild = INT32_MAX;  // the first tile whose infinite values and NaN were left out

  for (int32_t tile = (int32_t)split * per + wave; tile < t_end; tile += W) {
    const int32_t s0 = tile * kPagedTile;
    // The two halves of 16 slots each lie inside one page.
    const uint16_t *k_base[2], *v_base[2];
    bool there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t at = s0 + 16 * i;
      const int32_t pg = at < max_seen ? table[at >> lps] : -1;
      there[i] = (uint32_t)pg < (uint32_t)p.t.num_pages;
      const int64_t row0 = (((int64_t)(there[i] ? pg : 0) * p.nkv + h) << lps) + (at & ((1 << lps) - 1));
      k_base[i] = p.k_pages + row0 * D;
      v_base[i] = p.v_pages + row0 * D;
    }
    bf16x8 kf[2][NC];
    vpiece_t vr[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (FULL || c * 32 + g * 8 < D) x = *reinterpret_cast<const uint4*>(k_base[i] + k_at + c * 32);
        kf[i][c] = __builtin_bit_cast(bf16x8, x);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        vpiece_t x{};
        if (v_on) x = *reinterpret_cast<const vpiece_t*>(v_base[i] + v_at + r * D);
        vr[4 * i + r] = x;
      }
    }
    float s[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][c], qf[c], a, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * i + r] = a[r] * p.scale_log2;
    }
    uint32_t* vw = reinterpret_cast<uint32_t*>(vr);  // [8 rows][DPL / 2]
    constexpr int RW = DPL / 2;
    if (s0 + kPagedTile > min_seen || !there[0] || !there[1]) {
      // Slots past what a query sees weigh nothing, and values that no query sees must not count
      // either (0 * NaN is NaN); a page that is not in the pool makes a query that sees it NaN.
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int32_t slot = s0 + 16 * (i / 4) + 4 * g + i % 4;
        const bool ok = there[i / 4];
        s[i] = slot >= seen ? -INFINITY : (ok ? s[i] : __builtin_nanf(""));
        if (slot >= max_seen || !ok) vr[i] = vpiece_t{};
      }
      // Infinite values and NaN that some queries may see and others not are added at the end.
      u16x2_t top = {0, 0};
#pragma unroll
      for (int w = 0; w < 8 * RW; ++w) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, vw[w] & 0x7fff7fffu));
      if (__builtin_amdgcn_ballot_w64(max(top[0], top[1]) >= 0x7f80) != 0) {
        wild = min(wild, tile);
#pragma unroll
        for (int w = 0; w < 8 * RW; ++w) vw[w] = without_special(vw[w]);
      }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
    const float m_new = fmaxf(m, max_over_groups(mx));
    const float m_ref = m_new == -INFINITY ? 0.f : m_new;  // scores of -inf weigh nothing, also the first ones
    const float alpha = __builtin_amdgcn_exp2f(m - m_ref);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int j = 0; j < DPL; ++j) acc[j] *= alpha;
    float pf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pf[i] = __builtin_amdgcn_exp2f(s[i] - m_ref);
      l += pf[i];
    }
    // P in two bf16 parts, to 2^-16 of it.
    const uint4 p_hi = pack8(pf);
    float hi[8];
    unpack8(p_hi, hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) pf[i] -= hi[i];
    const bf16x8 pb = __builtin_bit_cast(bf16x8, p_hi), pb_low = __builtin_bit_cast(bf16x8, pack8(pf));
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      uint4 a;
      const int w = j / 2;
      if (j & 1) {
        a.x = high_halves(vw[0 * RW + w], vw[1 * RW + w]);
        a.y = high_halves(vw[2 * RW + w], vw[3 * RW + w]);
        a.z = high_halves(vw[4 * RW + w], vw[5 * RW + w]);
        a.w = high_halves(vw[6 * RW + w], vw[7 * RW + w]);
      } else {
        a.x = low_halves(vw[0 * RW + w], vw[1 * RW + w]);
        a.y = low_halves(vw[2 * RW + w], vw[3 * RW + w]);
        a.z = low_halves(vw[4 * RW + w], vw[5 * RW + w]);
        a.w = low_halves(vw[6 * RW + w], vw[7 * RW + w]);
      }
      acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), pb, acc[j], 0, 0, 0);
      // The low part is 0 or negative where the high part is exact or rounded up, and 0 Inf has no
      // value: an infinite value counts once, by the high part, and is a finite one here.
      a = make_uint4(finite_halves(a.x), finite_halves(a.y), finite_halves(a.z), finite_halves(a.w));
      acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), pb_low, acc[j], 0, 0, 0);
    }
  }

  // An infinite value or NaN makes the column so of each query that sees it, whatever its weight: added as
  // it is (twice is once where a product has added it already).
  for (int32_t tile = wild; tile < t_end; tile += W) {
#pragma unroll 1
    for (int32_t slot = tile * kPagedTile; slot < min(tile * kPagedTile + kPagedTile, max_seen); ++slot) {
      const int64_t row = p.t.row(ct.b, h, p.nkv, slot);
      if (row < 0 || slot >= seen) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < DPL; ++j) {
          const int d = (4 * g + r) * DPL + j;
          const uint32_t x = d < D ? p.v_pages[row * D + d] : 0u;
          if ((x & 0x7f80u) == 0x7f80u) acc[j][r] += bf16_bits_to_f32(x);
        }
    }
  }

  // Join the waves: lane (n, g) holds query n, columns (4 g + r) DPL + j.
  l = sum_over_groups(l);
  if (g == 0) {
    lds_m[wave][n] = m;
    lds_l[wave][n] = l;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < DPL; ++j) lds_o[wave][n][(4 * g + r) * DPL + j] = acc[j][r];
  __syncthreads();
  for (int i = threadIdx.x; i < queries * (p.D / 4); i += 64 * W) {
    const int c = i / (p.D / 4), d = (i - c * (p.D / 4)) * 4;
    float M = lds_m[0][c];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, lds_m[w][c]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(lds_m[w][c] - ref);
      L = __builtin_fmaf(f, lds_l[w][c], L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(f, lds_o[w][c][d + e], o[e]);
    }
    const int64_t row = query(c);
    const bool sees = ct.seen(ct.m0 + c, p.group, cap) > 0;
    if (p.splits > 1) {
      const int64_t at = (int64_t)split * p.rows * p.nq + row;
      if (d == 0) p.part_ml[at] = make_float2(M, sees ? L : -1.f);
      *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = make_float4(o[0], o[1], o[2], o[3]);
    } else {
      // No keys at all: zeros.  Keys whose scores are all -inf: 0 / 0, as softmax has it.
      // (No product with 0: the sums of a column that sees nothing may hold infinite values.)
      const float inv = 1.f / L;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = sees ? o[e] * inv : 0.f;
      head_store4(p.out + row * p.D + d, o);
    }
  }
}

// ---- many queries ---------------------------------------------------------------

constexpr int kKeys = 64;     // slots of a tile
constexpr float kLazy = 8.f;  // log2-domain headroom before the running maximum is moved

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

// Both values of x held by lanes l and l ^ 32.
__device__ __forceinline__ float max_of_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// f(0) .. f(N - 1) with the numbers as constants.
template <typename F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

constexpr int kTileM = 128;  // queries of a tile

// The tile kernel's tile of this number: what takes longest comes first, so that the blocks that are left at the
// end are short ones (16 sequences of 1 .. 777 over up to 4099: 120 us by sequence, 82 so; 8 of 1024 over 2048:
// 118 by sequence, the longest first, 113 so).  Of 64 sequences each, by the keys that a tile's last query
// sees, in steps of 64; a sequence of fewer queries than a tile counts by the waves that they occupy (a
// key costs one wave about half of what it costs four, the fetch being the same).  How many tiles there
// are of so many keys or more is known for each sequence, so that the step of a number is found bit by
// bit, and the tile among those of the step.  By a whole wave; without queries if there are fewer tiles.
__device__ __forceinline__ ChunkTile chunk_tile(const ChunkParams& p, uint32_t number, int lane) {
  ChunkTile t{};
  int32_t at = (int32_t)number;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int n_seq = min(64, p.B - b0);
    const int b = b0 + min(lane, n_seq - 1);
    const int32_t first = p.starts[b], asked = max(p.counts[b], 0), length = p.lengths[b];
    // (Rows outside the call's are dropped.)
    const int32_t count = lane >= n_seq || first < 0 ? 0 : min(asked, max(p.rows - first, 0));
    const int32_t queries = count * p.group, tiles = (queries + kTileM - 1) / kTileM;
    const int32_t all = wave_sum(tiles);
    if (at >= all) {
      at -= all;
      continue;
    }
    const int32_t before = min(max(length - asked, 0), p.t.capacity());
    // Steps of a sequence of one tile, and the most that a tile has (also a last one that is partly empty, as
    // ``from`` counts it): tile j sees before + (j + 1) kTileM / group keys.
    const int32_t steps = (int32_t)(((int64_t)before + count) / kKeys + 1);
    const int32_t only = steps * (2 + (min(queries, kTileM) + 31) / 32) / 6;
    const int32_t top = tiles <= 1 ? only : (int32_t)((before + (int64_t)tiles * kTileM / p.group) / kKeys);
    // Tiles of x steps or more.
    auto from = [&](int32_t x) {
      if (tiles <= 1) return only >= x ? tiles : 0;
      const int64_t j = (((int64_t)kKeys * x - before) * p.group + kTileM - 1) / kTileM - 1;
      return tiles - (int32_t)min(max(j, (int64_t)0), (int64_t)tiles);
    };
    int32_t above = 0, here = tiles;
    if (n_seq > 1) {  // (one sequence's tiles go from the last to the first)
      int32_t x = 0, most = max(top, 1);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) most = max(most, __shfl_xor(most, d, 64));
      for (int bit = 31 - __builtin_clz(__builtin_amdgcn_readfirstlane(most)); bit >= 0; --bit)
        if (wave_sum(from(x | 1 << bit)) > at) x |= 1 << bit;
      above = from(x + 1), here = from(x) - above;
      at -= wave_sum(above);
    }
    const int32_t upto = wave_inclusive(here);
    const int i = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > at));
    t.b = b0 + i;
    t.begin = t.first = read_lane(first, i);
    t.count = read_lane(count, i);
    t.before = (int32_t)max((int64_t)read_lane(length, i) - read_lane(asked, i), (int64_t)INT32_MIN);
    t.queries = t.count * p.group;
    t.m0 = (read_lane(tiles - above + upto - here, i) - 1 - at) * kTileM;
    return t;
  }
  return t;
}

// HD: dims of a row in LDS; NKD: steps of 16 dims (16 NKD >= D); GEN: D < HD, and the dims past D are zeros.
template <int HD, int NKD, bool GEN>
__global__ __launch_bounds__(256, 2) void paged_chunk_tile_kernel(const ChunkParams p) {
  constexpr int ROWB = HD * 2;            // bytes of a K or V row
  constexpr int CPR = HD / 8;             // 16-byte chunks of it
  constexpr int RPL = 256 / ROWB;         // rows in 256 bytes: all banks once
  constexpr int TILE = kKeys * ROWB;      // bytes of a K or V tile
  constexpr int NDB = (NKD + 1) / 2;      // blocks of 32 dims of O^T
  constexpr int DMAS = TILE / 1024 / 4;   // DMA instructions of a wave for a tile: 16 rows
  constexpr int DMA_ROWS = 1024 / ROWB;
  static_assert(HD == 32 || HD == 64 || HD == 128, "rows of 64, 128 or 256 bytes");
  static_assert(DMAS * DMA_ROWS == 16, "a wave fetches 16 rows, which lie in one page");
  const int D = GEN ? p.D : HD;
  // Two K tiles, two V tiles, each an object of its own: the compiler waits for DMAs into what a transposing
  // read may alias.
  __shared__ __attribute__((aligned(1024))) uint8_t lds_k0[TILE], lds_k1[TILE], lds_v0[TILE], lds_v1[TILE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hi = lane >> 5, r32 = lane & 31;
  // KV heads run fastest: with eight of them each XCD reads the cache of one.  Splits run slowest: the later ones
  // of short tiles have nothing to do, and blocks go to XCDs and CUs in turn, so that every second one
  // with nothing leaves half of the chip idle (16 sequences of up to 4099, heads of 80, two splits: 145
  // us so, 113 with the second ones behind the first).
  const int h = blockIdx.x % p.nkv;
  const uint32_t rest = blockIdx.x / p.nkv, number = rest % p.tiles;
  const int split = rest / p.tiles;
  if (split == 0) {
    // Rows that belong to no sequence are zeros: those behind each one's up to the next one's.
    auto zero = [&](int32_t from, int32_t to) {
      for (int64_t r = (int64_t)from + number; r < to; r += p.tiles)
        for (int c = lane; c < p.group * D / 8; c += 64)
          reinterpret_cast<uint4*>(p.out + (r * p.nq + h * p.group) * D)[c] = make_uint4(0u, 0u, 0u, 0u);
    };
    for (int b0 = wave * 64; b0 < p.B; b0 += 256) {
      const int b = b0 + lane;
      int32_t from = 0, to = 0;
      if (b < p.B) {
        from = (int32_t)min(max((int64_t)p.starts[b] + max(p.counts[b], 0), (int64_t)0), (int64_t)p.rows);
        to = b + 1 < p.B ? min(p.starts[b + 1], p.rows) : p.rows;
      }
      for (uint64_t left = __builtin_amdgcn_ballot_w64(from < to); left != 0; left &= left - 1) {
        const int i = __builtin_ctzll(left);
        zero(read_lane(from, i), read_lane(to, i));
      }
    }
    if (wave == 0) zero(0, min(p.starts[0], p.rows));  // (and those ahead of the first)
  }
  const ChunkTile ct = chunk_tile(p, number, lane);
  if (!ct.any()) return;
  const int32_t cap = p.t.capacity(), group = p.group, b = ct.b;
  const int32_t m0 = ct.m0, end_m = min(ct.queries, m0 + kTileM);  // past the tile's last query
  auto row_of = [&](int32_t m) { return (int64_t)(ct.begin + m / group) * p.nq + h * group + m % group; };
  // What the block's, and the wave's, queries see at most; of these, tiles t0 .. t0 + nt - 1 of keys are at hand.
  const int32_t block_seen = __builtin_amdgcn_readfirstlane(ct.most_seen(m0, end_m, group, cap));
  const int32_t all_tiles = (block_seen + kKeys - 1) / kKeys;
  const int32_t t0 = split * p.piece, nt = min(all_tiles - t0, p.piece);
  if (nt <= 0 && split > 0) return;
  const bool whole = all_tiles <= p.piece;
  const int32_t mw = m0 + wave * 32;
  const int32_t wave_seen = __builtin_amdgcn_readfirstlane(ct.most_seen(mw, min(end_m, mw + 32), group, cap));
  // Tiles of this wave, and the first one that some of its queries do not see whole.
  const int32_t ntw = max(min((wave_seen + kKeys - 1) / kKeys - t0, nt), 0);
  const int32_t full = __builtin_amdgcn_readfirstlane(ct.slots_of(max(ct.token(mw, group), 0), cap)) / kKeys - t0;
  const int32_t m = mw + r32;
  const int32_t seen = m < end_m ? ct.seen(m, group, cap) : 0;

  f32x16 o[NDB];
  float m_run = -INFINITY, m_ref = 0.f, l_run = 0.f, mx = -INFINITY;
  int32_t wild = INT32_MAX;  // the first tile whose infinite values and NaN were left out
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[db][v] = 0.f;

  if (nt > 0) {
    // Q fragments: the B operand, query r32 of the wave's, dims 16 k + 8 hi .. + 8.
    bf16x8 qf[NKD];
    const uint16_t* q_row = p.q + (seen > 0 ? row_of(m) * D : 0) + 8 * hi;
#pragma unroll
    for (int k = 0; k < NKD; ++k) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (seen > 0 && (!GEN || 16 * k + 8 * hi < D)) x = *reinterpret_cast<const uint4*>(q_row + 16 * k);
      qf[k] = __builtin_bit_cast(bf16x8, x);
    }

    // ---- pages -------------------------------------------------------------------
    // Lane i knows the page of this wave's 16 rows of tile window + i; a page's number is read off
    // when its tile is fetched.  missing: bit i for a tile with a page that is not in the pool.
    const int32_t* table = p.t.table + (int64_t)b * p.t.ld;
    const int lp = p.t.log2_page;
    int32_t page_ids = 0, window = t0;
    uint64_t missing = 0;
    auto look_up = [&]() __attribute__((always_inline)) {
      bool bad = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int64_t s = (int64_t)(window + lane) * kKeys + 16 * w;
        const int32_t pg = s < block_seen ? table[s >> lp] : 0;
        bad = bad || (uint32_t)pg >= (uint32_t)p.t.num_pages;
        if (w == wave) page_ids = (uint32_t)pg < (uint32_t)p.t.num_pages ? pg : -1;
      }
      missing = __builtin_amdgcn_ballot_w64(bad);
    };
    // K chunk c of tile row r lies at position c ^ (r / RPL % CPR): reads of one chunk of 32 rows spread over
    // the banks.  V chunk c at c ^ (4 (r / RPL % 4)): four rows' equal 64 bytes, which a transposing read
    // takes together, lie in different quarters of them.
    constexpr uint32_t kOutside = 0x80000000u;
    uint32_t k_off[DMAS], v_off[DMAS];
#pragma unroll
    for (int j = 0; j < DMAS; ++j) {
      const int r = wave * 16 + j * DMA_ROWS + lane / CPR, row = j * DMA_ROWS + lane / CPR;
      const int ck = (lane % CPR) ^ ((r / RPL) % CPR), cv = (lane % CPR) ^ (CPR > 4 ? 4 * (r / RPL % (CPR / 4)) : 0);
      k_off[j] = GEN && ck * 8 >= D ? kOutside : (uint32_t)(row * D + ck * 8) * 2;
      v_off[j] = GEN && cv * 8 >= D ? kOutside : (uint32_t)(row * D + cv * 8) * 2;
    }
    // Rows past what the block sees are read as zeros: they may hold anything, and 0 * NaN is NaN.
    auto fetch = [&](const uint16_t* pages, int32_t t, int32_t pg, const uint32_t(&off)[DMAS],
                     uint8_t* dst) __attribute__((always_inline)) {
      const int32_t s = (t0 + t) * kKeys + wave * 16;
      const int64_t row = (((int64_t)max(pg, 0) * p.nkv + h) << lp) + (s & ((1 << lp) - 1));
      const int32_t rows = pg < 0 ? 0 : min(max(block_seen - s, 0), 16);
      // (The whole wave's: said so, as a descriptor that the compiler takes for a lane's costs a loop over lanes.)
      const uint64_t base = (uint64_t)(pages + row * D);
      const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)base), up = __builtin_amdgcn_readfirstlane(base >> 32);
      const uint32_t bytes = __builtin_amdgcn_readfirstlane(rows * D * 2);
      const __amdgpu_buffer_rsrc_t rs = make_rsrc((const void*)((uint64_t)up << 32 | lo), bytes);
#pragma unroll
      for (int j = 0; j < DMAS; ++j) buf_dma16(rs, off[j], 0u, dst + (wave * DMAS + j) * 1024);
    };
    int32_t pg_ahead = -1;  // of the tile after the next one
    bool bad_next = false, bad_ahead = false;
    auto advance = [&](int32_t t) __attribute__((always_inline)) {  // to tile t
      if (t0 + t >= window + 64) {
        window = t0 + t;
        look_up();
      }
      const int i = t0 + t - window;
      pg_ahead = __builtin_amdgcn_readlane(page_ids, i);
      bad_next = bad_ahead;
      bad_ahead = (missing >> i & 1) != 0;
    };

    // ---- fragments -----------------------------------------------------------------
    int kf_off[NKD];
#pragma unroll
    for (int k = 0; k < NKD; ++k) kf_off[k] = r32 * ROWB + (((2 * k + hi) ^ ((r32 / RPL) % CPR)) << 4);
    // V^T: a group of 16 lanes reads 4 keys x 16 dims and receives them transposed; lane: key
    // 4 hi + (lane % 16) / 4, 4 dims from 16 (lane / 16 % 2) + 4 (lane % 4) on.
    const int v_key = 4 * hi + (lane & 15) / 4;
    int vf_off[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const int c = 4 * db + 2 * (lane >> 4 & 1) + (lane & 3) / 2;
      vf_off[db] = v_key * ROWB + ((c ^ (CPR > 4 ? 4 * (v_key / RPL % (CPR / 4)) : 0)) << 4) + (lane & 1) * 8;
    }
    // Every product takes one operand from LDS, K's rows or V^T's: they are read RING - 1 products ahead.
    constexpr int RING = 5;
    bf16x8 fr[RING], pf[4];
    f32x16 s[2][2];  // S^T of two tiles: the one in the softmax and the next one
    auto k_read = [&](int slot, int buf, int i) __attribute__((always_inline)) {
      fr[slot] = *reinterpret_cast<const bf16x8*>((buf ? lds_k1 : lds_k0) + kf_off[i % NKD] + (i / NKD) * 32 * ROWB);
    };
    auto qk = [&](int slot, int set, int i) __attribute__((always_inline)) {
      const int kb = i / NKD, k = i % NKD;
      s[set][kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[slot], qf[k], k == 0 ? f32x16{} : s[set][kb], 0, 0, 0);
    };
    auto v_read = [&](int slot, int buf, int i) __attribute__((always_inline)) {
      const int sl = i / NDB, db = i % NDB;
      const uint8_t* at = (buf ? lds_v1 : lds_v0) + vf_off[db] + sl * 16 * ROWB;
      typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
      const s16x4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 8 * ROWB));
      fr[slot] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto pv = [&](int slot, int i) __attribute__((always_inline)) {
      const int sl = i / NDB, db = i % NDB;
      o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[slot], pf[sl], o[db], 0, 0, 0);
    };

    // ---- softmax -------------------------------------------------------------------
    // Score v of key block kb in a lane is key 32 kb + 8 (v / 4) + 4 hi + v % 4 of query r32.
    // What tile t's queries see of it, and their maxima in log2 units.
    auto row_max = [&](int set, int32_t t, bool bad) __attribute__((always_inline)) {
      if (__builtin_expect(bad, 0)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int32_t key = (t0 + t) * kKeys + 16 * w;
          if (key < block_seen && (uint32_t)table[key >> lp] >= (uint32_t)p.t.num_pages)
#pragma unroll
            for (int v = 8 * (w & 1); v < 8 * (w & 1) + 8; ++v) s[set][w >> 1][v] = __builtin_nanf("");
        }
      }
      if (t >= full || bad) {
        const int32_t lim = seen - (t0 + t) * kKeys - 4 * hi;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int key = kb * 32 + 8 * (v >> 2) + (v & 3);
            s[set][kb][v] = key >= lim ? -INFINITY : s[set][kb][v];
          }
      }
      float x[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        x[kb] = fmaxf(s[set][kb][0], s[set][kb][1]);
#pragma unroll
        for (int v = 2; v < 16; v += 2) x[kb] = fmaxf(fmaxf(x[kb], s[set][kb][v]), s[set][kb][v + 1]);
      }
      mx = max_of_halves(fmaxf(x[0], x[1])) * p.scale_log2;
    };
    // The reference m_run moves only when a query's maximum passes it by more than kLazy; until then
    // P = 2^(t - m_run) <= 2^kLazy, which bf16 and fp32 hold, and the division by l cancels it.
    auto move_max = [&]() __attribute__((always_inline)) {
      if (__builtin_amdgcn_ballot_w64(mx > m_run + kLazy) != 0) {
        const float m_new = fmaxf(m_run, mx);
        m_ref = m_new == -INFINITY ? 0.f : m_new;  // scores of -inf weigh nothing, also the first ones
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
      }
    };
    // P of two neighbouring keys of slab sl, rounded to bf16 (the sum l is of the rounded ones, so that the
    // weights that V is multiplied by add up to 1), and its place among the slab's operand.  One bf16 part leaves
    // 2^-9 of a weight, and 0.0023 of the output against 64 bits where rounding the result alone leaves 0.0017; a
    // second part, as in the few kernel, would be half as many products again where products bound the call.
    auto p_pair = [&](int set, int u) __attribute__((always_inline)) {
      const int sl = u / 4, j = u % 4, kb = sl >> 1, v = 8 * (sl & 1) + 2 * j;
      const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[set][kb][v], p.scale_log2, -m_ref));
      const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[set][kb][v + 1], p.scale_log2, -m_ref));
      uint32_t w = pack_bf16x2(a, b);
      asm volatile("" : "+v"(w));  // here, between the products, and not where the operand is used
      l_run = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w),
                                                  __builtin_bit_cast(bf16x2_t, 0x3F803F80u), l_run, false);
      reinterpret_cast<uint32_t*>(&pf[sl])[j] = w;
    };
    // Infinite values and NaN in a tile that some queries do not see whole (0 of P times them has no
    // value) leave V^T, operand by operand, and are added at the end.
    auto tame = [&](int slot) __attribute__((always_inline)) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&fr[slot]);
      u16x2_t top = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
      if (__builtin_amdgcn_ballot_w64(max(top[0], top[1]) >= 0x7f80) == 0) return false;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = without_special(w[i]);
      return true;
    };

    // ---- pipeline --------------------------------------------------------------------
    // Tile t's softmax and O += V(t)^T P(t), with the QK products of tile t + 1 between.  Its DMAs, issued
    // behind its barrier, fetch K(t + 2) into the buffer of K(t) and V(t + 1) into that of V(t - 1); both
    // land before the next barrier.
    auto sync = [&](int32_t t, int cur) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
      __syncthreads();
      const int32_t pg_next = pg_ahead;
      if (t + 2 < nt) {
        advance(t + 2);
        fetch(p.k_pages, t + 2, pg_ahead, k_off, cur ? lds_k1 : lds_k0);
      } else {
        bad_next = bad_ahead;
      }
      if (t + 1 < nt) fetch(p.v_pages, t + 1, pg_next, v_off, cur ? lds_v0 : lds_v1);
    };
    auto body = [&](int32_t t, auto par, auto more) __attribute__((always_inline)) {
      constexpr int cur = decltype(par)::value, nxt = cur ^ 1;
      constexpr bool next = decltype(more)::value;
      constexpr int QK = next ? 2 * NKD : 0, PV = NDB, PAIRS = 16;
      constexpr int SPAN = QK + 3 * PV;  // products before the last slab's
      const bool masked = t >= full || bad_next;  // (bad_next: of tile t until sync has gone on)
      sync(t, cur);
      constexpr int ALL = QK + 4 * PV;
      auto read = [&](auto index) __attribute__((always_inline)) {
        constexpr int i = decltype(index)::value;
        if constexpr (i < QK)
          k_read(i % RING, nxt, i);
        else if constexpr (i < ALL)
          v_read(i % RING, cur, i - QK);
      };
      each<RING - 1>(read);
      move_max();
      // Of the two waves of a SIMD the one among its products goes on with them (2048 tokens over 65536, heads of
      // 128: 1015 -> 990 us, 4 x 512 over 4096 of 64: 51 -> 47; where the head is padded, heads of 80, 81 -> 84).
      if constexpr (!GEN) __builtin_amdgcn_s_setprio(1);
      each<ALL>([&](auto index) __attribute__((always_inline)) {
        constexpr int i = decltype(index)::value;
        // The pairs of P are spread over the products before the last slab's, each slab's before its own.
        each<PAIRS>([&](auto pair) __attribute__((always_inline)) {
          constexpr int u = decltype(pair)::value, before = QK + u / 4 * PV, even = u * SPAN / PAIRS;
          if constexpr ((even < before ? even : before) == i) p_pair(cur, u);
        });
        read(std::integral_constant<int, i + RING - 1>{});
        if constexpr (i < QK) {
          qk(i % RING, nxt, i);
        } else {
          if (__builtin_expect(masked, 0) && tame(i % RING)) wild = min(wild, t);
          pv(i % RING, i - QK);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (!GEN) __builtin_amdgcn_s_setprio(0);
      if constexpr (next) row_max(nxt, t + 1, bad_next);
    };

    look_up();
    advance(0);
    fetch(p.k_pages, 0, pg_ahead, k_off, lds_k0);
    fetch(p.v_pages, 0, pg_ahead, v_off, lds_v0);
    if (nt > 1) {
      advance(1);
      fetch(p.k_pages, 1, pg_ahead, k_off, lds_k1);
    } else {
      bad_next = bad_ahead;
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 15));
    __syncthreads();
    if (ntw > 0) {
      each<2 * NKD + RING - 1>([&](auto index) __attribute__((always_inline)) {
        constexpr int i = decltype(index)::value - (RING - 1);
        if constexpr (i >= 0) qk(i % RING, 0, i);
        if constexpr (i + RING - 1 < 2 * NKD) k_read((i + RING - 1) % RING, 0, i + RING - 1);
      });
      row_max(0, 0, bad_next);
    }
    // Every wave passes sync(t) once for each t < nt, in order, so the barriers pair up.
    int32_t t = 0;
    for (; t + 2 < ntw; t += 2) {
      body(t, std::integral_constant<int, 0>{}, std::true_type{});
      body(t + 1, std::integral_constant<int, 1>{}, std::true_type{});
    }
    if (t + 1 < ntw) {
      body(t, std::integral_constant<int, 0>{}, std::true_type{});
      ++t;
    }
    if (t < ntw) {
      if (t & 1)
        body(t, std::integral_constant<int, 1>{}, std::false_type{});
      else
        body(t, std::integral_constant<int, 0>{}, std::false_type{});
      ++t;
    }
    for (; t < nt; ++t) {
      if (t & 1)
        sync(t, 1);
      else
        sync(t, 0);
    }
  }

  // As in the few kernel: added as they are, whatever their weights.
  for (int32_t slot = wild < ntw ? (t0 + wild) * kKeys : INT32_MAX; slot < min((t0 + ntw) * kKeys, wave_seen); ++slot) {
    const int64_t row = p.t.row(b, h, p.nkv, slot);
    if (row < 0) continue;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int d = 32 * db + 8 * (v >> 2) + 4 * hi + (v & 3);
        const uint32_t x = !GEN || d < D ? p.v_pages[row * D + d] : 0u;
        if (slot < seen && (x & 0x7f80u) == 0x7f80u) o[db][v] += bf16_bits_to_f32(x);
      }
  }

  // ---- O^T / l ---------------------------------------------------------------------
  l_run = sum_of_halves(l_run);
  if (!whole) {
    if (m < end_m) {
      const int64_t at = (int64_t)split * p.rows * p.nq + row_of(m);
      if (hi == 0) p.part_ml[at] = make_float2(m_run, seen > 0 ? l_run : -1.f);
      if (ntw > 0) {  // (else a maximum of -inf: the sums are not read)
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int d = 32 * db + 8 * g + 4 * hi;
            if (!GEN || d < D)
              *reinterpret_cast<float4*>(p.part_o + at * D + d) =
                  make_float4(o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]);
          }
      }
    }
    return;
  }
  // A lane holds 8-byte pieces of one query: they are staged through LDS, 16-byte chunk c of row r at position
  // c ^ (r % CPR), and go out as whole rows.
  static_assert(2 * 32 * ROWB == TILE, "a block of 32 queries of two waves fills a K tile");
  __syncthreads();
  uint8_t* stage = (wave & 2 ? lds_k1 : lds_k0) + (wave & 1) * 32 * ROWB;
  const float inv = 1.f / l_run;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 w = make_uint2(pack_bf16x2(o[db][4 * g] * inv, o[db][4 * g + 1] * inv),
                           pack_bf16x2(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv));
      if (seen <= 0) w = make_uint2(0u, 0u);
      const int ch = (db * 4 + g) ^ (r32 % CPR);
      *reinterpret_cast<uint2*>(stage + r32 * ROWB + ch * 16 + hi * 8) = w;
    }
  // The wave's own LDS writes complete before its reads (and stay ahead of them).
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
  __builtin_amdgcn_wave_barrier();
  const int jc = lane % CPR;
#pragma unroll
  for (int i = 0; i < CPR / 2; ++i) {
    const int r = i * (64 / CPR) + lane / CPR;
    const uint4 x = *reinterpret_cast<const uint4*>(stage + r * ROWB + ((jc ^ (r % CPR)) << 4));
    if (mw + r < end_m && (!GEN || jc * 8 < D)) *reinterpret_cast<uint4*>(p.out + row_of(mw + r) * D + jc * 8) = x;
  }
}

constexpr int kJoinThreads = 256;

// The sums of tiles that several splits took, by tile and KV head; the others are done.
// parts: blocks that a tile's queries are joined by.
__global__ __launch_bounds__(kJoinThreads) void paged_chunk_join_kernel(const ChunkParams p, int parts) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int part = blockIdx.x % parts, rest = blockIdx.x / parts, h = rest % p.nkv;
  const ChunkTile ct = chunk_tile(p, rest / p.nkv, lane);
  if (!ct.any()) return;
  const int32_t end_m = min(ct.queries, ct.m0 + kTileM);
  const int32_t seen = ct.most_seen(ct.m0, end_m, p.group, p.t.capacity());
  const int pieces = ((seen + kKeys - 1) / kKeys + p.piece - 1) / p.piece;
  if (pieces <= 1) return;
  const int cols = p.D / 4;
  const int64_t step = (int64_t)p.rows * p.nq;
  for (int i = part * kJoinThreads + tid; i < (end_m - ct.m0) * cols; i += parts * kJoinThreads) {
    const int32_t m = ct.m0 + i / cols, d = i % cols * 4;
    const int64_t row = (int64_t)(ct.begin + m / p.group) * p.nq + h * p.group + m % p.group;
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    bool sees = true;
#pragma unroll 4
    for (int k = 0; k < pieces; ++k) {
      const float2 ml = p.part_ml[k * step + row];
      // (Where the maximum is -inf no sum was written, or one of nothing.)
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      if (ml.x != -INFINITY) y = *reinterpret_cast<const float4*>(p.part_o + (k * step + row) * p.D + d);
      sees = ml.y != -1.f;
      const float top = fmaxf(M, ml.x), ref = top == -INFINITY ? 0.f : top;
      const float f = __builtin_amdgcn_exp2f(M - ref), g = __builtin_amdgcn_exp2f(ml.x - ref);
      M = top;
      L = __builtin_fmaf(L, f, g * ml.y);
      o.x = __builtin_fmaf(o.x, f, g * y.x), o.y = __builtin_fmaf(o.y, f, g * y.y);
      o.z = __builtin_fmaf(o.z, f, g * y.z), o.w = __builtin_fmaf(o.w, f, g * y.w);
    }
    const float inv = 1.f / L;
    const float y[4] = {sees ? o.x * inv : 0.f, sees ? o.y * inv : 0.f, sees ? o.z * inv : 0.f, sees ? o.w * inv : 0.f};
    head_store4(p.out + row * p.D + d, y);
  }
}

// One (row, head) a block: its splits' sums by 256 threads over splits and columns.
__global__ __launch_bounds__(kJoinThreads) void paged_chunk_few_join_kernel(const ChunkParams p) {
  __shared__ float4 part[kJoinThreads];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x, step = (int64_t)p.rows * p.nq;
  const int cols = p.D / 4, groups = min(kJoinThreads / cols, 16);
  const int sg = tid / cols, d = (tid - sg * cols) * 4;
  float2 ml[kPagedMaxSplits / 64];
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPagedMaxSplits / 64; ++i) {
    const int s = i * 64 + lane;
    ml[i] = s < p.splits ? p.part_ml[s * step + row] : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[i].x);
  }
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) M = fmaxf(M, __shfl_xor(M, w, 64));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
#pragma unroll
  for (int i = 0; i < kPagedMaxSplits / 64; ++i) L = __builtin_fmaf(__builtin_amdgcn_exp2f(ml[i].x - ref), ml[i].y, L);
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) L += __shfl_xor(L, w, 64);
  const bool sees = __builtin_bit_cast(uint32_t, __shfl(ml[0].y, 0, 64)) != __builtin_bit_cast(uint32_t, -1.f);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (sg < groups) {
#pragma unroll 4
    for (int s = sg; s < p.splits; s += groups) {
      const int64_t at = s * step + row;
      const float top = p.part_ml[at].x;
      if (top == -INFINITY) continue;  // (a sum of nothing)
      const float f = __builtin_amdgcn_exp2f(top - ref);
      const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * p.D + d);
      o.x = __builtin_fmaf(f, x.x, o.x), o.y = __builtin_fmaf(f, x.y, o.y);
      o.z = __builtin_fmaf(f, x.z, o.z), o.w = __builtin_fmaf(f, x.w, o.w);
    }
  }
  part[tid] = o;
  __syncthreads();
  if (tid >= cols) return;
  for (int g = 1; g < groups; ++g) {
    const float4 x = part[g * cols + tid];
    o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
  }
  const float inv = 1.f / L;
  const float f[4] = {sees ? o.x * inv : 0.f, sees ? o.y * inv : 0.f, sees ? o.z * inv : 0.f, sees ? o.w * inv : 0.f};
  head_store4(p.out + row * p.D + d, f);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

struct ChunkPlan {
  bool few;
  int64_t tiles;  // numbers that they may have
  int splits, piece;
  size_t o, ml;
  size_t total() const { return o + ml; }
};

// Splits of a tile's slots, for so many blocks of key_tiles tiles of keys: blocks come in turns of two a CU, and a
// turn takes as long as its tiles and a beginning and end, which is about three; a second kernel takes as long
// as three, and every block's sums, written and read at 5 TB/s, 0.02 (a tile of 128 queries and 64 keys:
// 1.3 us).  4 x 512 tokens over 4096 of 12/4 heads of 64: one split 55 us, two 51, three 56; 64 over 8192
// of 16/8 heads of 128: one split 137, two 77, four 45, eight 31; 2048 over 65536: one 1133, two 994, four 999.
// The host knows the table's width alone, and not the lengths: 256 tokens over 4096 slots take 31 us in a table
// of that width, 33 in one of 16384 and 76 in one of 65536 slots; 2048 over 8192 136, 149 and 148.
int tile_splits(int64_t blocks, int64_t key_tiles) {
  const int64_t slots = 2 * device_cu_count();
  int best = 1;
  double cost = 1e30;
  for (int64_t s = 1; s <= std::min<int64_t>(kPagedMaxSplits, key_tiles); ++s) {
    const int64_t turns = (blocks * s + slots - 1) / slots, piece = (key_tiles + s - 1) / s;
    const double c = (double)(turns * (piece + 3)) + (s > 1 ? 3.0 + 0.02 * (double)(blocks * s) : 0.0);
    if (c < cost) cost = c, best = (int)s;
    if (turns > 4) break;
  }
  return best;
}

ChunkPlan chunk_plan(int64_t rows, int64_t B, int64_t nq, int64_t nkv, int64_t hd, int64_t cap, int64_t most) {
  ChunkPlan c{};
  const int64_t group = nq / nkv;
  // Calls of so few queries: 1 x 8 tokens over 4096 slots 13.4 us, by the tile kernel 21.5; 32 x 4 over 1024 29, 41;
  // 64 x 1 over 2048 94, 113; 64 x 4 over 1000 of 8/4 heads of 40 13, 27; but 64 x 8 over 2048 120, 100, which a
  // rule by the queries alone does not tell from the others.
  c.few = std::min(most, rows) * group <= kFew;
  const int64_t size = c.few ? kFew : kTileM;
  c.tiles = rows * group / size + B;
  const int64_t key_tiles = (cap + kKeys - 1) / kKeys;
  c.splits = c.few ? paged_splits(c.tiles * nkv, cap)
                   : tile_splits(((rows * group + kTileM - 1) / kTileM + (B - 1) / 2) * nkv, key_tiles);
  c.piece = (int)((key_tiles + c.splits - 1) / c.splits);
  if (c.splits > 1) {
    c.o = round16((size_t)(c.splits * rows * nq * hd) * sizeof(float));
    c.ml = round16((size_t)(c.splits * rows * nq) * sizeof(float2));
  }
  return c;
}

void launch_few(const ChunkParams& p, const dim3& grid, hipStream_t s) {
  const dim3 block(64 * kPagedWaves);
  if (p.D <= 32)
    paged_chunk_few_kernel<1, 4, false><<<grid, block, 0, s>>>(p);
  else if (p.D < 64)
    paged_chunk_few_kernel<2, 4, false><<<grid, block, 0, s>>>(p);
  else if (p.D == 64)
    paged_chunk_few_kernel<2, 4, true><<<grid, block, 0, s>>>(p);
  else if (p.D <= 96)
    paged_chunk_few_kernel<3, 8, false><<<grid, block, 0, s>>>(p);
  else if (p.D < 128)
    paged_chunk_few_kernel<4, 8, false><<<grid, block, 0, s>>>(p);
  else
    paged_chunk_few_kernel<4, 8, true><<<grid, block, 0, s>>>(p);
}

void launch_tile(const ChunkParams& p, const dim3& grid, hipStream_t s) {
  const dim3 block(256);
  switch (p.D) {
    case 32: return paged_chunk_tile_kernel<32, 2, false><<<grid, block, 0, s>>>(p);
    case 64: return paged_chunk_tile_kernel<64, 4, false><<<grid, block, 0, s>>>(p);
    case 128: return paged_chunk_tile_kernel<128, 8, false><<<grid, block, 0, s>>>(p);
    default: break;
  }
  switch ((p.D + 15) / 16) {
    case 1:
    case 2: return paged_chunk_tile_kernel<64, 2, true><<<grid, block, 0, s>>>(p);
    case 3: return paged_chunk_tile_kernel<64, 3, true><<<grid, block, 0, s>>>(p);
    case 4: return paged_chunk_tile_kernel<64, 4, true><<<grid, block, 0, s>>>(p);
    case 5: return paged_chunk_tile_kernel<128, 5, true><<<grid, block, 0, s>>>(p);
    case 6: return paged_chunk_tile_kernel<128, 6, true><<<grid, block, 0, s>>>(p);
    case 7: return paged_chunk_tile_kernel<128, 7, true><<<grid, block, 0, s>>>(p);
    default: return paged_chunk_tile_kernel<128, 8, true><<<grid, block, 0, s>>>(p);
  }
}

}  // namespace
}  // namespace cdx

extern "C" size_t cdx_paged_chunk_attention_workspace_bytes(int64_t rows, int64_t B, int32_t nq, int32_t nkv,
                                                            int32_t hd, int64_t capacity, int64_t max_tokens) {
  using namespace cdx;
  if (rows <= 0 || B <= 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || hd <= 0 || capacity <= 0 || max_tokens < 0)
    return 0;
  return chunk_plan(rows, B, nq, nkv, hd, capacity, max_tokens).total();
}

extern "C" int cdx_paged_chunk_attention_fwd(const uint16_t* q, int64_t rows, int64_t B, int32_t nq, int32_t nkv,
                                             int32_t hd, const uint16_t* k_pages, const uint16_t* v_pages,
                                             const int32_t* table, int64_t table_ld, int64_t width, int64_t num_pages,
                                             int32_t page_size, const int32_t* starts, const int32_t* counts,
                                             const int32_t* lengths, int64_t max_tokens, float scale, uint16_t* out,
                                             void* work, size_t work_bytes, void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_chunk_attention_fwd";
  clear_error();
  ChunkParams p{};
  if (int rc = paged_table(name, table, table_ld, width, num_pages, page_size, B, nkv, hd, &p.t)) return rc;
  if (rows < 0 || nq <= 0 || nq % nkv != 0)
    return fail(CDX_EINVAL, "%s: bad shape rows=%lld nq=%d nkv=%d", name, (long long)rows, nq, nkv);
  if (max_tokens < 0) return fail(CDX_EINVAL, "%s: max_tokens=%lld must be >= 0", name, (long long)max_tokens);
  if (!(scale > 0.f) || scale > 3e38f) return fail(CDX_EINVAL, "%s: scale must be > 0 and finite", name);
  if (rows == 0) return CDX_OK;
  if (B == 0 || width == 0 || num_pages == 0) return fail(CDX_EINVAL, "%s: empty block table or pool", name);
  const int64_t cap = width * page_size, group = nq / nkv;
  if (rows > INT32_MAX / 1024 || nq > 65535 || rows * nq > INT32_MAX)
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  const ChunkPlan c = chunk_plan(rows, B, nq, nkv, hd, cap, max_tokens);
  const int64_t blocks = c.tiles * nkv * c.splits;
  if (blocks > max_blocks(64 * kPagedWaves) || rows * nq > max_blocks(kJoinThreads))
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (!q || !k_pages || !v_pages || !table || !starts || !counts || !lengths || !out)
    return fail(CDX_EINVAL, "%s: null pointer", name);
  if (work_bytes < c.total() || (c.total() > 0 && !work))
    return fail(CDX_EWORKSPACE, "%s: workspace needs %zu bytes, got %zu", name, c.total(), work ? work_bytes : 0);
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) || !aligned16(work))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  p.q = q;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.starts = starts;
  p.counts = counts;
  p.lengths = lengths;
  p.B = (int32_t)B;
  p.rows = (int32_t)rows;
  p.nq = nq;
  p.nkv = nkv;
  p.D = hd;
  p.group = (int32_t)group;
  p.scale_log2 = scale * kLog2e;
  p.out = out;
  p.splits = c.splits;
  p.piece = c.piece;
  p.tiles = (uint32_t)c.tiles;
  p.part_o = static_cast<float*>(work);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(work) + c.o);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), joiners(kJoinThreads);
  if (c.few)
    launch_few(p, grid, s);
  else
    launch_tile(p, grid, s);
  if (int rc = check_launch(name)) return rc;
  if (c.splits == 1) return CDX_OK;
  if (c.few)
    paged_chunk_few_join_kernel<<<dim3((unsigned)(rows * nq)), joiners, 0, s>>>(p);
  else {
    const int parts = (int)std::min<int64_t>(16, (4 * device_cu_count() + c.tiles * nkv - 1) / (c.tiles * nkv));
    paged_chunk_join_kernel<<<dim3((unsigned)(c.tiles * nkv * parts)), joiners, 0, s>>>(p, parts);
  }
  return check_launch(name);
}
