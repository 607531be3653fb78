// Attention of any number of new tokens per sequence over a paged KV cache, for gfx950.
//
//   o[r, h] = sum_t p_t v_t,  p = softmax_t(scale q[r, h] . k_t),  t <= t(r),
//
// t(r) = length[b] - count[b] + i being the slot of row r, the i-th new token of sequence b: it attends to
// everything before it and to itself.  Sequences bring different numbers of rows, which only the
// device knows.  The (row, query head) pairs of one (sequence, KV head) are its queries, row by
// row, so that a tile of queries shares K and V over the heads of the group as well as over rows;
// tiles are numbered so that a block finds its sequence from the first rows alone (chunk_tile).
//
//   paged_chunk_few_kernel  16 queries a block: the cache's bytes bound it.  paged_attn_kernel's walk of the
//                           pages with the columns of the matrix instruction taken by queries of several rows.
#include <algorithm>
#include <type_traits>

#include "cdx_gemm.h"
#include "cdx_paged_attn.h"

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
  int32_t B, rows, nq, nkv, D, group, splits;
  int32_t few;       // sequences of so many queries are the few kernel's (0: none)
  bool by_sequence;  // the few kernel takes those sequences alone, a block each and head
  uint32_t tiles;    // numbers that a tile may have
  float scale_log2;
  uint16_t* out;    // [rows][nq][D]
  // Of each split, by (row, head), or by sequence [B][nkv][kFew]:
  int64_t part_rows;
  float* part_o;    // [splits][part_rows][D], unnormalised
  float2* part_ml;  // [splits][part_rows]: maximum (log2 units) and sum; a sum of -1: no key at all
};

constexpr int kFew = 16;  // queries of a block: the columns of a matrix instruction

// A tile of BM queries of one sequence.  Sequence b's own rows, with those that follow them up to the
// next one's, are rows begin .. end - 1 of the call; row r is token r - first of the sequence.
struct ChunkTile {
  int b;
  int32_t begin, first, count, before;  // before: slots in use ahead of the new tokens
  int32_t m0, queries;                  // the tile's first query, and how many [begin, end) has

  __device__ __forceinline__ bool any() const { return m0 < queries; }
  // The token that query m belongs to; outside 0 .. count - 1: none.
  __device__ __forceinline__ int32_t token(int32_t m, int group) const { return begin + m / group - first; }
  __device__ __forceinline__ int32_t slots_of(int32_t token, int32_t cap) const {
    return min(max(before + token + 1, 0), cap);
  }
  // Slots that query m sees; 0: a row without a token, or a token without slots.
  __device__ __forceinline__ int32_t seen(int32_t m, int group, int32_t cap) const {
    if (m >= queries) return 0;
    const int32_t i = token(m, group);
    return (uint32_t)i < (uint32_t)count ? slots_of(i, cap) : 0;
  }
};

__device__ __forceinline__ ChunkTile chunk_sequence(const ChunkParams& p, int b) {
  ChunkTile t;
  t.b = b;
  t.first = p.starts[b];
  t.count = max(p.counts[b], 0);
  t.before = (int32_t)min(max((int64_t)p.lengths[b] - t.count, (int64_t)INT32_MIN / 2), (int64_t)INT32_MAX / 2);
  t.begin = b == 0 ? 0 : min(max(t.first, 0), p.rows);
  const int32_t end = b + 1 < p.B ? min(max(p.starts[b + 1], t.begin), p.rows) : p.rows;
  t.queries = (end - t.begin) * p.group;  // (rows * nq fits 31 bits)
  t.m0 = 0;
  return t;
}

// The last sequence whose number is at most x, by the whole wave: 64 of them are looked at a time.
template <typename F>
__device__ __forceinline__ int last_sequence(int B, int64_t x, int lane, F number) {
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 63) >> 6, b = lo + lane * step;
    const bool upto = lane == 0 || (b < lo + n && number(b) <= x);
    const int at = (__popcll(__ballot(upto)) - 1) * step;
    lo += at;
    n = min(step, n - at);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Sequence b's tiles begin at number first_row * group / BM + b: ascending, and at least as far apart as
// the tiles of the rows between.
template <int BM>
__device__ __forceinline__ ChunkTile chunk_tile(const ChunkParams& p, uint32_t tile, int lane) {
  auto number = [&](int b) { return (int64_t)p.starts[b] * p.group / BM + b; };
  const int b = last_sequence(p.B, tile, lane, number);
  ChunkTile t = chunk_sequence(p, b);
  const int64_t at = b == 0 ? tile : tile - number(b);
  t.m0 = at < 0 || at * BM >= t.queries ? t.queries : (int32_t)at * BM;
  return t;
}

// Whether one of a word's two bf16 is infinite or no number.
__device__ __forceinline__ bool any_special(uint32_t x) {
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}
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
  ChunkTile ct;
  if (p.by_sequence) {
    ct = chunk_sequence(p, rest / p.nkv);
    if ((int64_t)ct.count * p.group > kFew || ct.first < ct.begin) return;
    const int64_t m0 = (int64_t)(ct.first - ct.begin) * p.group;
    ct.m0 = m0 < ct.queries ? (int32_t)m0 : ct.queries;
    ct.queries = min(ct.queries, ct.m0 + ct.count * p.group);
  } else {
    ct = chunk_tile<kFew>(p, rest / p.nkv, lane);
  }
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
    bool special = false;
    if (s0 + kPagedTile > min_seen || !there[0] || !there[1]) {
      // Slots past what a query sees weigh nothing, and values that no query sees must not count
      // either (0 * NaN is NaN); a page that is not in the pool makes a query that sees it NaN.
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int32_t slot = s0 + 16 * (i / 4) + 4 * g + i % 4;
        const bool ok = there[i / 4];
        s[i] = slot >= seen ? -INFINITY : (ok ? s[i] : __builtin_nanf(""));
        if (slot >= max_seen || !ok) vr[i] = vpiece_t{};
#pragma unroll
        for (int w = 0; w < RW; ++w) special = special || (slot >= min_seen && any_special(vw[i * RW + w]));
      }
      // Infinite values and NaN of a slot that some queries see and others do not are added at the end.
      if (__builtin_amdgcn_ballot_w64(special) != 0) {
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
      const int64_t at = split * p.part_rows + (p.by_sequence ? ((int64_t)ct.b * p.nkv + h) * kFew + c : row);
      if (d == 0) p.part_ml[at] = make_float2(M, sees ? L : -1.f);
      *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = make_float4(o[0], o[1], o[2], o[3]);
    } else {
      // No keys at all: zeros.  Keys whose scores are all -inf: 0 / 0, as softmax has it.
      const float inv = sees ? 1.f / L : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= inv;
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

// HD: dims of a row in LDS; NKD: steps of 16 dims (16 NKD >= D); GEN: D < HD, and the dims past D are zeros.
// RB: blocks of 32 queries of a wave, four waves a block.
template <int HD, int NKD, bool GEN, int RB>
__global__ __launch_bounds__(256, RB == 1 ? 2 : 1) void paged_chunk_tile_kernel(const ChunkParams p) {
  constexpr int BM = 128 * RB;
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
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TILE];  // two K tiles, two V tiles

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hi = lane >> 5, r32 = lane & 31;
  // KV heads run fastest: with eight of them each XCD reads the cache of one.  The last tiles of a
  // sequence, which see most, come first.
  const int h = blockIdx.x % p.nkv;
  uint32_t rest = blockIdx.x / p.nkv;
  const int split = rest % p.splits;
  const ChunkTile ct = chunk_tile<BM>(p, p.tiles - 1 - rest / p.splits, lane);
  if (!ct.any()) return;
  const int32_t cap = p.t.capacity(), group = p.group;
  const int32_t end_m = min(ct.queries, ct.m0 + BM);  // past the tile's last query
  auto row_of = [&](int32_t m) { return (int64_t)(ct.begin + m / group) * p.nq + h * group + m % group; };
  if ((int64_t)ct.count * group <= p.few) {
    // The other kernel's sequence: only the rows without a token are left, up to the next one's.
    if (split != 0) return;
    const int cpr = D / 8;
    for (int i = threadIdx.x; i < (end_m - ct.m0) * cpr; i += 256) {
      const int32_t m = ct.m0 + i / cpr;
      if ((uint32_t)ct.token(m, group) >= (uint32_t)ct.count)
        *reinterpret_cast<uint4*>(p.out + row_of(m) * D + i % cpr * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  // Slots seen by any of queries [m, to), and by the first token among them.
  auto most_seen = [&](int32_t m, int32_t to) {
    const int32_t first = max(ct.token(m, group), 0), last = min(ct.token(to - 1, group), ct.count - 1);
    return m < to && first <= last ? ct.slots_of(last, cap) : 0;
  };
  const int32_t block_seen = __builtin_amdgcn_readfirstlane(most_seen(ct.m0, end_m));
  const int32_t all_tiles = (block_seen + kKeys - 1) / kKeys, per = (all_tiles + p.splits - 1) / p.splits;
  const int32_t t0 = split * per, nt = max(min(all_tiles, t0 + per) - t0, 0);
  const int32_t mw = ct.m0 + wave * 32 * RB;
  const int32_t wave_seen = __builtin_amdgcn_readfirstlane(most_seen(mw, min(end_m, mw + 32 * RB)));
  // Tiles of this wave, and the first one that some of its queries do not see whole.
  const int32_t ntw = max(min((wave_seen + kKeys - 1) / kKeys - t0, nt), 0);
  const int32_t full = __builtin_amdgcn_readfirstlane(ct.slots_of(max(ct.token(mw, group), 0), cap)) / kKeys - t0;
  int32_t seen[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int32_t m = mw + rb * 32 + r32;
    seen[rb] = m < end_m ? ct.seen(m, group, cap) : 0;
  }

  f32x16 o[RB][NDB];
  float m_run[RB], m_ref[RB], l_run[RB], mx[RB];
  int32_t wild = INT32_MAX;  // the first tile whose infinite values and NaN were left out
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m_run[rb] = -INFINITY, m_ref[rb] = 0.f, l_run[rb] = 0.f, mx[rb] = -INFINITY;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[rb][db][v] = 0.f;
  }

  if (nt > 0) {
    // Q fragments: the B operand, query r32 of a block, dims 16 k + 8 hi .. + 8.
    bf16x8 qf[RB][NKD];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const uint16_t* q_row = p.q + (seen[rb] > 0 ? row_of(mw + rb * 32 + r32) * D : 0) + 8 * hi;
#pragma unroll
      for (int k = 0; k < NKD; ++k) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (seen[rb] > 0 && (!GEN || 16 * k + 8 * hi < D)) x = *reinterpret_cast<const uint4*>(q_row + 16 * k);
        qf[rb][k] = __builtin_bit_cast(bf16x8, x);
      }
    }

    // ---- pages -------------------------------------------------------------------
    // Lane i knows the page of this wave's 16 rows of tile window + i; a page's number is read off
    // when its tile is fetched.  missing: bit i for a tile with a page that is not in the pool.
    const int32_t* table = p.t.table + (int64_t)ct.b * p.t.ld;
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
    constexpr int KRING = RB == 1 ? 3 : 4;
    bf16x8 kfr[KRING], vfr[2][NDB], pf[RB][4];
    f32x16 s[2][RB][2];  // S^T of two tiles: the one in the softmax and the next one
    auto k_read = [&](int buf, int j) __attribute__((always_inline)) {
      kfr[j % KRING] = *reinterpret_cast<const bf16x8*>(lds + buf * TILE + kf_off[j % NKD] + (j / NKD) * 32 * ROWB);
    };
    auto qk = [&](int set, int i) __attribute__((always_inline)) {
      const int j = i / RB, rb = i % RB, kb = j / NKD, k = j % NKD;
      s[set][rb][kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kfr[j % KRING], qf[rb][k],
                                                              k == 0 ? f32x16{} : s[set][rb][kb], 0, 0, 0);
    };
    auto v_read = [&](int buf, int sl) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const uint8_t* at = lds + 2 * TILE + buf * TILE + vf_off[db] + sl * 16 * ROWB;
        typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
        const s16x4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 8 * ROWB));
        vfr[sl & 1][db] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    auto pv = [&](int sl, int i) __attribute__((always_inline)) {
      const int db = i / RB, rb = i % RB;
      o[rb][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vfr[sl & 1][db], pf[rb][sl], o[rb][db], 0, 0, 0);
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
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int v = 0; v < 16; ++v)
                if (v / 8 == (w & 1)) s[set][rb][w >> 1][v] = __builtin_nanf("");
        }
      }
      if (t >= full || bad) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const int32_t lim = seen[rb] - (t0 + t) * kKeys - 4 * hi;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const int c = kb * 32 + 8 * (v >> 2) + (v & 3);
              s[set][rb][kb][v] = c >= lim ? -INFINITY : s[set][rb][kb][v];
            }
        }
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float x[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          x[kb] = fmaxf(s[set][rb][kb][0], s[set][rb][kb][1]);
#pragma unroll
          for (int v = 2; v < 16; v += 2) x[kb] = fmaxf(fmaxf(x[kb], s[set][rb][kb][v]), s[set][rb][kb][v + 1]);
        }
        mx[rb] = max_of_halves(fmaxf(x[0], x[1])) * p.scale_log2;
      }
    };
    // The reference m_run moves only when a query's maximum passes it by more than kLazy; until then
    // P = 2^(t - m_run) <= 2^kLazy, which bf16 and fp32 hold, and the division by l cancels it.
    auto move_max = [&]() __attribute__((always_inline)) {
      bool over = false;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) over = over || mx[rb] > m_run[rb] + kLazy;
      if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const float m_new = fmaxf(m_run[rb], mx[rb]);
          m_ref[rb] = m_new == -INFINITY ? 0.f : m_new;  // scores of -inf weigh nothing, also the first ones
          const float alpha = __builtin_amdgcn_exp2f(m_run[rb] - m_ref[rb]);
          m_run[rb] = m_new;
          l_run[rb] *= alpha;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[rb][db][v] *= alpha;
        }
      }
    };
    // P of two neighbouring keys of slab sl, rounded to bf16 (the sum l is of the rounded ones, so that the
    // weights that V is multiplied by add up to 1), and its place among the slab's operand.
    auto p_pair = [&](int set, int u) __attribute__((always_inline)) {
      const int sl = u / (4 * RB), rb = u / 4 % RB, j = u % 4, kb = sl >> 1, v = 8 * (sl & 1) + 2 * j;
      const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[set][rb][kb][v], p.scale_log2, -m_ref[rb]));
      const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[set][rb][kb][v + 1], p.scale_log2, -m_ref[rb]));
      const uint32_t w = pack_bf16x2(a, b);
      l_run[rb] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w),
                                                  __builtin_bit_cast(bf16x2_t, 0x3F803F80u), l_run[rb], false);
      reinterpret_cast<uint32_t*>(&pf[rb][sl])[j] = w;
    };
    // Infinite values and NaN in a tile that some queries do not see whole (0 of P times them has no
    // value) leave V^T, slab by slab, and are added at the end.
    auto tame = [&](int sl) __attribute__((always_inline)) {
      typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
      uint32_t* w = reinterpret_cast<uint32_t*>(vfr[sl & 1]);
      u16x2 top = {0, 0};
#pragma unroll
      for (int i = 0; i < 4 * NDB; ++i)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
      if (__builtin_amdgcn_ballot_w64(max(top[0], top[1]) >= 0x7f80) == 0) return false;
#pragma unroll
      for (int i = 0; i < 4 * NDB; ++i) w[i] = without_special(w[i]);
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
        fetch(p.k_pages, t + 2, pg_ahead, k_off, lds + cur * TILE);
      } else {
        bad_next = bad_ahead;
      }
      if (t + 1 < nt) fetch(p.v_pages, t + 1, pg_next, v_off, lds + 2 * TILE + (cur ^ 1) * TILE);
    };
    auto body = [&](int32_t t, auto par, auto more) __attribute__((always_inline)) {
      constexpr int cur = decltype(par)::value, nxt = cur ^ 1;
      constexpr bool next = decltype(more)::value;
      constexpr int QK = next ? RB * 2 * NKD : 0, PV = RB * NDB, PAIRS = 16 * RB;
      constexpr int SPAN = QK + 3 * PV;  // products before the last slab's
      const bool masked = t >= full || bad_next;  // (bad_next: of tile t until sync has gone on)
      sync(t, cur);
      if constexpr (next) {
#pragma unroll
        for (int j = 0; j < KRING - 1 && j < 2 * NKD; ++j) k_read(nxt, j);
      } else {
        v_read(cur, 0);
      }
      move_max();
#pragma unroll
      for (int i = 0; i < QK + 4 * PV; ++i) {
        // The pairs of P are spread over the products before the last slab's, each slab's before its own.
#pragma unroll
        for (int u = 0; u < PAIRS; ++u) {
          const int before = QK + u / (4 * RB) * PV, even = u * SPAN / PAIRS;
          if ((even < before ? even : before) == i) p_pair(cur, u);
        }
        if (i < QK) {
          if (i % RB == 0 && i / RB + KRING - 1 < 2 * NKD) k_read(nxt, i / RB + KRING - 1);
          qk(nxt, i);
          if (i == (QK > 8 ? QK - 8 : 0)) v_read(cur, 0);
        } else {
          const int sl = (i - QK) / PV, at = (i - QK) % PV;
          if (at == 0) {
            if (sl < 3) v_read(cur, sl + 1);
            if (__builtin_expect(masked, 0) && tame(sl)) wild = min(wild, t);
          }
          pv(sl, at);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (next) row_max(nxt, t + 1, bad_next);
    };

    look_up();
    advance(0);
    fetch(p.k_pages, 0, pg_ahead, k_off, lds);
    fetch(p.v_pages, 0, pg_ahead, v_off, lds + 2 * TILE);
    if (nt > 1) {
      advance(1);
      fetch(p.k_pages, 1, pg_ahead, k_off, lds + TILE);
    } else {
      bad_next = bad_ahead;
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 15));
    __syncthreads();
    if (ntw > 0) {
#pragma unroll
      for (int j = 0; j < KRING - 1 && j < 2 * NKD; ++j) k_read(0, j);
#pragma unroll
      for (int i = 0; i < RB * 2 * NKD; ++i) {
        if (i % RB == 0 && i / RB + KRING - 1 < 2 * NKD) k_read(0, i / RB + KRING - 1);
        qk(0, i);
      }
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
    for (; t < nt; ++t) sync(t, t & 1);
  }

  // As in the few kernel: added as they are, whatever their weights.
  for (int32_t slot = wild < ntw ? (t0 + wild) * kKeys : INT32_MAX; slot < min((t0 + ntw) * kKeys, wave_seen); ++slot) {
    const int64_t row = p.t.row(ct.b, h, p.nkv, slot);
    if (row < 0) continue;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int d = 32 * db + 8 * (v >> 2) + 4 * hi + (v & 3);
          const uint32_t x = !GEN || d < D ? p.v_pages[row * D + d] : 0u;
          if (slot < seen[rb] && (x & 0x7f80u) == 0x7f80u) o[rb][db][v] += bf16_bits_to_f32(x);
        }
  }

  // ---- O^T / l ---------------------------------------------------------------------
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) l_run[rb] = sum_of_halves(l_run[rb]);
  if (p.splits > 1) {
    const int64_t base = split * p.part_rows;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int32_t m = mw + rb * 32 + r32;
      if (m >= end_m) continue;
      const int64_t at = base + row_of(m);
      if (hi == 0) p.part_ml[at] = make_float2(m_run[rb], seen[rb] > 0 ? l_run[rb] : -1.f);
      if (ntw == 0) continue;  // (a maximum of -inf: the sums are not read)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * db + 8 * g + 4 * hi;
          if (!GEN || d < D)
            *reinterpret_cast<float4*>(p.part_o + at * D + d) =
                make_float4(o[rb][db][4 * g], o[rb][db][4 * g + 1], o[rb][db][4 * g + 2], o[rb][db][4 * g + 3]);
        }
    }
    return;
  }
  // A lane holds 8-byte pieces of one query: they are staged through LDS, 16-byte chunk c of row r at position
  // c ^ (r % CPR), and go out as whole rows.
  static_assert(4 * 32 * RB * ROWB <= 4 * TILE, "output staging must fit the tiles");
  __syncthreads();
  uint8_t* stage = lds + wave * 32 * RB * ROWB;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float inv = 1.f / l_run[rb];
    const bool sees = seen[rb] > 0;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint2 w = make_uint2(pack_bf16x2(o[rb][db][4 * g] * inv, o[rb][db][4 * g + 1] * inv),
                             pack_bf16x2(o[rb][db][4 * g + 2] * inv, o[rb][db][4 * g + 3] * inv));
        if (!sees) w = make_uint2(0u, 0u);
        const int ch = (db * 4 + g) ^ (r32 % CPR);
        *reinterpret_cast<uint2*>(stage + (rb * 32 + r32) * ROWB + ch * 16 + hi * 8) = w;
      }
  }
  // The wave's own LDS writes complete before its reads (and stay ahead of them).
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
  __builtin_amdgcn_wave_barrier();
  const int jc = lane % CPR;
  if (GEN && jc * 8 >= D) return;
#pragma unroll
  for (int i = 0; i < 32 * RB * CPR / 64; ++i) {
    const int r = i * (64 / CPR) + lane / CPR;
    const uint4 x = *reinterpret_cast<const uint4*>(stage + r * ROWB + ((jc ^ (r % CPR)) << 4));
    if (mw + r < end_m) *reinterpret_cast<uint4*>(p.out + row_of(mw + r) * D + jc * 8) = x;
  }
}

constexpr int kJoinThreads = 256;

// One query a block: its splits' sums by 256 threads over splits and columns.  The first few_blocks are
// queries of the few kernel's sequences (f), the others the (row, head) pairs of p's.
__global__ __launch_bounds__(kJoinThreads) void paged_chunk_join_kernel(const ChunkParams f, uint32_t few_blocks,
                                                                        const ChunkParams p) {
  __shared__ float4 part[kJoinThreads];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool of_few = blockIdx.x < few_blocks;
  const int splits = of_few ? f.splits : p.splits;
  const int64_t step = of_few ? f.part_rows : p.part_rows, at0 = of_few ? blockIdx.x : blockIdx.x - few_blocks;
  const float* part_o = of_few ? f.part_o : p.part_o;
  const float2* part_ml = of_few ? f.part_ml : p.part_ml;
  int64_t row = at0;
  if (of_few) {
    const ChunkTile ct = chunk_sequence(f, (int)(at0 / (f.nkv * kFew)));
    const int h = (int)(at0 / kFew % f.nkv), c = (int)(at0 % kFew);
    const int64_t first = (int64_t)(ct.first - ct.begin) * f.group;
    if ((int64_t)ct.count * f.group > kFew || c >= ct.count * f.group || ct.first < ct.begin || first + c >= ct.queries)
      return;
    row = ((int64_t)ct.first + c / f.group) * f.nq + h * f.group + c % f.group;
  } else if (p.few > 0) {
    // A token of the few kernel's sequences is joined above.
    const int32_t r = (int32_t)(row / p.nq);
    const int b = last_sequence(p.B, r, lane, [&](int i) { return (int64_t)p.starts[i]; });
    const int32_t count = max(p.counts[b], 0);
    if ((int64_t)count * p.group <= p.few) return;
  }
  const int cols = p.D / 4, groups = min(kJoinThreads / cols, 16);
  const int sg = tid / cols, d = (tid - sg * cols) * 4;
  float2 ml[kPagedMaxSplits / 64];
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPagedMaxSplits / 64; ++i) {
    const int s = i * 64 + lane;
    ml[i] = s < splits ? part_ml[s * step + at0] : make_float2(-INFINITY, 0.f);
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
    for (int s = sg; s < splits; s += groups) {
      const int64_t at = s * step + at0;
      const float top = part_ml[at].x;
      if (top == -INFINITY) continue;  // (no sum was written, or one of nothing)
      const float f = __builtin_amdgcn_exp2f(top - ref);
      const float4 x = *reinterpret_cast<const float4*>(part_o + at * p.D + d);
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
  const float x[4] = {sees ? o.x * inv : 0.f, sees ? o.y * inv : 0.f, sees ? o.z * inv : 0.f, sees ? o.w * inv : 0.f};
  head_store4(p.out + row * p.D + d, x);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// What a call launches: the few kernel (over tiles, or a block per sequence beside the tile kernel), the tile
// kernel, and a join where slots are split.
struct ChunkPlan {
  bool few, tile;
  int64_t few_tiles, tiles;  // blocks a KV head and split
  int few_splits, splits;
  int64_t few_rows, rows;    // of their partial sums
  size_t few_o, few_ml, o, ml;
  size_t total() const { return few_o + few_ml + o + ml; }
};

// Splits of a tile's slots: blocks come in turns of two a CU, and a turn costs what its slots cost.
int tile_splits(int64_t blocks, int64_t cap) {
  const int64_t slots = 2 * device_cu_count();
  const int64_t most = std::min<int64_t>(kPagedMaxSplits, (cap + 8 * kKeys - 1) / (8 * kKeys));
  int best = 1;
  double cost = 1e30;
  for (int64_t s = 1; s <= most && (s == 1 || blocks * (s - 1) < slots); ++s) {
    const double c = (double)((blocks * s + slots - 1) / slots) / s + (s > 1 ? 0.02 * s : 0.0);
    if (c < cost) cost = c, best = (int)s;
  }
  return best;
}

ChunkPlan chunk_plan(int64_t rows, int64_t B, int64_t nq, int64_t nkv, int64_t hd, int64_t cap, int64_t most) {
  ChunkPlan c{};
  const int64_t group = nq / nkv;
  c.tile = std::min(most, rows) * group > kFew;
  c.few = !c.tile || (B > 1 && group <= kFew);
  if (c.few) {
    c.few_tiles = c.tile ? B : rows * group / kFew + B;
    c.few_splits = paged_splits(c.few_tiles * nkv, cap);
    c.few_rows = c.tile ? B * nkv * kFew : rows * nq;
    if (c.few_splits > 1) {
      c.few_o = round16((size_t)(c.few_splits * c.few_rows * hd) * sizeof(float));
      c.few_ml = round16((size_t)(c.few_splits * c.few_rows) * sizeof(float2));
    }
  }
  if (c.tile) {
    c.tiles = rows * group / 128 + B;
    c.splits = tile_splits(((rows * group + 127) / 128 + (B - 1) / 2) * nkv, cap);
    c.rows = rows * nq;
    if (c.splits > 1) {
      c.o = round16((size_t)(c.splits * c.rows * hd) * sizeof(float));
      c.ml = round16((size_t)(c.splits * c.rows) * sizeof(float2));
    }
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

template <int RB>
void launch_tile(const ChunkParams& p, const dim3& grid, hipStream_t s) {
  const dim3 block(256);
  switch (p.D) {
    case 32: return paged_chunk_tile_kernel<32, 2, false, RB><<<grid, block, 0, s>>>(p);
    case 64: return paged_chunk_tile_kernel<64, 4, false, RB><<<grid, block, 0, s>>>(p);
    case 128: return paged_chunk_tile_kernel<128, 8, false, RB><<<grid, block, 0, s>>>(p);
    default: break;
  }
  switch ((p.D + 15) / 16) {
    case 1:
    case 2: return paged_chunk_tile_kernel<64, 2, true, RB><<<grid, block, 0, s>>>(p);
    case 3: return paged_chunk_tile_kernel<64, 3, true, RB><<<grid, block, 0, s>>>(p);
    case 4: return paged_chunk_tile_kernel<64, 4, true, RB><<<grid, block, 0, s>>>(p);
    case 5: return paged_chunk_tile_kernel<128, 5, true, RB><<<grid, block, 0, s>>>(p);
    case 6: return paged_chunk_tile_kernel<128, 6, true, RB><<<grid, block, 0, s>>>(p);
    case 7: return paged_chunk_tile_kernel<128, 7, true, RB><<<grid, block, 0, s>>>(p);
    default: return paged_chunk_tile_kernel<128, 8, true, RB><<<grid, block, 0, s>>>(p);
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
  const int64_t few_blocks = c.few ? c.few_tiles * nkv * c.few_splits : 0;
  const int64_t blocks = c.tile ? c.tiles * nkv * c.splits : 0;
  const int64_t few_joins = c.few && c.few_splits > 1 ? c.few_rows : 0, joins = c.tile && c.splits > 1 ? c.rows : 0;
  if (few_blocks > max_blocks(64 * kPagedWaves) || blocks > max_blocks(256) ||
      few_joins + joins > max_blocks(kJoinThreads))
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
  ChunkParams f = p;
  char* at = static_cast<char*>(work);
  f.by_sequence = c.tile;
  f.splits = c.few_splits;
  f.part_rows = c.few_rows;
  f.part_o = reinterpret_cast<float*>(at);
  f.part_ml = reinterpret_cast<float2*>(at + c.few_o);
  at += c.few_o + c.few_ml;
  p.few = c.few ? kFew : 0;
  p.tiles = (uint32_t)c.tiles;
  p.splits = c.splits;
  p.part_rows = c.rows;
  p.part_o = reinterpret_cast<float*>(at);
  p.part_ml = reinterpret_cast<float2*>(at + c.o);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (c.few) {
    launch_few(f, dim3((unsigned)few_blocks), s);
    if (int rc = check_launch(name)) return rc;
  }
  if (c.tile) {
    launch_tile<1>(p, dim3((unsigned)blocks), s);
    if (int rc = check_launch(name)) return rc;
  }
  if (few_joins + joins == 0) return CDX_OK;
  // (Where the few kernel took every sequence, its sums lie by (row, head).)
  if (!c.tile)
    paged_chunk_join_kernel<<<dim3((unsigned)few_joins), dim3(kJoinThreads), 0, s>>>(f, 0, f);
  else
    paged_chunk_join_kernel<<<dim3((unsigned)(few_joins + joins)), dim3(kJoinThreads), 0, s>>>(f, (uint32_t)few_joins, p);
  return check_launch(name);
}
