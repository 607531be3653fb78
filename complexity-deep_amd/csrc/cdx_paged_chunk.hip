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
  float scale_log2;
  uint16_t* out;    // [rows][nq][D]
  float* part_o;    // [splits][rows][nq][D], unnormalised
  float2* part_ml;  // [splits][rows][nq]: maximum (log2 units) and sum; a sum of -1: no key at all
};

// A tile of BM queries of one sequence.  Sequence b's own rows, with those that follow them up to the
// next one's, are rows begin .. end - 1 of the call; row r is token r - first of the sequence.
struct ChunkTile {
  int b;
  int32_t begin, first, count, before;  // before: slots in use ahead of the new tokens
  int64_t m0, queries;                  // the tile's first query, and how many [begin, end) has

  __device__ __forceinline__ bool any() const { return m0 < queries; }
  // Slots that query m sees; 0: a row without a token, or a token without slots.
  __device__ __forceinline__ int32_t seen(int64_t m, int group, int32_t cap) const {
    if (m >= queries) return 0;
    const int32_t i = begin + (int32_t)(m / group) - first;
    return (uint32_t)i < (uint32_t)count ? min(max(before + i + 1, 0), cap) : 0;
  }
};

// Sequence b's tiles begin at number first_row * group / BM + b: ascending, and at least as far apart as
// the tiles of the rows between.  64 sequences are looked at a time.
template <int BM>
__device__ __forceinline__ ChunkTile chunk_tile(const ChunkParams& p, uint32_t tile, int lane) {
  auto number = [&](int b) { return (int64_t)p.starts[b] * p.group / BM + b; };
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
  t.before = (int32_t)min(max((int64_t)p.lengths[b] - t.count, (int64_t)INT32_MIN / 2), (int64_t)INT32_MAX / 2);
  t.begin = b == 0 ? 0 : min(max(t.first, 0), p.rows);
  const int32_t end = b + 1 < p.B ? min(max(p.starts[b + 1], t.begin), p.rows) : p.rows;
  t.queries = (int64_t)(end - t.begin) * p.group;
  const int64_t at = b == 0 ? tile : tile - number(b);
  t.m0 = at < 0 ? t.queries : at * BM;
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

constexpr int kFew = 16;  // queries of a block: the columns of a matrix instruction

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
  const ChunkTile ct = chunk_tile<kFew>(p, rest / p.nkv, lane);
  if (!ct.any()) return;
  const int queries = (int)min((int64_t)kFew, ct.queries - ct.m0);
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
    const int64_t m = ct.m0 + i, row = ct.begin + m / p.group;
    return row * p.nq + h * p.group + m % p.group;
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
      // Infinite values and NaN of a slot that some queries see and others do not: added one by one.
      special = __builtin_amdgcn_ballot_w64(special) != 0;
      if (special) {
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
    if (special) {
#pragma unroll 1
      for (int slot = 0; slot < kPagedTile; ++slot) {
        if (s0 + slot >= max_seen || !there[slot >> 4]) continue;
        // Query n's weight of the slot lies with the lanes of group (slot % 16) / 4.
        float w = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) w = i == 4 * (slot >> 4) + (slot & 3) ? pf[i] : w;
        w = __shfl(w, n + 4 * (slot & 12), 64);
        if (s0 + slot >= seen) continue;
        const uint16_t* v_row = v_base[slot >> 4] + (slot & 15) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < DPL; ++j) {
            const int d = (4 * g + r) * DPL + j;
            const uint32_t x = d < D ? v_row[d] : 0u;
            if ((x & 0x7f80u) == 0x7f80u) acc[j][r] = __builtin_fmaf(w, bf16_bits_to_f32(x), acc[j][r]);
          }
      }
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
      const float inv = sees ? 1.f / L : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= inv;
      head_store4(p.out + row * p.D + d, o);
    }
  }
}

constexpr int kJoinThreads = 256;

// One (row, head) a block: its splits' sums by 256 threads over splits and columns.
__global__ __launch_bounds__(kJoinThreads) void paged_chunk_join_kernel(const ChunkParams p) {
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
      const float f = __builtin_amdgcn_exp2f(p.part_ml[at].x - ref);
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
  int64_t tiles;  // numbers that a tile may have
  int splits;
  size_t part_o, total;
};

ChunkPlan chunk_plan(int64_t rows, int64_t B, int64_t nq, int64_t nkv, int64_t hd, int64_t cap) {
  ChunkPlan c{};
  c.tiles = rows * (nq / nkv) / kFew + B;
  c.splits = paged_splits(c.tiles * nkv, cap);
  if (c.splits > 1) {
    c.part_o = round16((size_t)(c.splits * rows * nq * hd) * sizeof(float));
    c.total = c.part_o + round16((size_t)(c.splits * rows * nq) * sizeof(float2));
  }
  return c;
}

}  // namespace
}  // namespace cdx

extern "C" size_t cdx_paged_chunk_attention_workspace_bytes(int64_t rows, int64_t B, int32_t nq, int32_t nkv,
                                                            int32_t hd, int64_t capacity, int64_t max_tokens) {
  using namespace cdx;
  if (rows <= 0 || B <= 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || hd <= 0 || capacity <= 0 || max_tokens < 0)
    return 0;
  return chunk_plan(rows, B, nq, nkv, hd, capacity).total;
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
  const ChunkPlan c = chunk_plan(rows, B, nq, nkv, hd, cap);
  const int64_t blocks = c.tiles * nkv * c.splits;
  if (blocks > max_blocks(64 * kPagedWaves) || rows * nq > max_blocks(kJoinThreads))
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (!q || !k_pages || !v_pages || !table || !starts || !counts || !lengths || !out)
    return fail(CDX_EINVAL, "%s: null pointer", name);
  if (work_bytes < c.total || (c.total > 0 && !work))
    return fail(CDX_EWORKSPACE, "%s: workspace needs %zu bytes, got %zu", name, c.total, work ? work_bytes : 0);
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
  p.splits = c.splits;
  p.scale_log2 = scale * kLog2e;
  p.out = out;
  p.part_o = static_cast<float*>(work);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(work) + c.part_o);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(64 * kPagedWaves);
  if (hd <= 32)
    paged_chunk_few_kernel<1, 4, false><<<grid, block, 0, s>>>(p);
  else if (hd < 64)
    paged_chunk_few_kernel<2, 4, false><<<grid, block, 0, s>>>(p);
  else if (hd == 64)
    paged_chunk_few_kernel<2, 4, true><<<grid, block, 0, s>>>(p);
  else if (hd <= 96)
    paged_chunk_few_kernel<3, 8, false><<<grid, block, 0, s>>>(p);
  else if (hd < 128)
    paged_chunk_few_kernel<4, 8, false><<<grid, block, 0, s>>>(p);
  else
    paged_chunk_few_kernel<4, 8, true><<<grid, block, 0, s>>>(p);
  if (int rc = check_launch(name)) return rc;
  if (c.splits == 1) return CDX_OK;
  paged_chunk_join_kernel<<<dim3((unsigned)(rows * nq)), dim3(kJoinThreads), 0, s>>>(p);
  return check_launch(name);
}
