// Attention of one new token per sequence over a paged KV cache, for gfx950.
//
//   o[b, h] = sum_t p_t v_t,  p = softmax_t(scale q[b, h] . k_t),  t < length[b],
//
// with the query heads of a group sharing one head of K and V.  Every key and value is read
// once for one row of scores, so the cache's bytes bound the operator; what the kernel arranges
// is that they arrive in whole 16-byte pieces, enough of them at a time, and that each is used
// for all query heads of its group.
//
//   * A wave walks tiles of 32 slots.  S^T = K Q^T with v_mfma_f32_16x16x32_bf16: the rows are
//     slots, the 16 columns query heads of one group (unused columns cost nothing: the matrix
//     cores wait for memory).  A lane holds one head's scores of 8 slots, 4 g .. 4 g + 3 of
//     each half of the tile (g = lane / 16).
//   * O^T = V^T P^T then wants, in the same lane, 8 slots of P and of V: P is there already, and
//     V's 8 rows are loaded in that slot order, a piece of DPL columns each, and transposed in
//     registers (two bf16 of neighbouring rows per v_perm).  Nothing goes through LDS.
//   * One pass: the running maximum and sum of the softmax, in log2 units and fp32, per wave.
//     The eight waves of a block take every eighth tile and are joined through LDS.  P enters
//     the product with V as two bf16 parts (2^-16 of it is lost; one part alone, 2^-8, takes 5.3
//     instead of 5.6 us for 1 x 500 slots, 48.8 instead of 49.4 for 64 x 1024 and the same for long ones).
//     The sums are divided at the end: finite values larger than 3.4e38 / length may overflow them.
//   * A sequence is split into `splits` runs of tiles over blocks; the partial sums (fp32, with
//     their maximum and sum) are joined by a second kernel, which also adds up the weights that
//     each slot received, from the scores that the first kernel left.
//
// Measured (us and TB/s of K and V, calls in a row, both kernels): 16/8 heads of 128, 4 x 65536
// slots 184 (5.8), 64 x 1024 49 (5.4), 64 sequences of 1 .. 2048 56.5 (4.8), 1 x 1000 11.5; 16/4 of
// 80, 64 x 4096 67 (5.0); 8/4 of 40, 1 x 500 5.3-5.6.  The plainest kernel reads 6.3 TB/s here.  What it took:
// eight waves of at most 128 registers, two blocks on a CU (with a base address per tile shared by
// the wave, and masks only in a sequence's last tile) 67 -> 56 us for the ragged 64; four waves of
// 140 registers had been the better form before.
#include <algorithm>

#include "cdx_paged_attn.h"

namespace cdx {

// Blocks that a sequence and head is split over: enough for two blocks on each CU, four where
// tables are long (lengths then differ more: 100 sequences of up to 8192 slots, 16/4 heads of 80,
// 119 against 110 us, 4 x 65536 slots 185 against 180), each with at least two tiles per wave (four:
// 1 x 2000 slots 11.5 against 16.4 us).  Short tables whose blocks fill the CUs are not split, which
// saves the second kernel (32 x 1024 slots 25.7 against 22.2 us).
int paged_splits(int64_t blocks, int64_t cap) {
  const int64_t cus = device_cu_count();
  if (blocks >= cus && cap <= 4 * kPagedWaves * kPagedTile) return 1;
  const int64_t want = ((cap >= 4096 ? 4 : 2) * cus + blocks - 1) / blocks;
  const int64_t most = (cap + 2 * kPagedWaves * kPagedTile - 1) / (2 * kPagedWaves * kPagedTile);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kPagedMaxSplits}));
}

namespace {

constexpr int kTile = kPagedTile, kWaves = kPagedWaves;
constexpr int kHeads = 16;  // query heads of a block: the columns of a matrix instruction

struct PagedAttnParams {
  const uint16_t* q;  // [B][nq][D]
  const uint16_t* k_pages;
  const uint16_t* v_pages;
  PagedTable t;
  const int32_t* lengths;
  int32_t B, nq, nkv, D, group, head_tiles, splits;
  float scale_log2;
  uint16_t* out;      // [B][nq][D]
  float* part_o;      // [splits][B][nq][D], unnormalised
  float2* part_ml;    // [splits][B][nq]: maximum (log2 units) and sum
  float* scores;      // [B][nq][cap] in log2 units, or nullptr
  const float* w_in;  // [B][nkv][cap]
  float* w_out;
};

// NC: pieces of 32 dims in a head; DPL: columns of V that a lane holds (16 DPL >= D); W: waves; FULL: D == 32 NC ==
// 16 DPL, so that every lane holds dims of the head.
template <int NC, int DPL, int W, bool FULL>
__global__ __launch_bounds__(64 * W, NC == 4 && !FULL ? 2 : 4) void paged_attn_kernel(const PagedAttnParams p) {
  typedef typename Piece<DPL>::type vpiece_t;
  constexpr int PITCH = 16 * DPL + 4;
  __shared__ float lds_o[W][kHeads][PITCH];
  __shared__ float lds_m[W][kHeads], lds_l[W][kHeads];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // Splits run fastest, so that the blocks of one sequence and head lie together.
  const uint32_t split = blockIdx.x % p.splits;
  uint32_t rest = blockIdx.x / p.splits;
  const int ht = rest % p.head_tiles;
  rest /= p.head_tiles;
  const int h = rest % p.nkv, b = rest / p.nkv;
  const int heads = min(kHeads, p.group - ht * kHeads);
  const int head0 = h * p.group + ht * kHeads;

  const int32_t cap = p.t.capacity();
  const int32_t len = min(p.lengths[b], cap);
  const int32_t tiles = len > 0 ? (len + kTile - 1) / kTile : 0;
  const int32_t per = (tiles + p.splits - 1) / p.splits;
  const int32_t t_end = min(tiles, (int32_t)(split + 1) * per);

  // Q^T: column n is head n, 8 dims per lane and piece; dims past the head and heads past the
  // group are zero.
  bf16x8 qf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    const int d = c * 32 + g * 8;
    if (n < heads && d < p.D) x = *reinterpret_cast<const uint4*>(p.q + ((int64_t)b * p.nq + head0 + n) * p.D + d);
    qf[c] = __builtin_bit_cast(bf16x8, x);
  }

  f32x4 acc[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const int32_t* table = p.t.table + (int64_t)b * p.t.ld;
  const int lps = p.t.log2_page;
  // A tile's rows lie at a base that the wave shares; a lane's offsets from it stay.
  const int D = FULL ? 32 * NC : p.D;
  const uint32_t k_at = n * D + g * 8, v_at = 4 * g * D + n * DPL;
  const bool v_on = FULL || n * DPL < D;

  for (int32_t tile = (int32_t)split * per + wave; tile < t_end; tile += W) {
    const int32_t s0 = tile * kTile;
    // The two halves of 16 slots each lie inside one page.
    const uint16_t *k_base[2], *v_base[2];
    bool there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t at = s0 + 16 * i;
      const int32_t pg = at < len ? table[at >> lps] : -1;
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
    if (s0 + kTile > len || !there[0] || !there[1]) {
      // Slots past the sequence weigh nothing, and their values must not count either (0 * NaN is
      // NaN); a page that is not in the pool makes the row NaN.
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool behind = s0 + 16 * (i / 4) + 4 * g + i % 4 >= len, ok = there[i / 4];
        s[i] = behind ? -INFINITY : (ok ? s[i] : __builtin_nanf(""));
        if (behind || !ok) vr[i] = vpiece_t{};
      }
    }
    if (p.scores != nullptr && n < heads) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (s0 + 16 * i < len)  // (then the 16 slots lie inside the capacity)
          *reinterpret_cast<f32x4*>(p.scores + ((int64_t)b * p.nq + head0 + n) * cap + s0 + 16 * i + 4 * g) =
              f32x4{s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
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
    const uint32_t* vw = reinterpret_cast<const uint32_t*>(vr);  // [8 rows][DPL / 2]
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      uint4 a;
      const int w = j / 2;
      constexpr int RW = DPL / 2;
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
      // value: an infinite value counts once, by the high part, and is a finite one here (two
      // packed minima a word: 1 x 500 slots 5.2 -> 5.3 us, 64 of 1 .. 2048 56.1 -> 56.5, 4 x 65536 none).
      a = make_uint4(finite_halves(a.x), finite_halves(a.y), finite_halves(a.z), finite_halves(a.w));
      acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), pb_low, acc[j], 0, 0, 0);
    }
  }

  // Join the waves: lane (n, g) holds head n, columns (4 g + r) DPL + j.
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
  for (int i = threadIdx.x; i < heads * (p.D / 4); i += 64 * W) {
    const int hd = i / (p.D / 4), d = (i - hd * (p.D / 4)) * 4;
    float M = lds_m[0][hd];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, lds_m[w][hd]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(lds_m[w][hd] - ref);
      L = __builtin_fmaf(f, lds_l[w][hd], L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(f, lds_o[w][hd][d + e], o[e]);
    }
    const int64_t row = (int64_t)b * p.nq + head0 + hd;
    if (p.splits > 1 || p.scores != nullptr) {
      const int64_t at = (int64_t)split * p.B * p.nq + row;
      if (d == 0) p.part_ml[at] = make_float2(M, L);
      if (p.splits > 1) *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = make_float4(o[0], o[1], o[2], o[3]);
    }
    if (p.splits == 1) {
      // No keys at all: zeros.  Keys whose scores are all -inf: 0 / 0, as softmax has it.
      const float inv = len > 0 ? 1.f / L : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= inv;
      head_store4(p.out + row * p.D + d, o);
    }
  }
}

constexpr int kJoinThreads = 256;
constexpr int kMaxSplits = kPagedMaxSplits;
constexpr int kJoinSlots = 512;  // slots of the weights that a block adds up

// Maximum (log2 units, 0 where there is none) and sum of a row of scores from its splits' own, by
// a whole wave, returned to every lane.
__device__ __forceinline__ float2 join_statistics(const PagedAttnParams& p, int64_t row, int lane) {
  const int64_t step = (int64_t)p.B * p.nq;
  float2 ml[kMaxSplits / 64];
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 64; ++i) {
    const int s = i * 64 + lane;
    ml[i] = s < p.splits ? p.part_ml[s * step + row] : make_float2(-INFINITY, 0.f);
  }
#pragma unroll
  for (int i = 0; i < kMaxSplits / 64; ++i) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 64; ++i) L = __builtin_fmaf(__builtin_amdgcn_exp2f(ml[i].x - ref), ml[i].y, L);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) L += __shfl_xor(L, d, 64);
  return make_float2(ref, L);
}

// The first `rows` blocks (none without splits) join the splits of one row each, 256 threads over
// splits and columns.  The others add up the softmax weights of 512 slots of one (sequence,
// KV head), over the heads of its group.
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(const PagedAttnParams p, uint32_t rows, int chunks) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t step = (int64_t)p.B * p.nq;
  const int32_t cap = p.t.capacity();
  if (blockIdx.x < rows) {
    __shared__ float4 part[kJoinThreads];
    const int64_t row = blockIdx.x;
    const int cols = p.D / 4, groups = min(kJoinThreads / cols, 16);
    const int sg = tid / cols, d = (tid - sg * cols) * 4;
    const float2 ml = join_statistics(p, row, lane);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (sg < groups) {
#pragma unroll 4
      for (int s = sg; s < p.splits; s += groups) {
        const int64_t at = s * step + row;
        const float f = __builtin_amdgcn_exp2f(p.part_ml[at].x - ml.x);
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
    const float inv = p.lengths[row / p.nq] > 0 ? 1.f / ml.y : 0.f;
    const float f[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    head_store4(p.out + row * p.D + d, f);
    return;
  }
  constexpr int PER = kJoinSlots / kJoinThreads;
  __shared__ float2 stats[kHeads];
  const uint32_t block = blockIdx.x - rows, slab = block / chunks;
  const int32_t s0 = (int32_t)(block - slab * chunks) * kJoinSlots + tid;
  const int b = slab / p.nkv, h = slab - b * p.nkv;
  const int32_t len = min(p.lengths[b], cap);
  float w[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int32_t s = s0 + u * kJoinThreads;
    w[u] = s < cap ? p.w_in[(int64_t)slab * cap + s] : 0.f;
  }
  if (s0 - tid < len) {
    for (int h0 = 0; h0 < p.group; h0 += kHeads) {
      const int heads = min(kHeads, p.group - h0);
      const int64_t row0 = (int64_t)b * p.nq + h * p.group + h0;
      __syncthreads();
      for (int i = wave; i < heads; i += kJoinThreads / 64) {
        const float2 ml = join_statistics(p, row0 + i, lane);
        if (lane == 0) stats[i] = make_float2(ml.x, 1.f / ml.y);
      }
      __syncthreads();
#pragma unroll 4
      for (int i = 0; i < heads; ++i) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const int32_t s = s0 + u * kJoinThreads;
          if (s < len) {
            const float e = __builtin_amdgcn_exp2f(p.scores[(row0 + i) * cap + s] - stats[i].x);
            w[u] = __builtin_fmaf(e, stats[i].y, w[u]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int32_t s = s0 + u * kJoinThreads;
    if (s < cap) p.w_out[(int64_t)slab * cap + s] = w[u];
  }
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

struct PagedWork {
  size_t o, ml, scores, total;
};
PagedWork paged_work(int64_t B, int64_t nq, int64_t hd, int64_t cap, int splits, bool weights) {
  PagedWork w{};
  w.o = splits > 1 ? round16((size_t)(splits * B * nq * hd) * sizeof(float)) : 0;
  w.ml = splits > 1 || weights ? round16((size_t)(splits * B * nq) * sizeof(float2)) : 0;
  w.scores = weights ? round16((size_t)(B * nq * cap) * sizeof(float)) : 0;
  w.total = w.o + w.ml + w.scores;
  return w;
}

}  // namespace
}  // namespace cdx

extern "C" size_t cdx_paged_attention_workspace_bytes(int64_t B, int32_t nq, int32_t nkv, int32_t hd,
                                                      int64_t capacity, int32_t with_weights) {
  using namespace cdx;
  if (B <= 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || hd <= 0 || capacity <= 0) return 0;
  const int64_t head_tiles = (nq / nkv + kHeads - 1) / kHeads;
  return paged_work(B, nq, hd, capacity, paged_splits(B * nkv * head_tiles, capacity), with_weights != 0).total;
}

extern "C" int cdx_paged_attention_fwd(const uint16_t* q, int64_t B, int32_t nq, int32_t nkv, int32_t hd,
                                       const uint16_t* k_pages, const uint16_t* v_pages, const int32_t* table,
                                       int64_t table_ld, int64_t width, int64_t num_pages, int32_t page_size,
                                       const int32_t* lengths, float scale, uint16_t* out, const float* weights_in,
                                       float* weights_out, void* work, size_t work_bytes, void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_attention_fwd";
  clear_error();
  PagedAttnParams p{};
  if (int rc = paged_table(name, table, table_ld, width, num_pages, page_size, B, nkv, hd, &p.t)) return rc;
  if (nq <= 0 || nq % nkv != 0) return fail(CDX_EINVAL, "%s: bad shape nq=%d nkv=%d", name, nq, nkv);
  if (!(scale > 0.f) || scale > 3e38f) return fail(CDX_EINVAL, "%s: scale must be > 0 and finite", name);
  if ((weights_in == nullptr) != (weights_out == nullptr))
    return fail(CDX_EINVAL, "%s: weights_in and weights_out must both be given or both be NULL", name);
  if (width == 0 || num_pages == 0) return fail(CDX_EINVAL, "%s: empty block table or pool", name);
  if (B == 0) return CDX_OK;
  const int64_t cap = width * page_size, group = nq / nkv, head_tiles = (group + kHeads - 1) / kHeads;
  const int64_t blocks = B * nkv * head_tiles;
  const int64_t chunks = weights_in ? (cap + kJoinSlots - 1) / kJoinSlots : 0;
  const int splits = paged_splits(blocks, cap);
  if (B * nq > INT32_MAX / 1024 || blocks * splits > max_blocks(64 * kWaves) ||
      B * (nkv * chunks + nq) > max_blocks(kJoinThreads))
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (!q || !k_pages || !v_pages || !table || !lengths || !out) return fail(CDX_EINVAL, "%s: null pointer", name);
  const PagedWork ws = paged_work(B, nq, hd, cap, splits, weights_in != nullptr);
  if (work_bytes < ws.total || (ws.total > 0 && !work))
    return fail(CDX_EWORKSPACE, "%s: workspace needs %zu bytes, got %zu", name, ws.total, work ? work_bytes : 0);
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) || !aligned16(work))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  p.q = q;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  p.lengths = lengths;
  p.B = (int32_t)B;
  p.nq = nq;
  p.nkv = nkv;
  p.D = hd;
  p.group = (int32_t)group;
  p.head_tiles = (int32_t)head_tiles;
  p.splits = splits;
  p.scale_log2 = scale * kLog2e;
  p.out = out;
  char* at = static_cast<char*>(work);
  p.part_o = reinterpret_cast<float*>(at);
  p.part_ml = reinterpret_cast<float2*>(at + ws.o);
  p.scores = weights_in ? reinterpret_cast<float*>(at + ws.o + ws.ml) : nullptr;
  p.w_in = weights_in;
  p.w_out = weights_out;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(blocks * splits)), block(64 * kWaves);
  if (hd <= 32)
    paged_attn_kernel<1, 4, kWaves, false><<<grid, block, 0, s>>>(p);
  else if (hd < 64)
    paged_attn_kernel<2, 4, kWaves, false><<<grid, block, 0, s>>>(p);
  else if (hd == 64)
    paged_attn_kernel<2, 4, kWaves, true><<<grid, block, 0, s>>>(p);
  else if (hd <= 96)
    paged_attn_kernel<3, 8, kWaves, false><<<grid, block, 0, s>>>(p);
  else if (hd < 128)
    paged_attn_kernel<4, 8, kWaves, false><<<grid, block, 0, s>>>(p);
  else
    paged_attn_kernel<4, 8, kWaves, true><<<grid, block, 0, s>>>(p);
  if (int rc = check_launch(name)) return rc;
  if (splits == 1 && !weights_in) return CDX_OK;
  const int64_t rows = splits > 1 ? B * nq : 0;
  paged_join_kernel<<<dim3((unsigned)(rows + B * nkv * chunks)), dim3(kJoinThreads), 0, s>>>(
      p, (uint32_t)rows, (int)std::max<int64_t>(chunks, 1));
  return check_launch(name);
}
