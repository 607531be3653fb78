// The paged KV cache for gfx950: the append of a step's heads, the write of prompts, and the
// eviction of a bounded cache by accumulated attention weight.
//
// The pages hold rows of D bf16 values, [pages][nkv][page size][D], so that one head's slots of
// a page are one contiguous piece; every kernel here moves whole rows in pieces of 8 or 16
// bytes per lane and is bound by memory, or for a step's few rows by its launch.
//
// Measured (us of a kernel): append of 256 tokens, 16/8 heads of 128, 3.3 (one token of 8/4 heads of
// 40: 2.2); write of 8 prompts of up to 2048 tokens (67 MB read and written) 12.9, 5.2 TB/s, where the
// plainest copy of 64 MB moves 5.3 (of 512 MB 6.2); eviction of one slot a head, 12 layers x 4 x 1025
// slots, 7.8 + 3.4, of half a prompt, 24 layers x 8 x up to 2048 slots of 8 x 128, 18.6 + 67 (292 MB of
// rows read and written, 4.4 TB/s).
//
//   paged_append_kernel   the packed projection of one new token per sequence, read once: per-head
//                         RMSNorm, RoPE at the sequence's own position, q out, k and v into the
//                         sequence's last slot.  16 lanes hold one head (lane i columns 4 i ..
//                         4 i + 3 of each half, so both elements of every RoPE pair).
//   paged_write_kernel    prompts' k and v [B][nkv][S][D] to slots 0 .. length - 1: 16 bytes per
//                         lane, K and V by the same lane.
//   evict_select_kernel   one block per (layer, sequence, head): the slots to keep by a radix
//                         descent over (recent, weight), then the pairs (hole, mover) in slot
//                         order.  Holes lie below `keep` and movers at or above it, so that the
//                         moves read and write disjoint rows and run in any order; one slot a
//                         head costs one row's move, where a cache kept in order would shift
//                         half of its rows.
//   evict_move_kernel     the rows of those pairs, 16 bytes per lane.
#include "cdx_paged.h"
#include "cdx_skinny.h"
#include "cdx_wave.h"

namespace cdx {

int paged_table(const char* name, const int32_t* table, int64_t table_ld, int64_t width, int64_t num_pages,
                int32_t page_size, int64_t B, int32_t nkv, int32_t hd, PagedTable* t) {
  if (B < 0 || nkv <= 0 || width < 0 || num_pages < 0)
    return fail(CDX_EINVAL, "%s: bad shape B=%lld nkv=%d table width=%lld pages=%lld", name, (long long)B, nkv,
                (long long)width, (long long)num_pages);
  if (hd <= 0 || hd > 128 || hd % 8 != 0)
    return fail(CDX_EUNSUPPORTED, "%s: head dim %d must be a multiple of 8 and <= 128", name, hd);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return fail(CDX_EUNSUPPORTED, "%s: page size %d must be 16, 32, 64, 128 or 256", name, page_size);
  if (table_ld < width) return fail(CDX_EINVAL, "%s: block table stride too small", name);
  if (width > (INT32_MAX - 4096) / page_size || num_pages > INT32_MAX || B > INT32_MAX / 1024 ||
      nkv > 65535 || B * nkv > INT32_MAX / 1024)
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  t->table = table;
  t->ld = table_ld;
  t->width = (int32_t)width;
  t->num_pages = (int32_t)num_pages;
  t->log2_page = __builtin_ctz((unsigned)page_size);
  return CDX_OK;
}

namespace {

struct AppendParams {
  const void* qkv;  // [B] rows of (nq + 2 nkv) D at stride ld, fp32 or bf16
  int64_t ld;
  int32_t B, nq, nkv, D;
  const uint16_t* q_norm_w;  // [D], nullptr = no QK norm
  const uint16_t* k_norm_w;
  float eps;
  const float* cos_sin;  // [n_pos][D / 2][2]
  int64_t n_pos;
  const int32_t* lengths;    // slots in use, the new token's included
  const int32_t* positions;  // rotary positions of the new tokens
  PagedTable t;
  uint16_t* k_pages;
  uint16_t* v_pages;
  uint16_t* q;  // [B][nq][D]
};

template <typename TIn>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendParams p) {
  const int g16 = threadIdx.x & 15;
  const int heads = p.nq + 2 * p.nkv;
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), rows = (int64_t)p.B * heads;
  const int half = p.D >> 1;
  // Lanes past the head (and groups past the last row) take part in the row sums with zeros
  // and store nothing.
  const bool on = row < rows && 4 * g16 < half;
  const int64_t rr = row < rows ? row : rows - 1;
  const int64_t b = rr / heads;
  const int head = (int)(rr - b * heads);
  const int kind = head < p.nq ? 0 : (head < p.nq + p.nkv ? 1 : 2);
  const int h = kind == 0 ? head : (kind == 1 ? head - p.nq : head - p.nq - p.nkv);
  const int c = on ? 4 * g16 : 0;

  const TIn* src = static_cast<const TIn*>(p.qkv) + b * p.ld + (int64_t)head * p.D + c;
  const uint16_t* nw = kind == 1 ? p.k_norm_w : p.q_norm_w;
  const int32_t pos = p.positions[b], slot = p.lengths[b] - 1;
  // A position outside the table has no angle: the head is NaN, as far as it is rotated.
  const bool known = (uint32_t)pos < (uint64_t)p.n_pos;
  const float* cs = p.cos_sin + ((int64_t)(known ? pos : 0) * half + c) * 2;
  float x1[4], x2[4], t[8], w1[4] = {1.f, 1.f, 1.f, 1.f}, w2[4] = {1.f, 1.f, 1.f, 1.f};
  head_load4(src, x1);
  head_load4(src + half, x2);
  head_load4(cs, t);
  head_load4(cs + 4, t + 4);
  if (nw != nullptr) {
    head_load4(nw + c, w1);
    head_load4(nw + c + half, w2);
  }
  if (kind != 2) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(x1[j], x1[j], __builtin_fmaf(x2[j], x2[j], ss));
    const float rs = rsqrtf(head16_sum(on ? ss : 0.f) / (float)p.D + p.eps);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x1[j] = nw != nullptr ? w1[j] * (x1[j] * rs) : x1[j];
      x2[j] = nw != nullptr ? w2[j] * (x2[j] * rs) : x2[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = x1[j], z = x2[j];
      x1[j] = known ? __builtin_fmaf(a, t[2 * j], -(z * t[2 * j + 1])) : __builtin_nanf("");
      x2[j] = known ? __builtin_fmaf(z, t[2 * j], a * t[2 * j + 1]) : __builtin_nanf("");
    }
  }
  if (!on) return;
  uint16_t* dst;
  if (kind == 0) {
    dst = p.q + (b * p.nq + h) * p.D + c;
  } else {
    if (slot < 0 || slot >= p.t.capacity()) return;
    const int64_t r = p.t.row(b, h, p.nkv, slot);
    if (r < 0) return;
    dst = (kind == 1 ? p.k_pages : p.v_pages) + r * p.D + c;
  }
  head_store4(dst, x1);
  head_store4(dst + half, x2);
}

constexpr int kWritePieces = 4;  // 16-byte pieces of K, and of V, that a lane moves

__global__ __launch_bounds__(256) void paged_write_kernel(const uint4* __restrict__ k, const uint4* __restrict__ v,
                                                          int S, int D, int nkv, const int32_t* __restrict__ lengths,
                                                          PagedTable t, uint32_t blocks, uint4* k_pages,
                                                          uint4* v_pages) {
  const uint32_t slab = blockIdx.x / blocks;  // (b, h)
  const int64_t b = slab / nkv;
  const int h = slab - (uint32_t)b * nkv, cpr = D / 8;
  const int valid = min(min(lengths[b], S), t.capacity());
  const int64_t n = (int64_t)max(valid, 0) * cpr;
  const int64_t i0 = (int64_t)(blockIdx.x - slab * blocks) * (256 * kWritePieces) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kWritePieces; ++u) {
    const int64_t i = i0 + u * 256;
    if (i >= n) return;
    const int32_t s = (int32_t)(i / cpr);
    const int64_t r = t.row(b, h, nkv, s);
    if (r < 0) continue;
    const int64_t from = (int64_t)slab * S * cpr + i, to = r * cpr + (i - (int64_t)s * cpr);
    const uint4 a = k[from], c = v[from];
    k_pages[to] = a;
    v_pages[to] = c;
  }
}

// ---- eviction ---------------------------------------------------------------

constexpr int kSelectThreads = 512;

struct EvictParams {
  int32_t B, nkv, D, cap, keep, recent, max_moves;
  int64_t row0;                // of layers x B x nkv rows, the launch's first
  const int32_t* lengths;      // [B]
  const int32_t* positions;    // [B], of the newest tokens
  const float* weights;        // [rows][cap]
  const int32_t* slot_pos;     // [rows][cap]
  int32_t* new_lengths;        // [B]
  float* new_weights;          // [rows][cap]
  int32_t* new_pos;            // [rows][cap]
  int32_t* count;              // [rows]
  int32_t* moves;              // [rows][2][max_moves]: holes, movers
  PagedTable t;
  int64_t layer_rows;          // rows of one layer's pool: pages x nkv x page size
  uint16_t* k_pages;
  uint16_t* v_pages;
};

// Order of weights as unsigned integers: -0 = +0, NaN below everything as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.f) w = 0.f;
  const uint32_t u = __float_as_uint(w);
  return u == 0x80000000u ? 0x80000000u : (u & 0x80000000u ? ~u : u | 0x80000000u);
}

// Exclusive sum over the block of a count per thread, and the block's total.
__device__ __forceinline__ int block_exclusive(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_inclusive(v);
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 64; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  return before + x - v;
}

// PER: slots that a thread holds in registers (capacity <= 512 PER), or 0: every pass reads them (24
// layers x 8 x 2048 slots: held 18.6 us, read again 24.3; 12 x 4 x 1088: 7.8, 10.0).
template <int PER>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
  __shared__ int hist[4][256];  // of each digit
  __shared__ int sums[kSelectThreads / 64];
  __shared__ int pick[2];
  const int64_t row = p.row0 + blockIdx.x;
  const int b = (int)(row / p.nkv % p.B);
  const int tid = threadIdx.x;
  const int len = max(0, min(p.lengths[b], p.cap));
  const float* w = p.weights + row * p.cap;
  const int32_t* sp = p.slot_pos + row * p.cap;
  float* nw = p.new_weights + row * p.cap;
  int32_t* np = p.new_pos + row * p.cap;
  if (row < (int64_t)p.B * p.nkv && row % p.nkv == 0 && tid == 0) p.new_lengths[b] = min(len, p.keep);
  if (len <= p.keep) {
    for (int i = tid; i < p.cap; i += kSelectThreads) {
      nw[i] = i < len ? w[i] : 0.f;
      np[i] = i < len ? sp[i] : -1;
    }
    if (tid == 0) p.count[row] = 0;
    return;
  }
  const int64_t first_recent = (int64_t)p.positions[b] - p.recent + 1;
  for (int i = tid; i < 4 * 256; i += kSelectThreads) hist[i >> 8][i & 255] = 0;

  uint32_t key[PER > 0 ? PER : 1];
  uint32_t recent_bits = 0;
  if constexpr (PER > 0) {
    float wv[PER];
    int32_t sv[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = u * kSelectThreads + tid;
      wv[u] = i < len ? w[i] : 0.f;
      sv[u] = i < len ? sp[i] : 0;
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      key[u] = weight_key(wv[u]);
      recent_bits |= (int64_t)sv[u] >= first_recent ? 1u << u : 0u;
    }
  }
  // f(slot, key, recent) of every slot in use, the block's 512 threads on neighbouring ones.
  auto each = [&](auto f) {
    if constexpr (PER > 0) {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int i = u * kSelectThreads + tid;
        if (i < len) f(i, key[u], (recent_bits >> u & 1) != 0);
      }
    } else {
      for (int i = tid; i < len; i += kSelectThreads) f(i, weight_key(w[i]), (int64_t)sp[i] >= first_recent);
    }
  };

  // The recent tokens are kept before any other.
  int mine = 0, n_recent;
  each([&](int, uint32_t, bool recent) { mine += recent ? 1 : 0; });
  block_exclusive(mine, sums, n_recent);
  const bool among_recent = n_recent > p.keep;  // (positions given twice: the tokens then rank by weight)
  int need = among_recent ? p.keep : p.keep - n_recent;
  // The need-th largest weight of the class: its bits from the highest byte down.
  uint32_t prefix = 0;
  int shift = 32;
  bool all = need == 0;  // no ties to count: the keys above `prefix` are kept, or all at it
  while (shift > 0 && !all) {
    shift -= 8;
    int* counts = hist[shift >> 3];  // (cleared before the sum over the block above)
    each([&](int, uint32_t k, bool recent) {
      const bool in = recent == among_recent && (shift == 24 || k >> (shift + 8) == prefix);
      if (in) atomicAdd(&counts[(k >> shift) & 255], 1);
    });
    __syncthreads();
    if (tid < 64) {
      // The digit from above at which the counts reach `need`: four to a lane.
      int n[4], lane_sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) lane_sum += n[i] = counts[255 - 4 * tid - i];
      int above = wave_inclusive(lane_sum) - lane_sum;
      if (above < need && above + lane_sum >= need) {  // (one lane)
        int i = 0;
        while (i < 3 && above + n[i] < need) above += n[i++];
        pick[0] = 255 - 4 * tid - i;
        pick[1] = above;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)pick[0];
    need -= pick[1];
    all = counts[pick[0]] == need;
  }
  const bool none = need == 0;  // (nothing of the class is kept)

  // In slot order: which slots stay, which of them are holes and which move.
  int32_t* holes = p.moves + row * 2 * p.max_moves;
  int32_t* movers = holes + p.max_moves;
  int ties = 0, n_holes = 0, n_movers = 0;
  auto order = [&](int i, uint32_t k, bool recent) {
    bool kept = false, tie = false;
    if (i < len) {
      kept = recent != among_recent ? recent : !none && k >> (shift & 31) > prefix;
      tie = recent == among_recent && !none && k >> (shift & 31) == prefix;
    }
    int total, before = 0;
    if (!all) {  // (else every tie is kept)
      before = block_exclusive(tie ? 1 : 0, sums, total);
      tie = tie && ties + before < need;
      ties += total;
    }
    kept = kept || tie;
    const bool hole = i < len && i < p.keep && !kept, mover = i >= p.keep && kept;
    // (Both counts in one word: at most 512 of each.)
    const int both = block_exclusive((hole ? 1 : 0) | (mover ? 1 << 16 : 0), sums, total);
    if (hole) holes[n_holes + (both & 0xffff)] = i;
    if (mover) movers[n_movers + (both >> 16)] = i;
    n_holes += total & 0xffff;
    n_movers += total >> 16;
    if (i < p.cap && !hole) {
      nw[i] = i < p.keep ? w[i] : 0.f;
      np[i] = i < p.keep ? sp[i] : -1;
    }
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (u * kSelectThreads < p.cap) order(u * kSelectThreads + tid, key[u], (recent_bits >> u & 1) != 0);
  } else {
    for (int base = 0; base < p.cap; base += kSelectThreads) {
      const int i = base + tid;
      order(i, i < len ? weight_key(w[i]) : 0u, i < len && (int64_t)sp[i] >= first_recent);
    }
  }
  __syncthreads();  // the lists are whole, and this block's own stores are seen by all of it
  if (tid == 0) p.count[row] = n_holes;
  // (n_holes == n_movers: keep slots are kept, and every hole below `keep` stands for one at or above it.)
  for (int i = tid; i < n_holes; i += kSelectThreads) {
    nw[holes[i]] = w[movers[i]];
    np[holes[i]] = sp[movers[i]];
  }
}

constexpr int kMoveBlock = 16;  // rows that a block moves, of K and of V: one per 16 lanes

// One row a group: 62 us, when it was tried, for 24 layers x 8 sequences of up to 2048 slots of 8 x 128
// values (292 MB read and written); two, four and eight rows, all loaded before the first is stored,
// 99, 95, 107.
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictParams p, uint32_t blocks) {
  const uint32_t r = blockIdx.x / blocks;
  const int64_t row = p.row0 + r;
  const int n = p.count[row], c = threadIdx.x & 15, cpr = p.D / 8;
  const int m = (int)(blockIdx.x - r * blocks) * kMoveBlock + (threadIdx.x >> 4);
  if (m >= n || c >= cpr) return;
  const int h = (int)(row % p.nkv);
  const int64_t slab = row / p.nkv, b = slab % p.B, layer = slab / p.B;
  const int32_t* holes = p.moves + row * 2 * p.max_moves;
  const int64_t to = p.t.row(b, h, p.nkv, holes[m]), from = p.t.row(b, h, p.nkv, holes[p.max_moves + m]);
  if (to < 0 || from < 0) return;
  uint4* k = reinterpret_cast<uint4*>(p.k_pages) + layer * p.layer_rows * cpr + c;
  uint4* v = reinterpret_cast<uint4*>(p.v_pages) + layer * p.layer_rows * cpr + c;
  const uint4 x = k[from * cpr], y = v[from * cpr];
  k[to * cpr] = x;
  v[to * cpr] = y;
}

}  // namespace
}  // namespace cdx

extern "C" int cdx_paged_append_fwd(const void* qkv, int32_t qkv_fp32, int64_t ldqkv, int64_t B, int32_t nq,
                                    int32_t nkv, int32_t hd, const uint16_t* q_norm_w, const uint16_t* k_norm_w,
                                    float eps, const float* cos_sin, int64_t n_pos, const int32_t* lengths,
                                    const int32_t* positions, const int32_t* table, int64_t table_ld, int64_t width,
                                    int64_t num_pages, int32_t page_size, uint16_t* k_pages, uint16_t* v_pages,
                                    uint16_t* q_out, void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_append_fwd";
  clear_error();
  AppendParams p{};
  if (int rc = paged_table(name, table, table_ld, width, num_pages, page_size, B, nkv, hd, &p.t)) return rc;
  if (nq <= 0 || nq % nkv != 0 || n_pos < 0)
    return fail(CDX_EINVAL, "%s: bad shape nq=%d nkv=%d n_pos=%lld", name, nq, nkv, (long long)n_pos);
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(CDX_EINVAL, "%s: q and k norm weights must both be given or both be NULL", name);
  if (!(eps >= 0.f)) return fail(CDX_EINVAL, "%s: eps must be >= 0", name);
  const int64_t heads = (int64_t)nq + 2 * (int64_t)nkv;
  if (ldqkv < heads * hd) return fail(CDX_EINVAL, "%s: leading dimension too small", name);
  if (ldqkv % 8) return fail(CDX_EUNSUPPORTED, "%s: leading dimensions must be multiples of 8", name);
  if (heads > 65535 || B * heads > INT32_MAX) return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (B == 0) return CDX_OK;
  if (n_pos == 0) return fail(CDX_EINVAL, "%s: empty cos/sin table", name);
  if (!qkv || !cos_sin || !lengths || !positions || !q_out ||
      (width > 0 && (!table || (num_pages > 0 && (!k_pages || !v_pages)))))
    return fail(CDX_EINVAL, "%s: null pointer", name);
  if (!aligned16(qkv) || !aligned16(cos_sin) || !aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(q_norm_w) || !aligned16(k_norm_w))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  p.ld = ldqkv;
  p.nq = nq;
  p.nkv = nkv;
  p.D = hd;
  p.q_norm_w = q_norm_w;
  p.k_norm_w = k_norm_w;
  p.eps = eps;
  p.cos_sin = cos_sin;
  p.n_pos = n_pos;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t per = max_blocks(256) * 16 / heads;  // sequences of one launch
  for (int64_t b0 = 0; b0 < B; b0 += per) {
    const int64_t n = B - b0 < per ? B - b0 : per;
    p.B = (int32_t)n;
    p.qkv = static_cast<const char*>(qkv) + b0 * ldqkv * (qkv_fp32 ? 4 : 2);
    p.lengths = lengths + b0;
    p.positions = positions + b0;
    p.t.table = table ? table + b0 * table_ld : nullptr;
    p.q = q_out + b0 * nq * hd;
    const dim3 grid((unsigned)((n * heads + 15) / 16));
    if (qkv_fp32)
      paged_append_kernel<float><<<grid, dim3(256), 0, s>>>(p);
    else
      paged_append_kernel<uint16_t><<<grid, dim3(256), 0, s>>>(p);
    if (int rc = check_launch(name)) return rc;
  }
  return CDX_OK;
}

extern "C" int cdx_qkv_paged_fwd(const uint16_t* x, int64_t ldx, const uint16_t* x_norm_w, float x_eps,
                                 const uint16_t* mu, int64_t ldmu, const uint16_t* w, const uint16_t* w_mu,
                                 int64_t ldw, int64_t B, int32_t H, int32_t nq, int32_t nkv, int32_t hd,
                                 const uint16_t* q_norm_w, const uint16_t* k_norm_w, float eps, const float* cos_sin,
                                 int64_t n_pos, const int32_t* lengths, const int32_t* positions,
                                 const int32_t* table, int64_t table_ld, int64_t width, int64_t num_pages,
                                 int32_t page_size, uint16_t* k_pages, uint16_t* v_pages, uint16_t* q_out, void* work,
                                 size_t work_bytes, void* stream) {
  using namespace cdx;
  const char* name = "cdx_qkv_paged_fwd";
  clear_error();
  PagedTable t{};
  if (int rc = paged_table(name, table, table_ld, width, num_pages, page_size, B, nkv, hd, &t)) return rc;
  if (H <= 0 || nq <= 0 || nq % nkv != 0) return fail(CDX_EINVAL, "%s: bad shape H=%d nq=%d nkv=%d", name, H, nq, nkv);
  if (H % 64 != 0) return fail(CDX_EUNSUPPORTED, "%s: H=%d must be a multiple of 64", name, H);
  if (x_norm_w && !(x_eps >= 0.f)) return fail(CDX_EINVAL, "%s: eps must be >= 0", name);
  if (ldx < H || ldw < H || (mu && ldmu != 0 && ldmu < H))
    return fail(CDX_EINVAL, "%s: leading dimension too small", name);
  if (ldx % 8 || ldw % 8 || (mu && ldmu % 8))
    return fail(CDX_EUNSUPPORTED, "%s: leading dimensions must be multiples of 8", name);
  const int64_t N = ((int64_t)nq + 2 * (int64_t)nkv) * hd;
  if (N > INT32_MAX) return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (B == 0) return CDX_OK;
  if (!x || !w || (mu && !w_mu) || !work) return fail(CDX_EINVAL, "%s: null pointer", name);
  if (!aligned16(x) || !aligned16(w) || (mu && (!aligned16(mu) || !aligned16(w_mu))) || !aligned16(work) ||
      !aligned16(x_norm_w))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  const bool few = skinny_fits(B, N);
  if (x_norm_w && (!few || B > kNormRows))
    return fail(CDX_EUNSUPPORTED, "%s: a folded norm needs B <= %d", name, kNormRows);
  const size_t need = cdx_qkv_cache_workspace_bytes(B, 1, nq, nkv, hd);
  if (work_bytes < need)
    return fail(CDX_EWORKSPACE, "%s: workspace needs %zu bytes, got %zu", name, need, work_bytes);
  if (!cos_sin || !lengths || !positions || !q_out || !table || !k_pages || !v_pages || n_pos <= 0 || !(eps >= 0.f) ||
      (q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(CDX_EINVAL, "%s: null pointer, empty cos/sin table, bad eps or one QK norm weight only", name);
  if (!aligned16(cos_sin) || !aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(q_norm_w) ||
      !aligned16(k_norm_w))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  if (few) {
    SkinnyParams sp{};
    sp.a = x;
    sp.lda = ldx;
    sp.a2 = mu ? mu : x;
    sp.lda2 = mu ? ldmu : ldx;
    sp.b = w;
    sp.b2 = mu ? w_mu : w;
    sp.ldb = ldw;
    sp.k_split = H;
    sp.M = (int32_t)B;
    sp.N = (int32_t)N;
    sp.K = mu ? 2 * H : H;
    sp.c = work;
    sp.ldc = N;
    sp.norm_w = x_norm_w;
    sp.eps = x_eps;
    if (int rc = skinny_gemm(sp, SkinnyEpi::kF32, reinterpret_cast<hipStream_t>(stream), name)) return rc;
  } else if (int rc = cdx_mu_qkv_fwd(x, ldx, mu, ldmu, w, w_mu, ldw, B, H, (int32_t)N, static_cast<uint16_t*>(work), N,
                                     stream)) {
    return rc;
  }
  return cdx_paged_append_fwd(work, few, N, B, nq, nkv, hd, q_norm_w, k_norm_w, eps, cos_sin, n_pos, lengths, positions,
                              table, table_ld, width, num_pages, page_size, k_pages, v_pages, q_out, stream);
}

extern "C" int cdx_paged_write(const uint16_t* k, const uint16_t* v, int64_t B, int32_t nkv, int64_t S, int32_t hd,
                               const int32_t* lengths, const int32_t* table, int64_t table_ld, int64_t width,
                               int64_t num_pages, int32_t page_size, uint16_t* k_pages, uint16_t* v_pages,
                               void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_write";
  clear_error();
  PagedTable t{};
  if (int rc = paged_table(name, table, table_ld, width, num_pages, page_size, B, nkv, hd, &t)) return rc;
  if (S < 0) return fail(CDX_EINVAL, "%s: bad shape S=%lld", name, (long long)S);
  if (B == 0 || S == 0 || width == 0 || num_pages == 0) return CDX_OK;
  const int64_t pieces = S * (hd / 8), blocks = (pieces + 256 * kWritePieces - 1) / (256 * kWritePieces);
  if (S > INT32_MAX || B * nkv * blocks > max_blocks(256)) return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (!k || !v || !lengths || !table || !k_pages || !v_pages) return fail(CDX_EINVAL, "%s: null pointer", name);
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  paged_write_kernel<<<dim3((unsigned)(B * nkv * blocks)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      reinterpret_cast<const uint4*>(k), reinterpret_cast<const uint4*>(v), (int)S, hd, nkv, lengths, t,
      (uint32_t)blocks, reinterpret_cast<uint4*>(k_pages), reinterpret_cast<uint4*>(v_pages));
  return check_launch(name);
}

namespace {
// The longest list of moves of one head: as many holes as there are slots past `keep`.
inline int64_t evict_max_moves(int64_t cap, int64_t keep) {
  return cap > keep ? (cap - keep < keep ? cap - keep : keep) : 0;
}
}  // namespace

extern "C" size_t cdx_paged_evict_workspace_bytes(int64_t layers, int64_t B, int32_t nkv, int64_t capacity,
                                                  int64_t keep) {
  if (layers <= 0 || B <= 0 || nkv <= 0 || capacity <= 0 || keep <= 0) return 0;
  return (size_t)(layers * B * nkv) * (1 + 2 * (size_t)evict_max_moves(capacity, keep)) * sizeof(int32_t);
}

extern "C" int cdx_paged_evict(int64_t layers, int64_t B, int32_t nkv, int32_t hd, const int32_t* lengths,
                               const int32_t* positions, const int32_t* table, int64_t table_ld, int64_t width,
                               int64_t num_pages, int32_t page_size, uint16_t* k_pages, uint16_t* v_pages,
                               const float* weights, const int32_t* slot_positions, int64_t keep, int64_t recent,
                               int32_t* new_lengths, float* new_weights, int32_t* new_slot_positions, void* work,
                               size_t work_bytes, void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_evict";
  clear_error();
  EvictParams p{};
  if (int rc = paged_table(name, table, table_ld, width, num_pages, page_size, B, nkv, hd, &p.t)) return rc;
  if (layers < 0) return fail(CDX_EINVAL, "%s: bad layer count %lld", name, (long long)layers);
  if (keep <= 0 || recent < 0 || recent > keep)
    return fail(CDX_EINVAL, "%s: keep=%lld must be positive and recent=%lld lie in 0 .. keep", name, (long long)keep,
                (long long)recent);
  if (layers == 0 || B == 0 || width == 0 || num_pages == 0) return CDX_OK;
  const int64_t cap = width * page_size, rows = layers * B * nkv, moves = evict_max_moves(cap, keep);
  const int64_t blocks = (moves + kMoveBlock - 1) / kMoveBlock;
  if (layers > 65535 || rows > INT32_MAX || blocks > max_blocks(256))
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (!lengths || !positions || !table || !k_pages || !v_pages || !weights || !slot_positions || !new_lengths ||
      !new_weights || !new_slot_positions || !work)
    return fail(CDX_EINVAL, "%s: null pointer", name);
  if (new_weights == weights || new_slot_positions == slot_positions || new_lengths == lengths)
    return fail(CDX_EINVAL, "%s: the new weights, positions and lengths need memory of their own", name);
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(work))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  const size_t need = cdx_paged_evict_workspace_bytes(layers, B, nkv, cap, keep);
  if (work_bytes < need)
    return fail(CDX_EWORKSPACE, "%s: workspace needs %zu bytes, got %zu", name, need, work_bytes);
  p.B = (int32_t)B;
  p.nkv = nkv;
  p.D = hd;
  p.cap = (int32_t)cap;
  p.keep = (int32_t)(keep < cap ? keep : cap);
  p.recent = (int32_t)(recent < INT32_MAX ? recent : INT32_MAX);
  p.max_moves = (int32_t)moves;
  p.lengths = lengths;
  p.positions = positions;
  p.weights = weights;
  p.slot_pos = slot_positions;
  p.new_lengths = new_lengths;
  p.new_weights = new_weights;
  p.new_pos = new_slot_positions;
  p.count = static_cast<int32_t*>(work);
  p.moves = p.count + rows;
  p.layer_rows = num_pages * nkv * page_size;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t select = max_blocks(kSelectThreads);
  for (p.row0 = 0; p.row0 < rows; p.row0 += select) {
    const dim3 grid((unsigned)(rows - p.row0 < select ? rows - p.row0 : select)), block(kSelectThreads);
    if (cap <= 4 * kSelectThreads)
      evict_select_kernel<4><<<grid, block, 0, s>>>(p);
    else if (cap <= 16 * kSelectThreads)
      evict_select_kernel<16><<<grid, block, 0, s>>>(p);
    else
      evict_select_kernel<0><<<grid, block, 0, s>>>(p);
    if (int rc = check_launch(name)) return rc;
  }
  if (blocks == 0) return CDX_OK;
  const int64_t per = max_blocks(256) / blocks;
  for (p.row0 = 0; p.row0 < rows; p.row0 += per) {
    const int64_t n = rows - p.row0 < per ? rows - p.row0 : per;
    evict_move_kernel<<<dim3((unsigned)(n * blocks)), dim3(256), 0, s>>>(p, (uint32_t)blocks);
    if (int rc = check_launch(name)) return rc;
  }
  return CDX_OK;
}
