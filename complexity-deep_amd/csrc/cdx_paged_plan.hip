// Pages and rows of a call that brings any number of new tokens per sequence, for gfx950: the pages
// that the tokens need from a pool that the sequences share, the map from the call's rows to slots,
// the pages' way back, and the append of the rows themselves.
//
//   reserve_kernel   need_b = ceil((len + n) / page) - ceil(len / page) pages for n tokens more; sequence
//                    b has the pages free - 1 - (need_0 + .. + need_(b-1)) downwards of the list, if the
//                    needs up to its own are there.  Nothing that a block reads is written by another
//                    (the lists and counts that a call changes come out beside the old ones; a new
//                    page's table entry is written by the row in its first slot, and read by
//                    nobody), so that one launch without any wait between blocks does: every block sums
//                    up the needs itself, 512 sequences at a time, and maps 512 rows.
//   truncate_kernel  the pages past ceil(new length / page), put on the list so that the ones that
//                    reserve took last come off it first: reserve and truncate undo each other.
//   chunk_append_kernel  per row of the packed projection: per-head RMSNorm, RoPE, q out, k and v into the
//                    row's slot; 16 lanes a head, as paged_append_kernel.
//
// Measured (us of a kernel): reserve 3.1 for one sequence, 4.6 for 256 with 8432 rows or 64 with 131072 (launch and
// two rounds of loads); truncate 2.9 for 256 sequences, 5.2 for 1024 that give 32000 pages back; append of 8192
// rows of 16/8 heads of 128 25 (134 MB read and written, 5.4 TB/s, a plain copy's rate), of 5 rows 2.9.  Two heads a
// group of lanes, loaded together, took as long.  Narrower heads leave lanes of their 16 without dims: 8192 rows of
// 16/4 heads of 80 17 (63 MB: 3.7 TB/s), 12/4 of 64 14 (42 MB: 3.0), 8/4 of 40 12 (21 MB: 1.8).
#include "cdx_paged.h"
#include "cdx_wave.h"

namespace cdx {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanRows = kPlanThreads;  // rows that a block maps

typedef long long i64;

// Sums over the block of a value per thread: those before this thread's, and the whole.
__device__ __forceinline__ i64 block_before(i64 v, i64* lds, i64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const i64 x = (i64)wave_inclusive((u64)v);
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  i64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  return before + x - v;
}

// The last of n ascending values that is <= x (0 if none is).
template <typename T>
__device__ __forceinline__ int last_at_most(const T* values, int n, T x) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (values[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
}

// Arrays of a call on the host's side.
struct Extent {
  const void* at;
  int64_t bytes;
};
// Whether any result lies over an array that blocks still read while another one writes results.
template <size_t NIn, size_t NOut>
bool overlap(const Extent (&in)[NIn], const Extent (&out)[NOut]) {
  for (const Extent& o : out)
    for (const Extent& i : in) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(o.at), b = reinterpret_cast<uintptr_t>(i.at);
      if (o.at && i.at && o.bytes > 0 && a < b + (uintptr_t)i.bytes && b < a + (uintptr_t)o.bytes) return true;
    }
  return false;
}

struct ReserveParams {
  const int32_t* counts;     // [B]
  const int32_t* lengths;    // [B]
  const int32_t* positions;  // [B], of the newest tokens
  int32_t B, stride, rows;   // stride 0: rows one behind the other
  int32_t* table;
  int64_t ld;
  int32_t width, log2_page;
  const int32_t* free_pages;  // [free_cap], or nullptr: no pages are needed
  int32_t free_cap;
  const int32_t* free_count;
  int32_t* starts;
  int32_t* counts_out;
  int32_t* lengths_out;
  int32_t* positions_out;
  int32_t* free_out;
  int64_t* row_slots;
  int32_t* row_positions;
};

__global__ __launch_bounds__(kPlanThreads) void reserve_kernel(const ReserveParams p) {
  __shared__ i64 sums[kPlanThreads / 64];
  __shared__ int32_t s_start[kPlanThreads], s_count[kPlanThreads], s_len[kPlanThreads], s_pos[kPlanThreads];
  __shared__ i64 s_taken[kPlanThreads];
  const int tid = threadIdx.x;
  const int lp = p.log2_page, page_mask = (1 << lp) - 1;
  const bool pool = p.free_pages != nullptr;
  const i64 cap = (i64)p.width << lp;
  const i64 free = pool ? min(max(*p.free_count, 0), p.free_cap) : 0;
  const int64_t r_begin = (int64_t)blockIdx.x * kPlanRows;
  const int32_t r_end = (int32_t)min(r_begin + kPlanRows, (int64_t)p.rows);

  i64 rows_before = 0, need_before = 0, taken = 0;
  for (int32_t b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int n_seq = min(kPlanThreads, p.B - b0);
    const int32_t b = b0 + tid;
    const bool on = tid < n_seq;
    const int32_t asked = on ? max(p.counts[b], 0) : 0, given = on ? p.lengths[b] : 0, pos = on ? p.positions[b] : 0;
    const i64 len = max(given, 0);
    i64 rows, needs;
    i64 start = rows_before + block_before(asked, sums, rows);
    if (p.stride) start = (i64)b * p.stride;
    const bool fits = start + asked <= p.rows && len + asked <= cap && (!p.stride || asked <= p.stride);
    const i64 need = pool && fits ? ((len + asked + page_mask) >> lp) - ((len + page_mask) >> lp) : 0;
    const i64 need_at = need_before + block_before(need, sums, needs);
    const bool ok = fits && (need == 0 || need_at + need <= free);
    const int32_t count = ok ? asked : 0;
    const int32_t from = (int32_t)min(start, (i64)p.rows);
    i64 got;
    block_before(ok ? need : 0, sums, got);  // (its barriers also part the last round's reads from these writes)
    s_start[tid] = from;
    s_count[tid] = count;
    s_len[tid] = (int32_t)len;
    s_pos[tid] = pos;
    s_taken[tid] = need_at;
    if (on && blockIdx.x == 0) {
      p.starts[b] = from;
      p.counts_out[b] = count;
      p.lengths_out[b] = count > 0 ? (int32_t)len + count : given;
      p.positions_out[b] = pos + count;
    }
    __syncthreads();
    rows_before += rows;
    need_before += needs;
    taken += got;
    // This block's rows among those of the 512 sequences; the last ones' reach to the end.
    const bool last = b0 + kPlanThreads >= p.B;
    const i64 next = last ? p.rows : (p.stride ? (i64)(b0 + kPlanThreads) * p.stride : rows_before);
    const int32_t to = (int32_t)min((i64)r_end, next);
    for (int64_t r = max(r_begin, (int64_t)s_start[0]) + tid; r < to; r += kPlanThreads) {
      const int s = last_at_most(s_start, n_seq, (int32_t)r);
      const int32_t i = (int32_t)r - s_start[s];
      int64_t row_slot = -1;
      int32_t row_pos = -1;
      if (i < s_count[s]) {
        const int32_t slot = s_len[s] + i, col = slot >> lp, have = (s_len[s] + page_mask) >> lp;
        int32_t* entry = p.table + (int64_t)(b0 + s) * p.ld + col;
        int32_t page;
        if (pool && col >= have) {
          page = p.free_pages[free - 1 - (s_taken[s] + (col - have))];
          if ((slot & page_mask) == 0) *entry = page;
        } else {
          page = *entry;
        }
        row_slot = page >= 0 ? ((int64_t)page << lp) + (slot & page_mask) : -1;
        row_pos = s_pos[s] + 1 + i;
      }
      p.row_slots[r] = row_slot;
      p.row_positions[r] = row_pos;
    }
    // (Rows ascend with the sequences: the others are behind this block's.)
    if (blockIdx.x != 0 && next >= r_end) return;
  }
  if (blockIdx.x == 0 && tid == 0 && pool) *p.free_out = (int32_t)(free - taken);
}

struct TruncateParams {
  const int32_t* to;
  const int32_t* lengths;
  const int32_t* positions;
  int32_t B;
  const int32_t* table;
  int64_t ld;
  int32_t width, log2_page;
  int32_t* free_pages;
  int32_t free_cap;
  const int32_t* free_count;
  int32_t* lengths_out;
  int32_t* positions_out;
  int32_t* free_out;
};

__global__ __launch_bounds__(kPlanThreads) void truncate_kernel(const TruncateParams p) {
  __shared__ i64 sums[kPlanThreads / 64];
  __shared__ i64 s_at[kPlanThreads];
  __shared__ int32_t s_keep[kPlanThreads];
  const int tid = threadIdx.x;
  const int lp = p.log2_page, page_mask = (1 << lp) - 1;
  const int32_t cap = p.width << lp;
  const i64 free = min(max(*p.free_count, 0), p.free_cap);
  // Pages that sequence b keeps, and those that it gives back.
  auto pages = [&](int32_t b, int32_t& keep) {
    const int32_t had = min(max(p.lengths[b], 0), cap), has = min(had, max(p.to[b], 0));
    keep = (has + page_mask) >> lp;
    return ((had + page_mask) >> lp) - keep;
  };
  i64 mine = 0, total;
  for (int32_t b = tid; b < p.B; b += kPlanThreads) {
    int32_t keep;
    mine += pages(b, keep);
  }
  block_before(mine, sums, total);
  i64 before = 0;
  for (int32_t b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int n_seq = min(kPlanThreads, p.B - b0);
    const int32_t b = b0 + tid;
    int32_t keep = 0;
    const i64 gone = tid < n_seq ? pages(b, keep) : 0;
    i64 sum;
    const i64 at = before + block_before(gone, sums, sum);
    s_at[tid] = at;
    s_keep[tid] = keep;
    __syncthreads();
    if (tid < n_seq && blockIdx.x == 0) {
      const int32_t had = p.lengths[b], to = max(p.to[b], 0), has = min(had, to);
      p.lengths_out[b] = has;
      p.positions_out[b] = p.positions[b] - (had - has);
    }
    for (i64 r = before + (i64)blockIdx.x * kPlanThreads + tid; r < before + sum; r += (i64)gridDim.x * kPlanThreads) {
      const int s = last_at_most(s_at, n_seq, r);
      const i64 to = free + total - 1 - r;
      if (to < p.free_cap) p.free_pages[to] = p.table[(int64_t)(b0 + s) * p.ld + s_keep[s] + (r - s_at[s])];
    }
    before += sum;
  }
  if (blockIdx.x == 0 && tid == 0) *p.free_out = (int32_t)min(free + total, (i64)p.free_cap);
}

struct ChunkAppendParams {
  const void* qkv;  // [rows] of (nq + 2 nkv) D at stride ld, fp32 or bf16
  int64_t ld, rows;
  int32_t nq, nkv, D;
  const uint16_t* q_norm_w;  // [D], nullptr = no QK norm
  const uint16_t* k_norm_w;
  float eps;
  const float* cos_sin;  // [n_pos][D / 2][2]
  int64_t n_pos;
  const int64_t* row_slots;  // of the pool: page * page size + row in it
  const int32_t* row_positions;
  int64_t pool_slots;
  int32_t log2_page;
  uint16_t* k_pages;
  uint16_t* v_pages;
  uint16_t* q;  // [rows][nq][D]
};

template <typename TIn>
__global__ __launch_bounds__(256) void chunk_append_kernel(const ChunkAppendParams p) {
  const int g16 = threadIdx.x & 15;
  const int heads = p.nq + 2 * p.nkv;
  const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), items = p.rows * heads;
  const int half = p.D >> 1;
  // Lanes past the head (and groups past the last row) take part in the row sums with zeros
  // and store nothing.
  const bool on = item < items && 4 * g16 < half;
  const int64_t it = item < items ? item : items - 1;
  const int64_t row = it / heads;
  const int head = (int)(it - row * heads);
  const int kind = head < p.nq ? 0 : (head < p.nq + p.nkv ? 1 : 2);
  const int h = kind == 0 ? head : (kind == 1 ? head - p.nq : head - p.nq - p.nkv);
  const int c = on ? 4 * g16 : 0;

  const TIn* src = static_cast<const TIn*>(p.qkv) + row * p.ld + (int64_t)head * p.D + c;
  const uint16_t* nw = kind == 1 ? p.k_norm_w : p.q_norm_w;
  const int32_t pos = p.row_positions[row];
  const int64_t slot = p.row_slots[row];
  const bool mapped = (uint64_t)slot < (uint64_t)p.pool_slots;
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
    if (!mapped) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x1[j] = x2[j] = 0.f;
    }
    dst = p.q + (row * p.nq + h) * p.D + c;
  } else {
    if (!mapped) return;
    const int64_t page = slot >> p.log2_page;
    const int64_t r = ((page * p.nkv + h) << p.log2_page) + (slot - (page << p.log2_page));
    dst = (kind == 1 ? p.k_pages : p.v_pages) + r * p.D + c;
  }
  head_store4(dst, x1);
  head_store4(dst + half, x2);
}

}  // namespace
}  // namespace cdx

extern "C" int cdx_paged_reserve(const int32_t* counts, const int32_t* lengths, const int32_t* positions, int64_t B,
                                 int64_t stride, int64_t rows, int32_t* table, int64_t table_ld, int64_t width,
                                 int32_t page_size, const int32_t* free_pages, int64_t free_capacity,
                                 const int32_t* free_count, int32_t* starts, int32_t* new_counts,
                                 int32_t* new_lengths, int32_t* new_positions, int32_t* new_free_count,
                                 int64_t* row_slots, int32_t* row_positions, void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_reserve";
  clear_error();
  PagedTable t{};
  if (int rc = paged_table(name, table, table_ld, width, 0, page_size, B, 1, 8, &t)) return rc;
  if (stride < 0 || rows < 0 || free_capacity < 0)
    return fail(CDX_EINVAL, "%s: bad shape rows=%lld stride=%lld free pages=%lld", name, (long long)rows,
                (long long)stride, (long long)free_capacity);
  if (rows > INT32_MAX - kPlanRows || stride > INT32_MAX || free_capacity > INT32_MAX)
    return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (B == 0) return fail(CDX_EINVAL, "%s: no sequences", name);
  const bool pool = free_count != nullptr;
  if (!counts || !lengths || !positions || !starts || !new_counts || !new_lengths || !new_positions ||
      (width > 0 && !table) || (rows > 0 && (!row_slots || !row_positions)) || pool != (new_free_count != nullptr) ||
      (free_pages && !pool) || (pool && free_capacity > 0 && !free_pages))
    return fail(CDX_EINVAL, "%s: null pointer", name);
  const Extent in[] = {{counts, 4 * B}, {lengths, 4 * B}, {positions, 4 * B}, {free_count, 4}};
  const Extent out[] = {{starts, 4 * B}, {new_counts, 4 * B}, {new_lengths, 4 * B}, {new_positions, 4 * B},
                        {new_free_count, 4}, {row_slots, 8 * rows}, {row_positions, 4 * rows}};
  if (overlap(in, out)) return fail(CDX_EINVAL, "%s: the results need memory of their own", name);
  ReserveParams p{};
  p.counts = counts;
  p.lengths = lengths;
  p.positions = positions;
  p.B = (int32_t)B;
  p.stride = (int32_t)stride;
  p.rows = (int32_t)rows;
  p.table = table;
  p.ld = table_ld;
  p.width = (int32_t)width;
  p.log2_page = t.log2_page;
  // (A pool of no pages still is one: any pointer that is not read.)
  p.free_pages = pool ? (free_pages ? free_pages : free_count) : nullptr;
  p.free_cap = (int32_t)free_capacity;
  p.free_count = free_count;
  p.starts = starts;
  p.counts_out = new_counts;
  p.lengths_out = new_lengths;
  p.positions_out = new_positions;
  p.free_out = new_free_count;
  p.row_slots = row_slots;
  p.row_positions = row_positions;
  const int64_t blocks = rows > 0 ? (rows + kPlanRows - 1) / kPlanRows : 1;
  reserve_kernel<<<dim3((unsigned)blocks), dim3(kPlanThreads), 0, reinterpret_cast<hipStream_t>(stream)>>>(p);
  return check_launch(name);
}

extern "C" int cdx_paged_truncate(const int32_t* to, const int32_t* lengths, const int32_t* positions, int64_t B,
                                  const int32_t* table, int64_t table_ld, int64_t width, int32_t page_size,
                                  int32_t* free_pages, int64_t free_capacity, const int32_t* free_count,
                                  int32_t* new_lengths, int32_t* new_positions, int32_t* new_free_count,
                                  void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_truncate";
  clear_error();
  PagedTable t{};
  if (int rc = paged_table(name, table, table_ld, width, 0, page_size, B, 1, 8, &t)) return rc;
  if (free_capacity < 0) return fail(CDX_EINVAL, "%s: bad shape free pages=%lld", name, (long long)free_capacity);
  if (free_capacity > INT32_MAX) return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (B == 0) return fail(CDX_EINVAL, "%s: no sequences", name);
  if (!to || !lengths || !positions || !free_count || !new_lengths || !new_positions || !new_free_count ||
      (width > 0 && !table) || (free_capacity > 0 && !free_pages))
    return fail(CDX_EINVAL, "%s: null pointer", name);
  const Extent in[] = {{to, 4 * B}, {lengths, 4 * B}, {positions, 4 * B}, {free_count, 4}};
  const Extent out[] = {{new_lengths, 4 * B}, {new_positions, 4 * B}, {new_free_count, 4}};
  if (overlap(in, out)) return fail(CDX_EINVAL, "%s: the results need memory of their own", name);
  TruncateParams p{};
  p.to = to;
  p.lengths = lengths;
  p.positions = positions;
  p.B = (int32_t)B;
  p.table = table;
  p.ld = table_ld;
  p.width = (int32_t)width;
  p.log2_page = t.log2_page;
  p.free_pages = free_pages;
  p.free_cap = (int32_t)free_capacity;
  p.free_count = free_count;
  p.lengths_out = new_lengths;
  p.positions_out = new_positions;
  p.free_out = new_free_count;
  // As many pages as the table has may come back; blocks walk them in turn.
  const int64_t pages = B * width, most = (pages + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  const int64_t blocks = most < 1 ? 1 : (most > 64 ? 64 : most);
  truncate_kernel<<<dim3((unsigned)blocks), dim3(kPlanThreads), 0, reinterpret_cast<hipStream_t>(stream)>>>(p);
  return check_launch(name);
}

extern "C" int cdx_paged_chunk_append_fwd(const void* qkv, int32_t qkv_fp32, int64_t ldqkv, int64_t rows, int32_t nq,
                                          int32_t nkv, int32_t hd, const uint16_t* q_norm_w, const uint16_t* k_norm_w,
                                          float eps, const float* cos_sin, int64_t n_pos, const int64_t* row_slots,
                                          const int32_t* row_positions, int64_t num_pages, int32_t page_size,
                                          uint16_t* k_pages, uint16_t* v_pages, uint16_t* q_out, void* stream) {
  using namespace cdx;
  const char* name = "cdx_paged_chunk_append_fwd";
  clear_error();
  PagedTable t{};
  if (int rc = paged_table(name, nullptr, 0, 0, num_pages, page_size, 1, nkv, hd, &t)) return rc;
  if (rows < 0 || nq <= 0 || nq % nkv != 0 || n_pos < 0)
    return fail(CDX_EINVAL, "%s: bad shape rows=%lld nq=%d nkv=%d n_pos=%lld", name, (long long)rows, nq, nkv,
                (long long)n_pos);
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(CDX_EINVAL, "%s: q and k norm weights must both be given or both be NULL", name);
  if (!(eps >= 0.f)) return fail(CDX_EINVAL, "%s: eps must be >= 0", name);
  const int64_t heads = (int64_t)nq + 2 * (int64_t)nkv;
  if (ldqkv < heads * hd) return fail(CDX_EINVAL, "%s: leading dimension too small", name);
  if (ldqkv % 8) return fail(CDX_EUNSUPPORTED, "%s: leading dimensions must be multiples of 8", name);
  if (heads > 65535 || rows > INT32_MAX) return fail(CDX_EUNSUPPORTED, "%s: problem too large", name);
  if (rows == 0) return CDX_OK;
  if (n_pos == 0) return fail(CDX_EINVAL, "%s: empty cos/sin table", name);
  if (!qkv || !cos_sin || !row_slots || !row_positions || !q_out || (num_pages > 0 && (!k_pages || !v_pages)))
    return fail(CDX_EINVAL, "%s: null pointer", name);
  if (!aligned16(qkv) || !aligned16(cos_sin) || !aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) ||
      !aligned16(q_norm_w) || !aligned16(k_norm_w))
    return fail(CDX_EUNSUPPORTED, "%s: pointers must be 16-byte aligned", name);
  ChunkAppendParams p{};
  p.ld = ldqkv;
  p.nq = nq;
  p.nkv = nkv;
  p.D = hd;
  p.q_norm_w = q_norm_w;
  p.k_norm_w = k_norm_w;
  p.eps = eps;
  p.cos_sin = cos_sin;
  p.n_pos = n_pos;
  p.pool_slots = num_pages * page_size;
  p.log2_page = t.log2_page;
  p.k_pages = k_pages;
  p.v_pages = v_pages;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t per = max_blocks(256) * 16 / heads;  // rows of one launch
  for (int64_t r0 = 0; r0 < rows; r0 += per) {
    const int64_t n = rows - r0 < per ? rows - r0 : per;
    p.rows = n;
    p.qkv = static_cast<const char*>(qkv) + r0 * ldqkv * (qkv_fp32 ? 4 : 2);
    p.row_slots = row_slots + r0;
    p.row_positions = row_positions + r0;
    p.q = q_out + r0 * nq * hd;
    const dim3 grid((unsigned)((n * heads + 15) / 16));
    if (qkv_fp32)
      chunk_append_kernel<float><<<grid, dim3(256), 0, s>>>(p);
    else
      chunk_append_kernel<uint16_t><<<grid, dim3(256), 0, s>>>(p);
    if (int rc = check_launch(name)) return rc;
  }
  return CDX_OK;
}
