// Native call paths of the package's operators (module complexity_deep._host).
//
// A forward of few tokens is paced by its host side: checks, output tensors and ctypes
// conversions in Python took 6 to 20 us per operator against 2 to 10 us of kernel time.
// Measured (us per call, issued back to back): 1B attention step of 4 rows 46 -> 22, MoE step
// 32 -> 21, 150M block of 2048 tokens 148 -> 90, 150M model step 1360 -> 762 (with block_step
// 510).
// Each function here is the usual case of one Python operator of the same name: it checks
// its operands, allocates the outputs through torch's allocator, and calls the C-ABI on the
// current stream.  For anything else (a tensor to be made contiguous, cast or broadcast, a
// wrong shape, another device than the current one, an empty call) it launches nothing and
// returns None, and the Python operator goes its general way, which converts or raises.
// Nothing is kept between calls.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../../include/cdx.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline void check(int rc, const char* what) {
  if (rc != CDX_OK)
    throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(rc) + "): " + cdx_last_error());
}

// A plain tensor of this dtype on the current device (no wrapper class, storage present).
inline bool plain(const Tensor& t, at::ScalarType dtype = at::kBFloat16) {
  return t.defined() && t.is_cuda() && t.scalar_type() == dtype && t.has_storage() &&
         !t.key_set().has(c10::DispatchKey::Python) && t.get_device() == c10::hip::current_device();
}
inline bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// Plain, contiguous and 16-byte aligned.
inline bool dense(const Tensor& t, at::ScalarType dtype = at::kBFloat16) {
  return plain(t, dtype) && t.is_contiguous() && aligned(t);
}
inline const uint16_t* u16(const Tensor& t) { return reinterpret_cast<const uint16_t*>(t.data_ptr()); }
inline uint16_t* w16(const Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }
inline const uint16_t* u16(const OptTensor& t) { return t ? u16(*t) : nullptr; }
inline void* stream() { return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream().stream()); }
inline Tensor like(const Tensor& t, at::IntArrayRef shape) { return at::empty(shape, t.options().requires_grad(false)); }
inline Tensor ints(const Tensor& t, at::IntArrayRef shape) {
  return at::empty(shape, t.options().dtype(at::kInt).requires_grad(false));
}

// Row stride of a [..., H] view whose rows are evenly spaced with unit stride inside (0: one
// row for all), or -1.  Dimensions of size 1 have no say: expand() leaves them any stride.
int64_t row_ld(const Tensor& t, int64_t H) {
  if (t.dim() < 1 || t.size(-1) != H || t.stride(-1) != 1) return -1;
  if (t.is_contiguous()) return H;
  int64_t ld = -1, next = 0;
  bool bcast = t.dim() > 1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (t.stride(d) != 0) bcast = false;
    if (ld < 0)
      ld = t.stride(d);
    else if (t.stride(d) != next)
      return bcast ? 0 : -1;
    next = t.stride(d) * t.size(d);
  }
  if (bcast) return 0;
  if (ld < 0) ld = H;
  return ld < H || ld % 8 != 0 ? -1 : ld;
}

OptTensor rms_norm(const Tensor& x, const Tensor& w, double eps, const OptTensor& out) {
  if (!dense(x) || !dense(w) || x.dim() < 1 || x.numel() == 0) return {};
  const int64_t H = x.size(-1);
  if (w.numel() != H || H % 8 != 0 || H > 8192 || !(eps >= 0)) return {};
  int64_t ldo = H;
  if (out) {
    if (!plain(*out) || !aligned(*out) || out->sizes() != x.sizes()) return {};
    ldo = row_ld(*out, H);
    if (ldo < H) return {};
  }
  Tensor y = out ? *out : like(x, x.sizes());
  check(cdx_rmsnorm_ld_fwd(u16(x), u16(w), (float)eps, x.numel() / H, (int32_t)H, w16(y), ldo, stream()),
        "cdx_rmsnorm_ld_fwd");
  return y;
}

std::optional<std::tuple<Tensor, OptTensor>> add_rms_norm(const Tensor& x, const Tensor& r, const Tensor& w,
                                                          double eps, bool store) {
  if (!dense(x) || !dense(r) || !dense(w) || x.dim() < 1 || x.numel() == 0 || r.sizes() != x.sizes()) return {};
  const int64_t H = x.size(-1);
  if (w.numel() != H || H % 8 != 0 || H > 8192 || !(eps >= 0)) return {};
  Tensor y = like(x, x.sizes());
  OptTensor h;
  if (store) h = like(x, x.sizes());
  check(cdx_add_rmsnorm_fwd(u16(x), u16(r), u16(w), (float)eps, x.numel() / H, (int32_t)H, w16(y),
                            h ? w16(*h) : nullptr, stream()),
        "cdx_add_rmsnorm_fwd");
  return std::make_tuple(y, h);
}

OptTensor embedding(const Tensor& ids, const Tensor& table) {
  if (!plain(ids, at::kLong) || !ids.is_contiguous() || !dense(table) || table.dim() != 2 || ids.numel() == 0) return {};
  const int64_t H = table.size(1);
  if (H % 8 != 0 || H > 16384 || table.size(0) == 0) return {};
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(H);
  Tensor out = like(table, shape);
  check(cdx_embedding_fwd(ids.data_ptr<int64_t>(), ids.numel(), u16(table), table.size(0), (int32_t)H, w16(out),
                          stream()),
        "cdx_embedding_fwd");
  return out;
}

OptTensor linear(const Tensor& x, const Tensor& w) {
  if (!dense(x) || !dense(w) || w.dim() != 2 || x.dim() < 2 || x.numel() == 0) return {};
  const int64_t N = w.size(0), K = w.size(1);
  if (x.size(-1) != K || K % 64 != 0 || N % 8 != 0 || N == 0 || N > INT32_MAX || K > INT32_MAX) return {};
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  Tensor out = like(x, shape);
  check(cdx_linear_fwd(u16(x), K, u16(w), K, x.numel() / K, (int32_t)K, (int32_t)N, w16(out), N, stream()),
        "cdx_linear_fwd");
  return out;
}

bool linear_accumulate(const Tensor& x, const Tensor& w, const Tensor& residual) {
  if (!dense(x) || !dense(w) || !dense(residual) || w.dim() != 2 || x.dim() < 2 || x.numel() == 0) return false;
  const int64_t N = w.size(0), K = w.size(1);
  if (x.size(-1) != K || residual.dim() != x.dim() || residual.size(-1) != N ||
      residual.sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1) || K % 64 != 0 || N % 8 != 0 || N == 0 ||
      N > INT32_MAX || K > INT32_MAX)
    return false;
  const int64_t M = x.numel() / K;
  if (!cdx_few_rows(M, N)) return false;
  check(cdx_linear_accum_fwd(u16(x), K, u16(w), K, M, (int32_t)K, (int32_t)N, w16(residual), N, stream()),
        "cdx_linear_accum_fwd");
  return true;
}

OptTensor mu_guidance(const Tensor& h, const Tensor& w, const Tensor& mu, double mu_lo, double mu_hi, double lo,
                      double hi, const OptTensor& out) {
  if (!dense(h) || !dense(w) || !dense(mu) || h.dim() < 1 || h.numel() == 0) return {};
  const int64_t H = h.size(-1);
  if (H % 64 != 0 || H > INT32_MAX || mu.dim() != 1 || mu.size(0) != H || w.dim() != 2 || w.size(0) != H ||
      w.size(1) != H || !(lo <= hi) || !(mu_lo <= mu_hi))
    return {};
  int64_t ldo = H;
  if (out) {
    if (!plain(*out) || !aligned(*out) || out->sizes() != h.sizes()) return {};
    ldo = row_ld(*out, H);
    if (ldo < H) return {};
  }
  Tensor y = out ? *out : like(h, h.sizes());
  check(cdx_mu_guidance_fwd(u16(h), h.numel() / H, (int32_t)H, u16(w), u16(mu), (float)mu_lo, (float)mu_hi, (float)lo,
                            (float)hi, w16(y), ldo, stream()),
        "cdx_mu_guidance_fwd");
  return y;
}

using Plan = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;  // expert_id, perm, inv_perm, counts, offsets

// The plan of ids through a map (without one, ids are expert ids already).
std::optional<Plan> route_plan(const Tensor& ids, const OptTensor& map, int64_t E) {
  const int64_t T = ids.numel();
  if (T == 0 || T > INT32_MAX || E <= 0 || E > 64 || !plain(ids, at::kLong) || !ids.is_contiguous()) return {};
  if (map && (!plain(*map, at::kLong) || !map->is_contiguous() || map->dim() != 1 || map->size(0) == 0)) return {};
  Tensor eid = ints(ids, {T}), perm = ints(ids, {T}), inv = ints(ids, {T}), counts = ints(ids, {E});
  Tensor offsets = ints(ids, {E + 1});
  const size_t bytes = cdx_route_workspace_bytes(T, (int32_t)E);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 16)}, ids.options().dtype(at::kByte));
  check(cdx_route_plan(ids.data_ptr<int64_t>(), T, map ? map->data_ptr<int64_t>() : nullptr, map ? map->size(0) : 0,
                       (int32_t)E, eid.data_ptr<int32_t>(), perm.data_ptr<int32_t>(), inv.data_ptr<int32_t>(),
                       counts.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), ws.data_ptr(), bytes, stream()),
        "cdx_route_plan");
  return Plan(eid, perm, inv, counts, offsets);
}

// One plan per map over the same ids, each the rows of common buffers.
std::optional<std::vector<Plan>> route_plans(const Tensor& ids, const std::vector<Tensor>& maps, int64_t E) {
  const int64_t L = (int64_t)maps.size(), T = ids.numel();
  if (L == 0 || T == 0 || E <= 0 || E > 64 || L * T > INT32_MAX || !plain(ids, at::kLong) || !ids.is_contiguous())
    return {};
  std::vector<const int64_t*> table;
  table.reserve(L);
  for (const Tensor& m : maps) {
    if (!plain(m, at::kLong) || !m.is_contiguous() || m.dim() != 1 || m.size(0) != maps[0].size(0) || m.size(0) == 0)
      return {};
    table.push_back(m.data_ptr<int64_t>());
  }
  Tensor eid = ints(ids, {L, T}), perm = ints(ids, {L, T}), inv = ints(ids, {L, T});
  Tensor counts = ints(ids, {L, E}), offsets = ints(ids, {L, E + 1});
  const size_t bytes = cdx_route_plans_workspace_bytes(T, (int32_t)E, (int32_t)L);
  Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 16)}, ids.options().dtype(at::kByte));
  check(cdx_route_plans(ids.data_ptr<int64_t>(), T, table.data(), (int32_t)L, maps[0].size(0), (int32_t)E,
                        eid.data_ptr<int32_t>(), perm.data_ptr<int32_t>(), inv.data_ptr<int32_t>(),
                        counts.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), ws.data_ptr(), bytes, stream()),
        "cdx_route_plans");
  std::vector<Plan> plans;
  plans.reserve(L);
  for (int64_t y = 0; y < L; ++y)
    plans.emplace_back(eid.select(0, y), perm.select(0, y), inv.select(0, y), counts.select(0, y), offsets.select(0, y));
  return plans;
}

OptTensor moe_swiglu(const Tensor& x, const Tensor& perm, const Tensor& offsets, int64_t E, const Tensor& w_gu,
                     const Tensor& w_down, int64_t ie, bool shared, const OptTensor& residual) {
  if (!dense(x) || !dense(w_gu) || !dense(w_down) || x.dim() != 2 || x.numel() == 0 || w_gu.dim() != 4 ||
      w_down.dim() != 3 || !plain(perm, at::kInt) || !plain(offsets, at::kInt) || !perm.is_contiguous() ||
      !offsets.is_contiguous())
    return {};
  const int64_t T = x.size(0), H = x.size(1), P = (ie + 63) / 64 * 64, nb = E + (shared ? 1 : 0);
  if (E <= 0 || E > 64 || H % 64 != 0 || perm.numel() < T || offsets.numel() < E + 1 || w_gu.size(0) != nb ||
      w_gu.size(1) != 2 || w_gu.size(2) != P || w_gu.size(3) != H || w_down.size(0) != nb || w_down.size(1) != H ||
      w_down.size(2) != P)
    return {};
  if (residual && (!dense(*residual) || residual->sizes() != x.sizes())) return {};
  Tensor out = residual ? *residual : like(x, x.sizes());
  Tensor inter = like(x, {T, (shared ? 2 : 1) * P});
  auto fn = residual ? cdx_moe_swiglu_residual_fwd : cdx_moe_swiglu_fwd;
  check(fn(u16(x), T, (int32_t)H, (int32_t)ie, (int32_t)E, shared, perm.data_ptr<int32_t>(),
           offsets.data_ptr<int32_t>(), u16(w_gu), u16(w_down), w16(inter), w16(out), stream()),
        residual ? "cdx_moe_swiglu_residual_fwd" : "cdx_moe_swiglu_fwd");
  return out;
}

// sort_tokens_by_expert: (rows in expert order, their indices, offsets, counts), indices in 64 bits.
std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> sort_tokens(const Tensor& tokens, const Tensor& experts,
                                                                       int64_t E) {
  const int64_t T = experts.numel();
  if (!tokens.is_cuda() || !plain(tokens, tokens.scalar_type()) || !tokens.is_contiguous() || !aligned(tokens) ||
      tokens.dim() < 1 || tokens.size(0) != T || tokens.numel() == 0)
    return {};
  auto plan = route_plan(experts, {}, E);
  if (!plan) return {};
  const auto& [eid, perm, inv, counts, offsets] = *plan;
  Tensor rows = like(tokens, tokens.sizes());
  check(cdx_permute_rows(tokens.data_ptr(), perm.data_ptr<int32_t>(), T, tokens.nbytes() / T, rows.data_ptr(), stream()),
        "cdx_permute_rows");
  auto longs = [&](int64_t n) { return at::empty({n}, experts.options()); };
  Tensor index = longs(T), off64 = longs(E + 1), cnt64 = longs(E);
  check(cdx_widen_plan(perm.data_ptr<int32_t>(), T, offsets.data_ptr<int32_t>(), counts.data_ptr<int32_t>(), (int32_t)E,
                       index.data_ptr<int64_t>(), off64.data_ptr<int64_t>(), cnt64.data_ptr<int64_t>(), stream()),
        "cdx_widen_plan");
  return std::make_tuple(rows, index, off64, cnt64);
}

// persistent_swiglu_cggr: pack the weights and prepare the rows in one launch, then both passes.
OptTensor swiglu_cggr(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down,
                      const Tensor& offsets) {
  if (!dense(x) || x.dim() != 2 || x.numel() == 0 || !dense(gate) || !dense(up) || !dense(down) || gate.dim() != 3 ||
      !plain(offsets, at::kLong) || !offsets.is_contiguous() || offsets.dim() != 1)
    return {};
  const int64_t T = x.size(0), H = x.size(1), E = gate.size(0), I = gate.size(2), P = (I + 63) / 64 * 64;
  if (gate.size(1) != H || up.sizes() != gate.sizes() || down.dim() != 3 || down.size(0) != E || down.size(1) != I ||
      down.size(2) != H || H % 64 != 0 || I % 8 != 0 || I == 0 || E > 64 || E == 0 || offsets.numel() != E + 1 ||
      T > INT32_MAX - 256 || T * H * 2 > (int64_t)UINT32_MAX || E * 2 * P * H * 2 > (int64_t)UINT32_MAX)
    return {};
  Tensor w_gu = like(x, {E, 2, P, H}), w_down = like(x, {E, H, P}), out = like(x, {T, H}), inter = like(x, {T, P});
  Tensor off32 = ints(x, {E + 1}), ident = ints(x, {T});
  void* st = stream();
  check(cdx_cggr_prepare(u16(gate), u16(up), u16(down), (int32_t)E, (int32_t)H, (int32_t)I, offsets.data_ptr<int64_t>(),
                         T, w16(w_gu), w16(w_down), off32.data_ptr<int32_t>(), ident.data_ptr<int32_t>(), w16(out), st),
        "cdx_cggr_prepare");
  check(cdx_moe_swiglu_fwd(u16(x), T, (int32_t)H, (int32_t)I, (int32_t)E, 0, ident.data_ptr<int32_t>(),
                           off32.data_ptr<int32_t>(), u16(w_gu), u16(w_down), w16(inter), w16(out), st),
        "cdx_moe_swiglu_fwd");
  return out;
}

// The attention of a call without a mask, up to o_proj: (merged heads [B, S, nq D], k, v),
// k and v only with a cache.  w is the [N, 2 H] buffer of the projection and mu weights side
// by side.  past: both or neither.  Covers the fused projection (heads of 32, 64 and 128)
// and the few-row / other-head-dim form, chosen as in ComplexityAttention.forward.
std::optional<std::tuple<Tensor, OptTensor, OptTensor>> attention(
    const Tensor& x, const OptTensor& mu_in, const Tensor& w, int64_t nq, int64_t nkv, int64_t D, const OptTensor& qn,
    const OptTensor& kn, double eps, const Tensor& cos_sin, const OptTensor& past_k, const OptTensor& past_v,
    bool use_cache) {
  if (!plain(x) || !aligned(x) || x.dim() != 3 || x.numel() == 0 || !dense(w) || w.dim() != 2) return {};
  const int64_t B = x.size(0), S = x.size(1), H = x.size(2), M = B * S, N = (nq + 2 * nkv) * D;
  if (H % 64 != 0 || w.size(0) != N || w.size(1) != 2 * H || nkv <= 0 || nq % nkv != 0 || D <= 0 || D % 8 != 0 ||
      D > 128)
    return {};
  const int64_t ldx = row_ld(x, H);
  if (ldx < H) return {};
  OptTensor mu = mu_in;
  int64_t ldmu = 0;
  if (mu) {
    if (!plain(*mu) || !aligned(*mu) || mu->dim() != 3 || mu->size(0) != B || mu->size(1) != S || mu->size(2) != H)
      return {};
    ldmu = row_ld(*mu, H);
    if (ldmu < 0) return {};
    if (ldmu == 0 && M == 1) ldmu = H;
  }
  if (qn.has_value() != kn.has_value()) return {};
  if (qn && (!dense(*qn) || !dense(*kn) || qn->numel() != D || kn->numel() != D)) return {};
  if (past_k.has_value() != past_v.has_value() || (past_k && past_k->dim() != 4)) return {};
  const int64_t P = past_k ? past_k->size(2) : 0;
  if (!plain(cos_sin, at::kFloat) || !cos_sin.is_contiguous() || cos_sin.size(0) < P + S || !(eps >= 0)) return {};
  const float scale = (float)(1.0 / std::sqrt((double)D));
  const uint16_t* w_mu = u16(w) + H;
  const int64_t ldw = 2 * H, vt_ld = (S + 63) / 64 * 64, n_pos = cos_sin.size(0);
  const float* table = cos_sin.data_ptr<float>();
  void* st = stream();
  const bool fused_dim = D == 32 || D == 64 || D == 128, few = cdx_few_rows(M, N) != 0;

  if (fused_dim && !few && !past_k && !use_cache) {
    Tensor q = like(x, {B, nq, S, D}), k = like(x, {B, nkv, S, D}), vt = like(x, {B, nkv, D, vt_ld});
    // Columns of the key positions S .. vt_ld - 1 are masked but must be finite (the order
    // inside a 16-group moves some of them below S).
    if (vt_ld > S) vt.narrow(3, S / 16 * 16, vt_ld - S / 16 * 16).zero_();
    const bool side = mu && ldmu == ldx && ldx >= 2 * H && mu->data_ptr() == static_cast<const void*>(u16(x) + H);
    if (mu && ldmu == 0 && H > 64) {
      Tensor work = like(x, {N * ldw + 64});
      check(cdx_mu_qkv_rope_bcast_fwd(u16(x), ldx, u16(*mu), u16(w), w_mu, ldw, B, S, (int32_t)H, (int32_t)nq,
                                      (int32_t)nkv, (int32_t)D, u16(qn), u16(kn), (float)eps, table, n_pos, 0, w16(q),
                                      w16(k), w16(vt), vt_ld, w16(work), st),
            "cdx_mu_qkv_rope_bcast_fwd");
    } else {
      check(cdx_mu_qkv_rope_fwd(u16(x), ldx, side ? nullptr : u16(mu), side ? 0 : ldmu, u16(w), side ? nullptr : w_mu,
                                ldw, B, S, (int32_t)(side ? 2 * H : H), (int32_t)nq, (int32_t)nkv, (int32_t)D, u16(qn),
                                u16(kn), (float)eps, table, n_pos, 0, w16(q), w16(k), w16(vt), vt_ld, st),
            "cdx_mu_qkv_rope_fwd");
    }
    Tensor out = like(x, {B, S, nq * D});
    check(cdx_attention_fwd(u16(q), u16(k), u16(vt), B, S, (int32_t)nq, (int32_t)nkv, (int32_t)D, vt_ld, scale,
                            w16(out), st),
          "cdx_attention_fwd");
    return std::make_tuple(out, OptTensor(), OptTensor());
  }
  if (fused_dim && !few) return {};  // a long prompt into a cache
  if (past_k && (!dense(*past_k) || !dense(*past_v) || past_k->dim() != 4 || past_k->size(0) != B ||
                 past_k->size(1) != nkv || past_k->size(3) != D || past_v->sizes() != past_k->sizes() || P == 0 ||
                 (at::GradMode::is_enabled() && (past_k->requires_grad() || past_v->requires_grad()))))
    return {};
  if (2 * B * nkv * (P + S) > INT32_MAX / (D / 8) || M > INT32_MAX / (nq + 2 * nkv)) return {};
  const bool attend = S <= 16 && P >= S;
  OptTensor q;
  if (!attend) q = like(x, {B, nq, S, D});
  Tensor out = like(x, {B, S, nq * D});
  Tensor k = like(x, {B, nkv, P + S, D}), v = like(x, {B, nkv, P + S, D});
  const size_t bytes = cdx_qkv_cache_workspace_bytes(B, S, (int32_t)nq, (int32_t)nkv, (int32_t)D);
  Tensor work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte).requires_grad(false));
  Tensor vt;
  if (!attend) vt = like(x, {B, nkv, D, vt_ld});
  if (!attend && P == 0) {
    check(cdx_qkv_prompt_fwd(u16(x), ldx, u16(mu), ldmu, u16(w), w_mu, ldw, B, S, (int32_t)H, (int32_t)nq, (int32_t)nkv,
                             (int32_t)D, u16(qn), u16(kn), (float)eps, table, n_pos, w16(*q), w16(k), w16(v), w16(vt),
                             vt_ld, work.data_ptr(), bytes, st),
          "cdx_qkv_prompt_fwd");
  } else {
    check(cdx_qkv_cache_fwd(u16(x), ldx, u16(mu), ldmu, u16(w), w_mu, ldw, B, S, (int32_t)H, (int32_t)nq, (int32_t)nkv,
                            (int32_t)D, u16(qn), u16(kn), (float)eps, table, n_pos, u16(past_k), u16(past_v), P,
                            q ? w16(*q) : nullptr, w16(k), w16(v), attend ? w16(out) : nullptr, scale, work.data_ptr(),
                            bytes, st),
          "cdx_qkv_cache_fwd");
    if (!attend) check(cdx_vt_pack(u16(v), B * nkv, P + S, S, (int32_t)D, w16(vt), vt_ld, st), "cdx_vt_pack");
  }
  if (!attend)
    check(cdx_attention_cache_fwd(u16(*q), u16(k), u16(vt), B, S, P + S, (int32_t)nq, (int32_t)nkv, (int32_t)D, vt_ld,
                                  scale, w16(out), st),
          "cdx_attention_cache_fwd");
  return std::make_tuple(out, OptTensor(k), OptTensor(v));
}

// ---- paged generation -------------------------------------------------------

// A paged cache's tensors as the C-ABI takes them.  dims 5: with a leading layer dimension.
struct Pages {
  int64_t layers = 1, pages = 0, nkv = 0, page = 0, D = 0, B = 0, width = 0, ld = 0;
  uint16_t *k = nullptr, *v = nullptr;
  const int32_t* table = nullptr;
  int64_t capacity() const { return width * page; }
};

inline bool no_grad(const Tensor& t) { return !(at::GradMode::is_enabled() && t.requires_grad()); }

bool paged_cache(const Tensor& k, const Tensor& v, const Tensor& table, int64_t dims, Pages* c) {
  if (!dense(k) || !dense(v) || !no_grad(k) || !no_grad(v) || k.dim() != dims || v.sizes() != k.sizes() ||
      k.numel() == 0 || !plain(table, at::kInt) || table.dim() != 2 || table.size(0) == 0 || table.size(1) == 0 ||
      table.stride(1) != 1)
    return false;
  c->layers = dims == 5 ? k.size(0) : 1;
  c->pages = k.size(-4);
  c->nkv = k.size(-3);
  c->page = k.size(-2);
  c->D = k.size(-1);
  c->B = table.size(0);
  c->width = table.size(1);
  c->ld = c->B > 1 ? table.stride(0) : c->width;
  c->k = w16(k);
  c->v = w16(v);
  c->table = table.data_ptr<int32_t>();
  const bool page_ok = c->page >= 16 && c->page <= 256 && (c->page & (c->page - 1)) == 0;
  return page_ok && c->ld >= c->width && c->D % 8 == 0 && c->D <= 128 && c->nkv <= 65535;
}

// A plain contiguous int32 tensor with one value per sequence.
inline bool per_sequence(const Tensor& t, int64_t B) {
  return plain(t, at::kInt) && t.is_contiguous() && t.dim() == 1 && t.size(0) == B;
}

OptTensor paged_append(const Tensor& qkv, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths,
                       const Tensor& positions, int64_t nq, const Tensor& cos_sin, const OptTensor& qn,
                       const OptTensor& kn, double eps) {
  Pages c;
  const bool fp32 = qkv.defined() && qkv.scalar_type() == at::kFloat;
  if (!paged_cache(k, v, table, 4, &c) || !dense(qkv, fp32 ? at::kFloat : at::kBFloat16) || !no_grad(qkv) ||
      !per_sequence(lengths, c.B) || !per_sequence(positions, c.B) || nq <= 0 || nq > 65535 || nq % c.nkv != 0 ||
      qkv.dim() != 2 || qkv.size(0) != c.B || qkv.size(1) != (nq + 2 * c.nkv) * c.D || !dense(cos_sin, at::kFloat) ||
      cos_sin.dim() != 3 || cos_sin.size(0) == 0 || cos_sin.size(1) != c.D / 2 || cos_sin.size(2) != 2 ||
      qn.has_value() != kn.has_value() || !(eps >= 0))
    return {};
  if (qn && (!dense(*qn) || !dense(*kn) || qn->numel() != c.D || kn->numel() != c.D || !no_grad(*qn) || !no_grad(*kn)))
    return {};
  Tensor q = like(k, {c.B, nq, c.D});
  check(cdx_paged_append_fwd(qkv.data_ptr(), fp32, qkv.size(1), c.B, (int32_t)nq, (int32_t)c.nkv, (int32_t)c.D,
                             u16(qn), u16(kn), (float)eps, cos_sin.data_ptr<float>(), cos_sin.size(0),
                             lengths.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), c.table, c.ld, c.width,
                             c.pages, (int32_t)c.page, c.k, c.v, w16(q), stream()),
        "cdx_paged_append_fwd");
  return q;
}

bool paged_write(const Tensor& k_new, const Tensor& v_new, const Tensor& k, const Tensor& v, const Tensor& table,
                 const Tensor& lengths) {
  Pages c;
  if (!paged_cache(k, v, table, 4, &c) || !dense(k_new) || !dense(v_new) || !no_grad(k_new) || !no_grad(v_new) ||
      k_new.dim() != 4 || k_new.sizes() != v_new.sizes() || k_new.size(0) != c.B || k_new.size(1) != c.nkv ||
      k_new.size(3) != c.D || k_new.size(2) == 0 || !per_sequence(lengths, c.B))
    return false;
  check(cdx_paged_write(u16(k_new), u16(v_new), c.B, (int32_t)c.nkv, k_new.size(2), (int32_t)c.D,
                        lengths.data_ptr<int32_t>(), c.table, c.ld, c.width, c.pages, (int32_t)c.page, c.k, c.v,
                        stream()),
        "cdx_paged_write");
  return true;
}

// (out, new weights or None)
std::optional<std::tuple<Tensor, OptTensor>> paged_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                                             const Tensor& table, const Tensor& lengths, double scale,
                                                             const OptTensor& weights, const OptTensor& weights_out) {
  Pages c;
  if (!paged_cache(k, v, table, 4, &c) || !dense(q) || !no_grad(q) || q.dim() != 3 || q.size(0) != c.B ||
      q.size(2) != c.D || q.size(1) == 0 || q.size(1) > 65535 || q.size(1) % c.nkv != 0 ||
      !per_sequence(lengths, c.B) || (weights_out && !weights))
    return {};
  auto rows = [&](const Tensor& t) {
    return plain(t, at::kFloat) && t.is_contiguous() && no_grad(t) && t.dim() == 3 && t.size(0) == c.B &&
           t.size(1) == c.nkv && t.size(2) == c.capacity();
  };
  if ((weights && !rows(*weights)) || (weights_out && !rows(*weights_out))) return {};
  const int64_t nq = q.size(1);
  Tensor out = like(q, {c.B, nq * c.D});
  OptTensor w_out = weights_out;
  if (weights && !w_out) w_out = like(*weights, weights->sizes());
  const size_t bytes = cdx_paged_attention_workspace_bytes(c.B, (int32_t)nq, (int32_t)c.nkv, (int32_t)c.D,
                                                           c.capacity(), weights.has_value());
  Tensor work;
  if (bytes) work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte).requires_grad(false));
  check(cdx_paged_attention_fwd(u16(q), c.B, (int32_t)nq, (int32_t)c.nkv, (int32_t)c.D, c.k, c.v, c.table, c.ld,
                                c.width, c.pages, (int32_t)c.page, lengths.data_ptr<int32_t>(), (float)scale, w16(out),
                                weights ? weights->data_ptr<float>() : nullptr,
                                w_out ? w_out->data_ptr<float>() : nullptr, bytes ? work.data_ptr() : nullptr, bytes,
                                stream()),
        "cdx_paged_attention_fwd");
  return std::make_tuple(out, w_out);
}

// (lengths, weights, slot positions)
std::optional<std::tuple<Tensor, Tensor, Tensor>> paged_evict(const Tensor& k, const Tensor& v, const Tensor& table,
                                                              const Tensor& lengths, const Tensor& positions,
                                                              const Tensor& weights, const Tensor& slot_positions,
                                                              int64_t keep, int64_t recent) {
  Pages c;
  if (!k.defined() || !paged_cache(k, v, table, k.dim() == 5 ? 5 : 4, &c) || !per_sequence(lengths, c.B) ||
      !per_sequence(positions, c.B) || keep <= 0 || recent < 0 || recent > keep)
    return {};
  std::vector<int64_t> shape{c.B, c.nkv, c.capacity()};
  if (k.dim() == 5) shape.insert(shape.begin(), c.layers);
  if (!plain(weights, at::kFloat) || !plain(slot_positions, at::kInt) || !weights.is_contiguous() ||
      !slot_positions.is_contiguous() || !no_grad(weights) || weights.sizes() != at::IntArrayRef(shape) ||
      slot_positions.sizes() != at::IntArrayRef(shape))
    return {};
  Tensor new_len = ints(lengths, {c.B}), new_w = like(weights, shape), new_pos = ints(slot_positions, shape);
  const size_t bytes = cdx_paged_evict_workspace_bytes(c.layers, c.B, (int32_t)c.nkv, c.capacity(), keep);
  Tensor work = at::empty({(int64_t)bytes}, k.options().dtype(at::kByte).requires_grad(false));
  check(cdx_paged_evict(c.layers, c.B, (int32_t)c.nkv, (int32_t)c.D, lengths.data_ptr<int32_t>(),
                        positions.data_ptr<int32_t>(), c.table, c.ld, c.width, c.pages, (int32_t)c.page, c.k, c.v,
                        weights.data_ptr<float>(), slot_positions.data_ptr<int32_t>(), keep, recent,
                        new_len.data_ptr<int32_t>(), new_w.data_ptr<float>(), new_pos.data_ptr<int32_t>(),
                        work.data_ptr(), bytes, stream()),
        "cdx_paged_evict");
  return std::make_tuple(new_len, new_w, new_pos);
}

// The attention of one new token per sequence on a layer of a paged cache, up to o_proj: the
// projection of x [B, 1, H] (of RMSNorm(x) with `norm`, B <= 8), its append and the attention, whose
// weights go to `weights`.  w as in `attention`.
struct PagedStep {
  Pages c;
  int64_t H = 0, nq = 0, ldx = 0, ldmu = 0;
  OptTensor mu;
};

bool paged_step_fits(const Tensor& x, const OptTensor& mu, const Tensor& w, int64_t nq, int64_t D, const OptTensor& qn,
                     const OptTensor& kn, double eps, const Tensor& cos_sin, const Tensor& k, const Tensor& v,
                     const Tensor& table, const Tensor& lengths, const Tensor& positions, const OptTensor& weights,
                     PagedStep* s) {
  Pages& c = s->c;
  if (!paged_cache(k, v, table, 4, &c) || !plain(x) || !aligned(x) || !no_grad(x) || x.dim() != 3 ||
      x.size(0) != c.B || x.size(1) != 1 || D != c.D || !dense(w) || w.dim() != 2 || nq <= 0 || nq > 65535 ||
      nq % c.nkv != 0 || !per_sequence(lengths, c.B) || !per_sequence(positions, c.B))
    return false;
  const int64_t H = x.size(2);
  s->H = H;
  s->nq = nq;
  s->ldx = row_ld(x, H);
  if (c.B == 1) s->ldx = H;
  if (H == 0 || H % 64 != 0 || s->ldx < H || s->ldx % 8 != 0 || w.size(0) != (nq + 2 * c.nkv) * D ||
      w.size(1) != 2 * H)
    return false;
  s->mu = mu;
  if (mu) {
    if (!plain(*mu) || !aligned(*mu) || mu->dim() != 3 || mu->size(0) != c.B || mu->size(1) != 1 || mu->size(2) != H)
      return false;
    s->ldmu = c.B == 1 ? H : row_ld(*mu, H);
    if (s->ldmu < 0 || mu->stride(2) != 1) return false;
  }
  if (qn.has_value() != kn.has_value() || !(eps >= 0) || !dense(cos_sin, at::kFloat) || cos_sin.dim() != 3 ||
      cos_sin.size(0) == 0 || cos_sin.size(1) != D / 2)
    return false;
  if (qn && (!dense(*qn) || !dense(*kn) || qn->numel() != D || kn->numel() != D)) return false;
  return !weights || (plain(*weights, at::kFloat) && weights->is_contiguous() && weights->dim() == 3 &&
                      weights->size(0) == c.B && weights->size(1) == c.nkv && weights->size(2) == c.capacity());
}

Tensor paged_step_run(const PagedStep& s, const Tensor& x, const uint16_t* norm, float norm_eps, const Tensor& w,
                      const OptTensor& qn, const OptTensor& kn, double eps, const Tensor& cos_sin,
                      const Tensor& lengths, const Tensor& positions, const OptTensor& weights, void* st) {
  const Pages& c = s.c;
  Tensor q = like(x, {c.B, s.nq, c.D}), out = like(x, {c.B, 1, s.nq * c.D});
  const size_t qkv = cdx_qkv_cache_workspace_bytes(c.B, 1, (int32_t)s.nq, (int32_t)c.nkv, (int32_t)c.D);
  const size_t attn = cdx_paged_attention_workspace_bytes(c.B, (int32_t)s.nq, (int32_t)c.nkv, (int32_t)c.D,
                                                          c.capacity(), weights.has_value());
  // (The attention's workspace may lie where the projection was: one follows the other.)
  const size_t bytes = std::max(qkv, attn);
  Tensor work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte).requires_grad(false));
  check(cdx_qkv_paged_fwd(u16(x), s.ldx, norm, norm_eps, u16(s.mu), s.ldmu, u16(w), u16(w) + s.H, 2 * s.H, c.B,
                          (int32_t)s.H, (int32_t)s.nq, (int32_t)c.nkv, (int32_t)c.D, u16(qn), u16(kn), (float)eps,
                          cos_sin.data_ptr<float>(), cos_sin.size(0), lengths.data_ptr<int32_t>(),
                          positions.data_ptr<int32_t>(), c.table, c.ld, c.width, c.pages, (int32_t)c.page, c.k, c.v,
                          w16(q), work.data_ptr(), bytes, st),
        "cdx_qkv_paged_fwd");
  float* acc = weights ? weights->data_ptr<float>() : nullptr;
  check(cdx_paged_attention_fwd(u16(q), c.B, (int32_t)s.nq, (int32_t)c.nkv, (int32_t)c.D, c.k, c.v, c.table, c.ld,
                                c.width, c.pages, (int32_t)c.page, lengths.data_ptr<int32_t>(),
                                (float)(1.0 / std::sqrt((double)c.D)), w16(out), acc, acc, work.data_ptr(), bytes, st),
        "cdx_paged_attention_fwd");
  return out;
}

OptTensor paged_step(const Tensor& x, const OptTensor& mu, const Tensor& w, int64_t nq, int64_t D, const OptTensor& qn,
                     const OptTensor& kn, double eps, const Tensor& cos_sin, const Tensor& k, const Tensor& v,
                     const Tensor& table, const Tensor& lengths, const Tensor& positions, const OptTensor& weights) {
  PagedStep s;
  if (!paged_step_fits(x, mu, w, nq, D, qn, kn, eps, cos_sin, k, v, table, lengths, positions, weights, &s)) return {};
  return paged_step_run(s, x, nullptr, 0.f, w, qn, kn, eps, cos_sin, lengths, positions, weights, stream());
}

// One decoder block of a generation step (B * S <= 8), h updated in place: the input norm, the
// attention with its cache, o_proj and its residual add, the post-attention norm, the MoE and
// its residual add, and mu for the next layer (with mu_w), in six launches: both norms are
// folded into the products that read them.  Returns (k, v, mu).  With a block table the past is a
// layer of a paged cache (S == 1), which is extended in place and returned.
std::optional<std::tuple<Tensor, Tensor, OptTensor>> block_step(
    const Tensor& h, const Tensor& ln1, double eps1, const OptTensor& mu, const Tensor& w, int64_t nq, int64_t nkv,
    int64_t D, const OptTensor& qn, const OptTensor& kn, double qk_eps, const Tensor& cos_sin,
    const OptTensor& past_k, const OptTensor& past_v, const Tensor& o_w, const Tensor& ln2, double eps2,
    const Tensor& perm, const Tensor& offsets, int64_t E, const Tensor& w_gu, const Tensor& w_down, int64_t ie,
    bool shared, const OptTensor& mu_w, const OptTensor& mu_param, double mu_lo, double mu_hi, double lo, double hi,
    const OptTensor& table, const OptTensor& lengths, const OptTensor& positions, const OptTensor& weights) {
  if (!dense(h) || h.dim() != 3 || h.numel() == 0 || !dense(ln1) || !dense(ln2) || !dense(w) || !dense(o_w) ||
      !dense(w_gu) || !dense(w_down) || w.dim() != 2 || o_w.dim() != 2 || w_gu.dim() != 4 || w_down.dim() != 3)
    return {};
  const int64_t B = h.size(0), S = h.size(1), H = h.size(2), M = B * S, N = (nq + 2 * nkv) * D;
  if (M > 8 || !cdx_few_rows(M, N) || !cdx_few_rows(M, H) || H % 64 != 0 || H > 8192 || ln1.numel() != H ||
      ln2.numel() != H || nkv <= 0 || nq % nkv != 0 || D <= 0 || D % 8 != 0 || D > 128 || w.size(0) != N ||
      w.size(1) != 2 * H || o_w.size(0) != H || o_w.size(1) != nq * D || (nq * D) % 64 != 0 || !(eps1 >= 0) ||
      !(eps2 >= 0) || !(qk_eps >= 0))
    return {};
  int64_t ldmu = 0;
  if (mu) {
    if (!plain(*mu) || !aligned(*mu) || mu->dim() != 3 || mu->size(0) != B || mu->size(1) != S || mu->size(2) != H)
      return {};
    ldmu = row_ld(*mu, H);
    if (ldmu < 0) return {};
  }
  if (qn.has_value() != kn.has_value() || past_k.has_value() != past_v.has_value()) return {};
  if (qn && (!dense(*qn) || !dense(*kn) || qn->numel() != D || kn->numel() != D)) return {};
  PagedStep paged;
  if (table && (!past_k || !lengths || !positions || past_k->dim() != 4 || past_k->size(1) != nkv ||
                !paged_step_fits(h, mu, w, nq, D, qn, kn, qk_eps, cos_sin, *past_k, *past_v, *table, *lengths,
                                 *positions, weights, &paged)))
    return {};
  if (!table && past_k &&
      (!dense(*past_k) || !dense(*past_v) || past_k->dim() != 4 || past_k->size(0) != B || past_k->size(1) != nkv ||
       past_k->size(2) == 0 || past_k->size(3) != D || past_v->sizes() != past_k->sizes() || !no_grad(*past_k) ||
       !no_grad(*past_v)))
    return {};
  const int64_t past = past_k && !table ? past_k->size(2) : 0;
  if (!plain(cos_sin, at::kFloat) || !cos_sin.is_contiguous() || cos_sin.size(0) < past + S ||
      2 * B * nkv * (past + S) > INT32_MAX / (D / 8))
    return {};
  const int64_t P = (ie + 63) / 64 * 64, nb = E + (shared ? 1 : 0);
  if (!plain(perm, at::kInt) || !plain(offsets, at::kInt) || !perm.is_contiguous() || !offsets.is_contiguous() ||
      perm.numel() < M || E <= 0 || E > 64 || offsets.numel() < E + 1 || w_gu.size(0) != nb || w_gu.size(1) != 2 ||
      w_gu.size(2) != P || w_gu.size(3) != H || w_down.size(0) != nb || w_down.size(1) != H || w_down.size(2) != P)
    return {};
  if (mu_w && (!mu_param || !dense(*mu_w) || !dense(*mu_param) || mu_w->dim() != 2 || mu_w->size(0) != H ||
               mu_w->size(1) != H || mu_param->dim() != 1 || mu_param->size(0) != H || !(lo <= hi) || !(mu_lo <= mu_hi)))
    return {};

  void* st = stream();
  Tensor attn, k, v;
  if (table) {
    k = *past_k;
    v = *past_v;
    attn = paged_step_run(paged, h, u16(ln1), (float)eps1, w, qn, kn, qk_eps, cos_sin, *lengths, *positions, weights,
                          st);
  } else {
    const float scale = (float)(1.0 / std::sqrt((double)D));
    const bool attend = S <= 16 && past >= S;
    attn = like(h, {B, S, nq * D});
    k = like(h, {B, nkv, past + S, D});
    v = like(h, {B, nkv, past + S, D});
    OptTensor q;
    if (!attend) q = like(h, {B, nq, S, D});
    const size_t bytes = cdx_qkv_cache_workspace_bytes(B, S, (int32_t)nq, (int32_t)nkv, (int32_t)D);
    Tensor work = at::empty({(int64_t)bytes}, h.options().dtype(at::kByte).requires_grad(false));
    check(cdx_qkv_cache_norm_fwd(u16(h), H, u16(ln1), (float)eps1, u16(mu), ldmu, u16(w), u16(w) + H, 2 * H, B, S,
                                 (int32_t)H, (int32_t)nq, (int32_t)nkv, (int32_t)D, u16(qn), u16(kn), (float)qk_eps,
                                 cos_sin.data_ptr<float>(), cos_sin.size(0), u16(past_k), u16(past_v), past,
                                 q ? w16(*q) : nullptr, w16(k), w16(v), attend ? w16(attn) : nullptr, scale,
                                 work.data_ptr(), bytes, st),
          "cdx_qkv_cache_norm_fwd");
    if (!attend) {
      Tensor vt = like(h, {B, nkv, D, 64});  // S <= 8
      check(cdx_vt_pack(u16(v), B * nkv, past + S, S, (int32_t)D, w16(vt), 64, st), "cdx_vt_pack");
      check(cdx_attention_cache_fwd(u16(*q), u16(k), u16(vt), B, S, past + S, (int32_t)nq, (int32_t)nkv, (int32_t)D, 64,
                                    scale, w16(attn), st),
            "cdx_attention_cache_fwd");
    }
  }
  check(cdx_linear_accum_fwd(u16(attn), nq * D, u16(o_w), nq * D, M, (int32_t)(nq * D), (int32_t)H, w16(h), H, st),
        "cdx_linear_accum_fwd");
  Tensor inter = like(h, {M, (shared ? 2 : 1) * P});
  check(cdx_moe_swiglu_norm_residual_fwd(w16(h), u16(ln2), (float)eps2, M, (int32_t)H, (int32_t)ie, (int32_t)E, shared,
                                         perm.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(), u16(w_gu),
                                         u16(w_down), w16(inter), st),
        "cdx_moe_swiglu_norm_residual_fwd");
  OptTensor mu_out;
  if (mu_w) {
    mu_out = like(h, h.sizes());
    check(cdx_mu_guidance_fwd(u16(h), M, (int32_t)H, u16(*mu_w), u16(*mu_param), (float)mu_lo, (float)mu_hi, (float)lo,
                              (float)hi, w16(*mu_out), H, st),
          "cdx_mu_guidance_fwd");
  }
  return std::make_tuple(k, v, mu_out);
}

// ---- sampling ---------------------------------------------------------------

// A setting of sample_tokens: a number within 0 .. top, or one value per row.
struct Setting {
  const void* rows = nullptr;
  double value = 0;
  bool ok = false;
};
Setting setting(const py::object& o, at::ScalarType dtype, int64_t B, double top) {
  Setting s;
  if (THPVariable_Check(o.ptr())) {
    const Tensor& t = THPVariable_Unpack(o.ptr());
    s.ok = plain(t, dtype) && t.is_contiguous() && t.dim() == 1 && t.size(0) == B;
    if (s.ok) s.rows = t.data_ptr();
  } else if (PyFloat_Check(o.ptr()) || PyLong_Check(o.ptr())) {
    s.value = PyFloat_AsDouble(o.ptr());
    if (s.value == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return s;
    }
    s.ok = s.value >= 0 && s.value <= top && (dtype != at::kInt || s.value == std::floor(s.value));
  }
  return s;
}

OptTensor sample_tokens(const Tensor& logits, const Tensor& uniforms, const py::object& temperature,
                        const py::object& top_k, const py::object& top_p, const py::object& min_p) {
  const bool fp32 = logits.defined() && logits.scalar_type() == at::kFloat;
  if (!plain(logits, fp32 ? at::kFloat : at::kBFloat16) || logits.dim() != 2 || logits.numel() == 0 ||
      !plain(uniforms, at::kFloat) || !uniforms.is_contiguous() || uniforms.dim() != 1)
    return {};
  const int64_t B = logits.size(0), V = logits.size(1), ld = B > 1 ? logits.stride(0) : V;
  if (uniforms.size(0) != B || V > (1 << 20) || ld < V || (V > 1 && logits.stride(1) != 1)) return {};
  const Setting t = setting(temperature, at::kFloat, B, 3e38), k = setting(top_k, at::kInt, B, 1e9);
  const Setting p = setting(top_p, at::kFloat, B, 1.0), m = setting(min_p, at::kFloat, B, 1.0);
  if (!t.ok || !k.ok || !p.ok || !m.ok) return {};
  Tensor tokens = at::empty({B}, logits.options().dtype(at::kLong).requires_grad(false));
  check(cdx_sample_tokens(logits.data_ptr(), fp32, ld, B, V, uniforms.data_ptr<float>(),
                          static_cast<const float*>(t.rows), (float)t.value, static_cast<const int32_t*>(k.rows),
                          (int32_t)k.value, static_cast<const float*>(p.rows), (float)p.value,
                          static_cast<const float*>(m.rows), (float)m.value, tokens.data_ptr<int64_t>(), stream()),
        "cdx_sample_tokens");
  return tokens;
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.def("rms_norm", &rms_norm);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("embedding", &embedding);
  m.def("linear", &linear);
  m.def("linear_accumulate", &linear_accumulate);
  m.def("mu_guidance", &mu_guidance);
  m.def("route_plan", &route_plan);
  m.def("route_plans", &route_plans);
  m.def("moe_swiglu", &moe_swiglu);
  m.def("sort_tokens", &sort_tokens);
  m.def("swiglu_cggr", &swiglu_cggr);
  m.def("attention", &attention);
  m.def("block_step", &block_step);
  m.def("paged_append", &paged_append);
  m.def("paged_step", &paged_step);
  m.def("paged_write", &paged_write);
  m.def("paged_attention", &paged_attention);
  m.def("paged_evict", &paged_evict);
  m.def("sample_tokens", &sample_tokens);
}
