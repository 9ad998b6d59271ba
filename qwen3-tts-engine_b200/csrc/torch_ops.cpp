// PyTorch bindings of the 8-bit cache, drafted-tree attention and log-probability entries (include/q3attn.h): schema,
// argument checks, outputs and the call, in C++. These ops run in a few microseconds, so their host side must not take
// longer than they do: through Python and ctypes a call costs 25 to 40 us of host time. Shapes for tracing are in
// q3attn/spec.py, which also documents each op.
#include <ATen/ops/clamp.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "q3attn.h"

namespace {

using at::Tensor;
using c10::ScalarType;
constexpr int64_t kHeads = 16, kKvHeads = 8, kDim = 128;

void check(int rc, const char* what) {
  if (rc == Q3_OK) return;
  TORCH_CHECK(rc != Q3_ERR_CUDA, what, ": ", q3_error_string(rc), " (", q3_last_cuda_error(), ")");
  TORCH_CHECK(false, what, ": ", q3_error_string(rc));
}

void on_device(const Tensor& t, const char* name, const Tensor& first) {
  TORCH_CHECK(t.is_cuda(), "q3attn: ", name, " must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(t.device() == first.device(), "q3attn: ", name, " is on ", t.device(), ", other arguments on ",
              first.device());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void* ptr(const std::optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

q3_quant_cache cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& first) {
  on_device(k, "k_cache", first);
  on_device(v, "v_cache", first);
  on_device(ks, "k_scale", first);
  on_device(vs, "v_scale", first);
  TORCH_CHECK(k.scalar_type() == ScalarType::Float8_e4m3fn && v.scalar_type() == ScalarType::Float8_e4m3fn,
              "q3attn: k_cache/v_cache must be float8_e4m3fn");
  TORCH_CHECK(ks.scalar_type() == ScalarType::Float8_e8m0fnu && vs.scalar_type() == ScalarType::Float8_e8m0fnu,
              "q3attn: k_scale/v_scale must be float8_e8m0fnu");
  TORCH_CHECK(k.dim() == 4 && k.size(2) == kKvHeads && k.size(3) == kDim && v.sizes() == k.sizes() && k.is_contiguous() &&
                  v.is_contiguous(),
              "q3attn: k_cache/v_cache must be contiguous [num_pages, page_size, 8, 128]");
  TORCH_CHECK(ks.sizes() == k.sizes().slice(0, 3) && vs.sizes() == ks.sizes() && ks.is_contiguous() && vs.is_contiguous(),
              "q3attn: k_scale/v_scale must be contiguous [num_pages, page_size, 8]");
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, "q3attn: too many pages");
  return {k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), static_cast<int32_t>(k.size(0)),
          static_cast<int32_t>(k.size(1))};
}

void check_table(const Tensor& bt, const Tensor& first) {
  on_device(bt, "block_table", first);
  TORCH_CHECK(bt.scalar_type() == ScalarType::Int && bt.dim() == 2 && (bt.size(1) <= 1 || bt.stride(1) == 1) &&
                  bt.size(0) <= INT32_MAX && bt.size(1) <= INT32_MAX,
              "q3attn: block_table must be int32 [seats, max_pages] with unit inner stride");
}

// A table of one column may have any inner stride; its row stride is at least its width.
int64_t table_stride(const Tensor& bt) { return bt.size(0) <= 1 && bt.stride(0) < bt.size(1) ? bt.size(1) : bt.stride(0); }

// Index vectors are taken as they are, or converted (int64 positions, strided slices). Narrowing saturates, so that what
// lies outside int32 stays out of range: -1 is no row, and neither is INT32_MAX (row_addresses).
Tensor index_of(const Tensor& t, const char* name, ScalarType type, int64_t n, const Tensor& first) {
  on_device(t, name, first);
  TORCH_CHECK(t.numel() == n, "q3attn: ", name, " must have one entry per row");
  TORCH_CHECK(t.scalar_type() == ScalarType::Int || t.scalar_type() == ScalarType::Long, "q3attn: ", name,
              " must be int32 or int64");
  if (t.scalar_type() == type) return t.is_contiguous() ? t : t.contiguous();
  return (type == ScalarType::Int ? at::clamp(t, -1, INT32_MAX) : t).to(type).contiguous();
}

// k and v rows [n, 8, 128] with one shared row stride (as the kernels take them), copied when theirs differ.
std::pair<Tensor, Tensor> kv_rows(const Tensor& k, const Tensor& v, const Tensor& first) {
  on_device(k, "k", first);
  on_device(v, "v", first);
  TORCH_CHECK(k.scalar_type() == ScalarType::BFloat16 && v.scalar_type() == ScalarType::BFloat16,
              "q3attn: k/v must be bfloat16");
  TORCH_CHECK(k.dim() == 3 && k.size(1) == kKvHeads && k.size(2) == kDim && v.sizes() == k.sizes() &&
                  k.size(0) <= INT32_MAX,
              "q3attn: k/v must be [n, 8, 128]");
  const bool rows = k.strides() == v.strides() && k.stride(2) == 1 && k.stride(1) == kDim &&
                    (k.size(0) <= 1 || k.stride(0) >= kKvHeads * kDim);
  return rows ? std::make_pair(k, v) : std::make_pair(k.contiguous(), v.contiguous());
}

int64_t row_stride(const Tensor& t) { return t.size(0) <= 1 ? kKvHeads * kDim : t.stride(0); }

void append_slots(const Tensor& k_, const Tensor& v_, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                  const Tensor& vs, const Tensor& slots) {
  const q3_quant_cache cache = cache_of(kc, vc, ks, vs, kc);
  const auto [k, v] = kv_rows(k_, v_, kc);
  const Tensor s = index_of(slots, "slots", ScalarType::Long, k.size(0), kc);
  c10::cuda::OptionalCUDAGuard guard(kc.device());
  check(q3_kv_quant_append_slots(k.data_ptr(), v.data_ptr(), row_stride(k), &cache, kKvHeads, kDim,
                                 s.data_ptr<int64_t>(), static_cast<int32_t>(k.size(0)), stream_of(kc)),
        "q3_kv_quant_append_slots");
}

struct Rows {
  Tensor pos;
  std::optional<Tensor> seat;
};

Rows row_addresses(int64_t n, const Tensor& positions, const Tensor& bt, const std::optional<Tensor>& seat_of_row,
                   const Tensor& first) {
  check_table(bt, first);
  TORCH_CHECK(positions.scalar_type() == ScalarType::Int || bt.size(1) * first.size(1) <= INT32_MAX,
              "q3attn: int64 positions with a block_table of 2^31 tokens a seat and more");
  Rows r{index_of(positions, "positions", ScalarType::Int, n, first), std::nullopt};
  if (seat_of_row.has_value()) r.seat = index_of(*seat_of_row, "seat_of_row", ScalarType::Int, n, first);
  else TORCH_CHECK(n <= bt.size(0), "q3attn: without seat_of_row row i is seat i's: block_table has too few rows");
  return r;
}

void append_paged(const Tensor& k_, const Tensor& v_, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                  const Tensor& vs, const Tensor& positions, const Tensor& bt, const std::optional<Tensor>& seat_of_row) {
  const q3_quant_cache cache = cache_of(kc, vc, ks, vs, kc);
  const auto [k, v] = kv_rows(k_, v_, kc);
  const Rows r = row_addresses(k.size(0), positions, bt, seat_of_row, kc);
  c10::cuda::OptionalCUDAGuard guard(kc.device());
  check(q3_kv_quant_append_paged(k.data_ptr(), v.data_ptr(), row_stride(k), &cache, kKvHeads, kDim,
                                 r.pos.data_ptr<int32_t>(), static_cast<const int32_t*>(ptr(r.seat)),
                                 bt.data_ptr<int32_t>(), table_stride(bt), static_cast<int32_t>(bt.size(0)),
                                 static_cast<int32_t>(bt.size(1)), static_cast<int32_t>(k.size(0)), stream_of(kc)),
        "q3_kv_quant_append_paged");
}

std::tuple<Tensor, Tensor> dequant_paged(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs,
                                         const Tensor& positions, const Tensor& bt,
                                         const std::optional<Tensor>& seat_of_row) {
  const q3_quant_cache cache = cache_of(kc, vc, ks, vs, kc);
  const int64_t n = positions.numel();
  TORCH_CHECK(n <= INT32_MAX, "q3attn: too many rows");
  const Rows r = row_addresses(n, positions, bt, seat_of_row, kc);
  c10::cuda::OptionalCUDAGuard guard(kc.device());
  Tensor k = at::empty({n, kKvHeads, kDim}, kc.options().dtype(ScalarType::BFloat16));
  Tensor v = at::empty({n, kKvHeads, kDim}, kc.options().dtype(ScalarType::BFloat16));
  check(q3_kv_dequant_paged(&cache, kKvHeads, kDim, r.pos.data_ptr<int32_t>(), static_cast<const int32_t*>(ptr(r.seat)),
                            bt.data_ptr<int32_t>(), table_stride(bt), static_cast<int32_t>(bt.size(0)),
                            static_cast<int32_t>(bt.size(1)), k.data_ptr(), v.data_ptr(), kKvHeads * kDim,
                            static_cast<int32_t>(n), stream_of(kc)),
        "q3_kv_dequant_paged");
  return {k, v};
}

// Fills what both attention ops share and runs: q [B, 16, 128] (T = 1) or [B, T, 16, 128].
Tensor attend(const Tensor& q_, q3_tree_attn& p, const Tensor& kc, const Tensor& vc, const std::optional<Tensor>& ks,
              const std::optional<Tensor>& vs, const Tensor& seqlens, const Tensor& bt, double scale) {
  const bool drafts = q_.dim() == 4;
  const int64_t B = q_.size(0), T = drafts ? q_.size(1) : 1;
  TORCH_CHECK(q_.scalar_type() == ScalarType::BFloat16, "q3attn: q must be bfloat16");
  TORCH_CHECK(B <= INT32_MAX, "q3attn: too many seats");
  TORCH_CHECK(ks.has_value() == vs.has_value(), "q3attn: k_scale and v_scale go together");
  if (ks.has_value()) {
    cache_of(kc, vc, *ks, *vs, q_);
  } else {
    on_device(kc, "k_cache", q_);
    on_device(vc, "v_cache", q_);
    TORCH_CHECK(kc.scalar_type() == ScalarType::BFloat16 && vc.scalar_type() == ScalarType::BFloat16,
                "q3attn: k_cache/v_cache must be bfloat16 (or float8_e4m3fn with scales)");
    TORCH_CHECK(kc.dim() == 4 && kc.size(2) == kKvHeads && kc.size(3) == kDim && vc.sizes() == kc.sizes() &&
                    kc.is_contiguous() && vc.is_contiguous() && kc.size(0) <= INT32_MAX && kc.size(1) <= INT32_MAX,
                "q3attn: k_cache/v_cache must be contiguous [num_pages, page_size, 8, 128]");
  }
  check_table(bt, q_);
  TORCH_CHECK(bt.size(0) == B, "q3attn: block_table must have one row per seat");
  on_device(seqlens, "cache_seqlens", q_);
  TORCH_CHECK(seqlens.scalar_type() == ScalarType::Int && seqlens.numel() == B && seqlens.is_contiguous(),
              "q3attn: cache_seqlens must be a contiguous int32 tensor [B]");
  c10::cuda::OptionalCUDAGuard guard(q_.device());
  const bool rows = q_.stride(-1) == 1 && q_.stride(-2) == kDim && (T == 1 || q_.stride(1) >= kHeads * kDim);
  const Tensor q = rows ? q_ : q_.contiguous();
  Tensor out = at::empty(q.sizes(), q.options());
  if (B == 0) return out;
  Tensor ws = at::empty({static_cast<int64_t>(q3_paged_tree_workspace_bytes(static_cast<int32_t>(B),
                                                                            static_cast<int32_t>(T), ks.has_value()))},
                        q.options().dtype(ScalarType::Byte));
  p.q = q.data_ptr();
  p.q_seat_stride = B == 1 ? T * kHeads * kDim : q.stride(0);
  p.q_token_stride = T == 1 ? kHeads * kDim : q.stride(1);
  p.k_pool = kc.data_ptr();
  p.v_pool = vc.data_ptr();
  p.k_scale = ptr(ks);
  p.v_scale = ptr(vs);
  p.num_pages = static_cast<int32_t>(kc.size(0));
  p.page_size = static_cast<int32_t>(kc.size(1));
  p.cache_seqlens = seqlens.data_ptr<int32_t>();
  p.block_table = bt.data_ptr<int32_t>();
  p.block_table_stride = table_stride(bt);
  p.max_pages_per_seat = static_cast<int32_t>(bt.size(1));
  p.batch = static_cast<int32_t>(B);
  p.tokens = static_cast<int32_t>(T);
  p.num_heads = kHeads;
  p.num_kv_heads = kKvHeads;
  p.head_dim = kDim;
  p.softmax_scale = static_cast<float>(scale);
  p.out = out.data_ptr();
  p.out_seat_stride = T * kHeads * kDim;
  p.out_token_stride = kHeads * kDim;
  check(q3_paged_tree_attn(&p, ws.data_ptr(), ws.numel(), stream_of(q)), "q3_paged_tree_attn");
  return out;
}

Tensor decode_quant(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs,
                    const Tensor& seqlens, const Tensor& bt, double scale) {
  on_device(q, "q", q);
  TORCH_CHECK(q.dim() == 3 && q.size(1) == kHeads && q.size(2) == kDim, "q3attn: q must be [B, 16, 128], got ", q.sizes());
  q3_tree_attn p{};
  return attend(q, p, kc, vc, ks, vs, seqlens, bt, scale);
}

Tensor tree_attn(const Tensor& q, const Tensor& k_, const Tensor& v_, const Tensor& mask_, const Tensor& kc,
                 const Tensor& vc, const Tensor& seqlens, const Tensor& bt, double scale, const std::optional<Tensor>& ks,
                 const std::optional<Tensor>& vs, const std::optional<Tensor>& draft_lens) {
  on_device(q, "q", q);
  TORCH_CHECK(q.dim() == 4 && q.size(2) == kHeads && q.size(3) == kDim, "q3attn: q must be [B, T, 16, 128], got ", q.sizes());
  const int64_t B = q.size(0), T = q.size(1);
  TORCH_CHECK(T >= 1 && T <= 64, "q3attn: 1 to 64 drafted tokens a seat, got ", T);
  on_device(k_, "k", q);
  on_device(v_, "v", q);
  on_device(mask_, "tree_mask", q);
  TORCH_CHECK(k_.scalar_type() == ScalarType::BFloat16 && v_.scalar_type() == ScalarType::BFloat16 && k_.dim() == 4 &&
                  k_.size(0) == B && k_.size(1) == T && k_.size(2) == kKvHeads && k_.size(3) == kDim &&
                  v_.sizes() == k_.sizes(),
              "q3attn: k/v must be bfloat16 [B, T, 8, 128]");
  const bool rows = k_.strides() == v_.strides() && k_.stride(3) == 1 && k_.stride(2) == kDim &&
                    (T == 1 || k_.stride(1) >= kKvHeads * kDim);
  c10::cuda::OptionalCUDAGuard guard(q.device());
  const Tensor k = rows ? k_ : k_.contiguous(), v = rows ? v_ : v_.contiguous();
  TORCH_CHECK(mask_.scalar_type() == ScalarType::Long &&
                  ((mask_.dim() == 1 && mask_.size(0) == T) || (mask_.dim() == 2 && mask_.size(0) == B && mask_.size(1) == T)),
              "q3attn: tree_mask must be int64 [B, T] or [T]");
  const Tensor mask = T == 1 || mask_.stride(-1) == 1 ? mask_ : mask_.contiguous();
  q3_tree_attn p{};
  if (draft_lens.has_value()) {
    on_device(*draft_lens, "draft_lens", q);
    TORCH_CHECK(draft_lens->scalar_type() == ScalarType::Int && draft_lens->numel() == B && draft_lens->is_contiguous(),
                "q3attn: draft_lens must be a contiguous int32 tensor [B]");
    p.draft_lens = draft_lens->data_ptr<int32_t>();
  }
  p.k_new = k.data_ptr();
  p.v_new = v.data_ptr();
  p.kv_new_seat_stride = B == 1 ? T * kKvHeads * kDim : k.stride(0);
  p.kv_new_token_stride = T == 1 ? kKvHeads * kDim : k.stride(1);
  p.tree_mask = mask.data_ptr<int64_t>();
  p.tree_mask_stride = mask.dim() == 2 ? mask.stride(0) : 0;
  return attend(q, p, kc, vc, ks, vs, seqlens, bt, scale);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& ids_, int64_t top_n,
                                                          double temperature) {
  on_device(logits, "logits", logits);
  const ScalarType type = logits.scalar_type();
  TORCH_CHECK(type == ScalarType::BFloat16 || type == ScalarType::Float || type == ScalarType::Half,
              "q3attn: logits must be bfloat16, float16 or float32");
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= (1 << 30),
              "q3attn: logits must be [rows, vocab]");
  const int64_t n = logits.size(0), V = logits.size(1);
  TORCH_CHECK(top_n >= 0 && top_n <= 64 && top_n <= V, "q3attn: top_n must be 0 to 64, and no more than the vocabulary");
  TORCH_CHECK(temperature >= 1e-30 && temperature <= 1e30, "q3attn: temperature must be 1e-30 to 1e30");
  on_device(ids_, "ids", logits);
  TORCH_CHECK(ids_.scalar_type() == ScalarType::Long && (ids_.dim() == 1 || ids_.dim() == 2) && ids_.size(0) == n,
              "q3attn: ids must be int64 [rows] or [rows, given]");
  TORCH_CHECK(n <= (1 << 27) && (ids_.dim() == 1 || ids_.size(1) <= INT32_MAX), "q3attn: too many rows or ids");
  c10::cuda::OptionalCUDAGuard guard(logits.device());
  const Tensor x = (V == 1 || logits.stride(1) == 1) && (n <= 1 || logits.stride(0) >= V) ? logits : logits.contiguous();
  const Tensor ids = ids_.is_contiguous() ? ids_ : ids_.contiguous();
  const auto f32 = x.options().dtype(ScalarType::Float);
  Tensor lp = at::empty(ids.sizes(), f32), entropy = at::empty({n}, f32);
  Tensor top_ids = at::empty({n, top_n}, x.options().dtype(ScalarType::Long)), top_lp = at::empty({n, top_n}, f32);
  q3_logprobs p{};
  p.logits = x.data_ptr();
  p.logits_dtype = type == ScalarType::BFloat16 ? 0 : type == ScalarType::Float ? 1 : 2;
  p.row_stride = n <= 1 ? V : x.stride(0);
  p.rows = n;
  p.vocab = static_cast<int32_t>(V);
  p.temperature = static_cast<float>(temperature);
  p.ids = ids.data_ptr<int64_t>();
  p.given = ids.dim() == 1 ? 1 : static_cast<int32_t>(ids.size(1));
  p.ids_row_stride = p.given;
  p.logprobs = lp.data_ptr<float>();
  p.entropy = entropy.data_ptr<float>();
  p.top_n = static_cast<int32_t>(top_n);
  p.top_ids = top_ids.data_ptr<int64_t>();
  p.top_logprobs = top_lp.data_ptr<float>();
  check(q3_token_logprobs(&p, stream_of(x)), "q3_token_logprobs");
  return {lp, entropy, top_ids, top_lp};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(q3attn, m) {
  m.def("kv_quant_append_slots(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor slots) -> ()");
  m.def("kv_quant_append_paged(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor positions, Tensor block_table, Tensor? seat_of_row=None) -> ()");
  m.def("kv_dequant_paged(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor positions, "
        "Tensor block_table, Tensor? seat_of_row=None) -> (Tensor, Tensor)");
  m.def("paged_decode_quant(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor cache_seqlens, Tensor block_table, float softmax_scale) -> Tensor");
  m.def("paged_tree_attn(Tensor q, Tensor k, Tensor v, Tensor tree_mask, Tensor k_cache, Tensor v_cache, "
        "Tensor cache_seqlens, Tensor block_table, float softmax_scale, Tensor? k_scale=None, Tensor? v_scale=None, "
        "Tensor? draft_lens=None) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor ids, int top_n=0, float temperature=1.0) -> "
        "(Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(q3attn, CompositeExplicitAutograd, m) {
  m.impl("kv_quant_append_slots", append_slots);
  m.impl("kv_quant_append_paged", append_paged);
  m.impl("kv_dequant_paged", dequant_paged);
  m.impl("paged_decode_quant", decode_quant);
  m.impl("paged_tree_attn", tree_attn);
  m.impl("token_logprobs", token_logprobs);
}
