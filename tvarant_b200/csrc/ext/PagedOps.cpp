// The paged KV cache of many requests on the tvarant device: tvarant::page_plan
// (block tables and slot maps), paged_append_, paged_attention and
// paged_attention_append, and tvarant::adjust_logits with history_append_ and
// advance_tokens_ for the choice of the next token.  The reference has none of
// them.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <array>
#include <tuple>

#include "TvarantExt.h"

namespace tvarant::ops {
namespace {

void check_ints(const at::Tensor& t, at::ScalarType type, const at::Tensor& like, const char* op,
                const char* name) {
  TORCH_CHECK(t.scalar_type() == type && t.device() == like.device(), op, ": ", name, " must be ",
              type, " on ", like.device(), ", got ", t.scalar_type(), " on ", t.device());
}

// A dense vector of `n` values.
void check_vector(const at::Tensor& t, int64_t n, at::ScalarType type, const at::Tensor& like,
                  const char* op, const char* name) {
  check_ints(t, type, like, op, name);
  TORCH_CHECK(t.numel() == n && t.is_contiguous(), op, ": ", name, " must hold ", n,
              " contiguous values, got ", t.sizes());
}

int page_type(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat: return TVR_PAGE_F32;
    case at::kHalf: return TVR_PAGE_F16;
    case at::kBFloat16: return TVR_PAGE_BF16;
    default: TORCH_CHECK(false, op, ": pages are float32, float16 or bfloat16, got ", t.scalar_type());
  }
}

// k_pages, v_pages [pages, kv heads, page size, head dim], any strides with a
// contiguous last dimension.
tvr_paged_kv descriptor(const at::Tensor& k, const at::Tensor& v, const char* op) {
  TORCH_CHECK(is_device(k) && k.dim() == 4 && v.sizes() == k.sizes() &&
                  v.scalar_type() == k.scalar_type() && v.device() == k.device(),
              op, ": expected k_pages and v_pages [pages, heads, page size, dim] of one type, got ",
              k.sizes(), " and ", v.sizes());
  TORCH_CHECK(k.numel() == 0 || (k.stride(3) == 1 && v.stride(3) == 1), op,
              ": the pages' last dimension must be contiguous");
  tvr_paged_kv c = {};
  c.k_pages = k.data_ptr();
  c.v_pages = v.data_ptr();
  c.page_type = page_type(k, op);
  c.num_pages = k.size(0);
  c.kv_heads = k.size(1);
  c.page_size = k.size(2);
  c.head_dim = k.size(3);
  for (int i = 0; i < 3; ++i) {
    c.k_strides[i] = k.stride(i);
    c.v_strides[i] = v.stride(i);
  }
  return c;
}

at::Tensor unit_last(const at::Tensor& t) {
  return t.numel() == 0 || t.stride(-1) == 1 ? t : contiguous_copy(t);
}

// block_table [R, max pages] int32 and free_pages [pages] int32 are updated
// in place, seq_lens [R] and free_count [1] too; returns slots (int64),
// positions and rows (int32) of the step's tokens: packed [tokens], or
// [R, tokens_per_request] where that is given (tokens is then ignored).  A
// request has max_len positions at most (0: what its table row holds).
std::tuple<at::Tensor, at::Tensor, at::Tensor> page_plan(at::Tensor& block_table,
                                                         at::Tensor& seq_lens,
                                                         const at::Tensor& new_lens,
                                                         at::Tensor& free_pages,
                                                         at::Tensor& free_count, int64_t page_size,
                                                         int64_t tokens,
                                                         int64_t tokens_per_request,
                                                         int64_t max_len) {
  constexpr const char* op = "page_plan";
  TORCH_CHECK(is_device(block_table) && block_table.scalar_type() == at::kInt &&
                  block_table.dim() == 2 &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              op, ": block_table must be an int32 [requests, max pages] tvarant tensor");
  const int64_t n = block_table.size(0);
  check_vector(seq_lens, n, at::kInt, block_table, op, "seq_lens");
  check_vector(new_lens, n, at::kInt, block_table, op, "new_lens");
  check_vector(free_count, 1, at::kInt, block_table, op, "free_count");
  check_vector(free_pages, free_pages.numel(), at::kInt, block_table, op, "free_pages");
  TORCH_CHECK(tokens >= 0 && tokens_per_request >= 0, op, ": negative number of tokens");
  c10::DeviceGuard guard(block_table.device());
  const bool rows_form = tokens_per_request > 0;
  const int64_t total = rows_form ? n * tokens_per_request : tokens;
  const std::vector<int64_t> shape =
      rows_form ? std::vector<int64_t>{n, tokens_per_request} : std::vector<int64_t>{tokens};
  at::Tensor slots = empty_device(shape, block_table.options().dtype(at::kLong));
  at::Tensor positions = empty_device(shape, block_table.options());
  at::Tensor rows = empty_device(shape, block_table.options());
  tvr_page_pool pool = {};
  pool.block_table = static_cast<int32_t*>(block_table.data_ptr());
  pool.table_stride = block_table.stride(0);
  pool.max_pages = block_table.size(1);
  pool.requests = n;
  pool.free_pages = static_cast<int32_t*>(free_pages.data_ptr());
  pool.num_pages = free_pages.numel();
  pool.page_size = page_size;
  pool.max_positions = max_len;
  auto ints = [](const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
  TVR_TRY(tvr_page_plan(&pool, ints(seq_lens), ints(new_lens), ints(seq_lens), ints(free_count),
                        ints(free_count), static_cast<int64_t*>(slots.data_ptr()),
                        ints(positions), ints(rows), total, tokens_per_request,
                        current_stream_handle()));
  return {slots, positions, rows};
}

// k_new, v_new [tokens, kv heads, head dim] fp32 into the slots [tokens] of
// the pages, rounded to the pages' type.
void paged_append_(at::Tensor& k_pages, at::Tensor& v_pages, const at::Tensor& k_new,
                   const at::Tensor& v_new, const at::Tensor& slots) {
  constexpr const char* op = "paged_append_";
  const tvr_paged_kv c = descriptor(k_pages, v_pages, op);
  check_fp32(k_new, op);
  check_fp32(v_new, op);
  TORCH_CHECK(k_new.dim() == 3 && v_new.sizes() == k_new.sizes() && k_new.size(1) == c.kv_heads &&
                  k_new.size(2) == c.head_dim && k_new.device() == k_pages.device() &&
                  v_new.device() == k_pages.device(),
              op, ": expected k_new and v_new [tokens, ", c.kv_heads, ", ", c.head_dim, "], got ",
              k_new.sizes(), " and ", v_new.sizes());
  check_vector(slots, k_new.size(0), at::kLong, k_pages, op, "slots");
  c10::DeviceGuard guard(k_pages.device());
  const at::Tensor k = unit_last(k_new), v = unit_last(v_new);
  const int64_t strides[4] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
  TVR_TRY(tvr_paged_append(&c, static_cast<const float*>(k.data_ptr()),
                           static_cast<const float*>(v.data_ptr()), strides,
                           static_cast<const int64_t*>(slots.data_ptr()), k.size(0),
                           current_stream_handle()));
}

std::tuple<at::Tensor, at::Tensor> attend(const at::Tensor& q_in, const at::Tensor* k_new_in,
                                          const at::Tensor* v_new_in, const at::Tensor* slots,
                                          const at::Tensor& k_pages, const at::Tensor& v_pages,
                                          const at::Tensor& block_table, const at::Tensor& seq_lens,
                                          double scale, const at::Tensor& workspace,
                                          const char* op) {
  const tvr_paged_kv c = descriptor(k_pages, v_pages, op);
  check_fp32(q_in, op);
  TORCH_CHECK(q_in.dim() == 3 && q_in.size(2) == c.head_dim && q_in.device() == k_pages.device(),
              op, ": expected q [requests, heads, ", c.head_dim, "], got ", q_in.sizes());
  const int64_t n = q_in.size(0), heads = q_in.size(1);
  check_ints(block_table, at::kInt, k_pages, op, "block_table");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == n &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              op, ": block_table must be [", n, ", max pages], got ", block_table.sizes());
  check_vector(seq_lens, n, at::kInt, k_pages, op, "seq_lens");
  check_ints(workspace, at::kByte, k_pages, op, "workspace");
  TORCH_CHECK(workspace.is_contiguous(), op, ": the workspace must be contiguous");
  c10::DeviceGuard guard(q_in.device());
  const at::Tensor q = unit_last(q_in);
  at::Tensor k_new, v_new;
  if (slots != nullptr) {
    for (const at::Tensor* t : {k_new_in, v_new_in}) {
      check_fp32(*t, op);
      TORCH_CHECK(t->dim() == 3 && t->size(0) == n && t->size(1) == c.kv_heads &&
                      t->size(2) == c.head_dim && t->device() == k_pages.device(),
                  op, ": expected k_new and v_new [", n, ", ", c.kv_heads, ", ", c.head_dim,
                  "], got ", t->sizes());
    }
    check_vector(*slots, n, at::kLong, k_pages, op, "slots");
    k_new = unit_last(*k_new_in);
    v_new = unit_last(*v_new_in);
  }
  at::Tensor out = empty_device({n, heads, c.head_dim}, q.options());
  at::Tensor lse = empty_device({n, heads}, q.options());
  const int64_t strides[8] = {
      q.stride(0), q.stride(1), slots ? k_new.stride(0) : 0, slots ? k_new.stride(1) : 0,
      slots ? v_new.stride(0) : 0, slots ? v_new.stride(1) : 0, heads * c.head_dim, c.head_dim};
  TVR_TRY(tvr_paged_attention(
      &c, static_cast<const float*>(q.data_ptr()),
      slots ? static_cast<const float*>(k_new.data_ptr()) : nullptr,
      slots ? static_cast<const float*>(v_new.data_ptr()) : nullptr,
      slots ? static_cast<const int64_t*>(slots->data_ptr()) : nullptr,
      static_cast<const int32_t*>(block_table.data_ptr()), block_table.stride(0),
      block_table.size(1), static_cast<const int32_t*>(seq_lens.data_ptr()),
      static_cast<float*>(out.data_ptr()), static_cast<float*>(lse.data_ptr()), n, heads, strides,
      static_cast<float>(scale), workspace.data_ptr(), workspace.numel(),
      current_stream_handle()));
  return {out, lse};
}

// q [R, heads, dim] over the first seq_lens[r] positions of each request's
// pages; returns out and lse [R, heads].
std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor& q, const at::Tensor& k_pages,
                                                   const at::Tensor& v_pages,
                                                   const at::Tensor& block_table,
                                                   const at::Tensor& seq_lens, double scale,
                                                   at::Tensor& workspace) {
  return attend(q, nullptr, nullptr, nullptr, k_pages, v_pages, block_table, seq_lens, scale,
                workspace, "paged_attention");
}

// The same after paged_append_(k_pages, v_pages, k_new, v_new, slots), in one
// launch; slots [R] are the requests' last positions' slots, -1 for none.
std::tuple<at::Tensor, at::Tensor> paged_attention_append(
    const at::Tensor& q, const at::Tensor& k_new, const at::Tensor& v_new, at::Tensor& k_pages,
    at::Tensor& v_pages, const at::Tensor& slots, const at::Tensor& block_table,
    const at::Tensor& seq_lens, double scale, at::Tensor& workspace) {
  return attend(q, &k_new, &v_new, &slots, k_pages, v_pages, block_table, seq_lens, scale,
                workspace, "paged_attention_append");
}

int64_t paged_attention_workspace(int64_t heads, int64_t kv_heads, int64_t head_dim) {
  int64_t bytes = 0;
  TVR_TRY(tvr_paged_attention_workspace(heads, kv_heads, head_dim, &bytes));
  return bytes;
}

using OptTensor = std::optional<at::Tensor>;

at::Tensor adjust_logits(const at::Tensor& logits_in, const OptTensor& tokens,
                         const OptTensor& prompt_lens, const OptTensor& total_lens,
                         const OptTensor& repetition, const OptTensor& presence,
                         const OptTensor& frequency, const OptTensor& bias_ids,
                         const OptTensor& bias_values, const OptTensor& bias_counts,
                         const OptTensor& masks, const OptTensor& mask_rows) {
  constexpr const char* op = "adjust_logits";
  check_fp32(logits_in, op);
  TORCH_CHECK(logits_in.dim() == 2, op, ": expected logits [rows, vocab], got ", logits_in.sizes());
  c10::DeviceGuard guard(logits_in.device());
  const at::Tensor x = unit_last(logits_in);
  const int64_t rows = x.size(0), vocab = x.size(1);
  tvr_logit_rules r = {};
  // a [rows] vector of int32 or float32
  auto vec = [&](const OptTensor& t, at::ScalarType type, const char* name) -> const void* {
    if (!t.has_value() || !t->defined()) return nullptr;
    check_vector(*t, rows, type, x, op, name);
    return t->data_ptr();
  };
  // a [rows', columns] array with contiguous rows
  auto array = [&](const OptTensor& t, const char* name) -> bool {
    if (!t.has_value() || !t->defined()) return false;
    TORCH_CHECK(t->dim() == 2 && t->device() == x.device() &&
                    (t->size(1) <= 1 || t->stride(1) == 1),
                op, ": ", name, " must be two-dimensional with contiguous rows on ", x.device());
    return true;
  };
  if (array(tokens, "tokens")) {
    TORCH_CHECK(tokens->size(0) == rows &&
                    (tokens->scalar_type() == at::kLong || tokens->scalar_type() == at::kInt),
                op, ": tokens must be int32 or int64 [", rows, ", history], got ", tokens->sizes());
    // the library bounds a history by its row stride
    TORCH_CHECK(tokens->is_contiguous(), op, ": tokens must be contiguous");
    r.tokens = tokens->data_ptr();
    r.token_bits = tokens->scalar_type() == at::kLong ? 64 : 32;
    r.tokens_stride = tokens->size(1);
    TORCH_CHECK(total_lens.has_value() && total_lens->defined(), op, ": tokens need total_lens");
    r.total_lens = static_cast<const int32_t*>(vec(total_lens, at::kInt, "total_lens"));
    r.prompt_lens = static_cast<const int32_t*>(vec(prompt_lens, at::kInt, "prompt_lens"));
  }
  r.repetition = static_cast<const float*>(vec(repetition, at::kFloat, "repetition"));
  r.presence = static_cast<const float*>(vec(presence, at::kFloat, "presence"));
  r.frequency = static_cast<const float*>(vec(frequency, at::kFloat, "frequency"));
  if (array(bias_ids, "bias_ids")) {
    check_ints(*bias_ids, at::kInt, x, op, "bias_ids");
    TORCH_CHECK(bias_values.has_value() && bias_values->defined() &&
                    bias_values->sizes() == bias_ids->sizes() && bias_ids->size(0) == rows &&
                    bias_values->scalar_type() == at::kFloat && bias_values->device() == x.device() &&
                    bias_ids->is_contiguous() && bias_values->is_contiguous(),
                op, ": bias_ids (int32) and bias_values (float32) must be contiguous [", rows,
                ", biases]");
    r.bias_ids = static_cast<const int32_t*>(bias_ids->data_ptr());
    r.bias_values = static_cast<const float*>(bias_values->data_ptr());
    r.bias_counts = static_cast<const int32_t*>(vec(bias_counts, at::kInt, "bias_counts"));
    r.bias_stride = bias_ids->size(1);
  }
  if (array(masks, "masks")) {
    check_ints(*masks, at::kInt, x, op, "masks");
    TORCH_CHECK(masks->size(1) >= (vocab + 31) / 32, op, ": masks have ", masks->size(1),
                " words a row, expected ", (vocab + 31) / 32);
    r.masks = static_cast<const uint32_t*>(masks->data_ptr());
    r.mask_stride = masks->stride(0);
    r.n_masks = masks->size(0);
    r.mask_rows = static_cast<const int32_t*>(vec(mask_rows, at::kInt, "mask_rows"));
  }
  at::Tensor out = empty_device({rows, vocab}, x.options());
  TVR_TRY(tvr_adjust_logits(static_cast<const float*>(x.data_ptr()), x.stride(0),
                            static_cast<float*>(out.data_ptr()), vocab, rows, vocab, &r,
                            current_stream_handle()));
  return out;
}

// tokens[r, lens[r]] = ids[r] and lens[r] += 1 where live[r] > 0 and the row
// has room (tvr_history_append).
void history_append_(at::Tensor& tokens, at::Tensor& lens, const at::Tensor& ids,
                     const OptTensor& live) {
  constexpr const char* op = "history_append_";
  TORCH_CHECK(is_device(tokens) && tokens.dim() == 2 && tokens.is_contiguous() &&
                  (tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt),
              op, ": tokens must be a contiguous int32 or int64 [rows, history] tvarant tensor");
  const int64_t rows = tokens.size(0);
  check_vector(lens, rows, at::kInt, tokens, op, "lens");
  check_vector(ids, rows, at::kLong, tokens, op, "ids");
  const bool some = live.has_value() && live->defined();
  if (some) check_vector(*live, rows, at::kInt, tokens, op, "live");
  c10::DeviceGuard guard(tokens.device());
  TVR_TRY(tvr_history_append(tokens.data_ptr(), tokens.scalar_type() == at::kLong ? 64 : 32,
                             tokens.size(1), static_cast<int32_t*>(lens.data_ptr()),
                             static_cast<const int64_t*>(ids.data_ptr()),
                             some ? static_cast<const int32_t*>(live->data_ptr()) : nullptr, rows,
                             tokens.size(1), current_stream_handle()));
}

// current[r] = next[r] for the rows with slots[r] >= 0, whose histories (tokens
// and lens, both or none) take next[r] too (tvr_advance_tokens).
void advance_tokens_(at::Tensor& current, const at::Tensor& next, const at::Tensor& slots,
                     std::optional<at::Tensor> tokens, std::optional<at::Tensor> lens) {
  constexpr const char* op = "advance_tokens_";
  TORCH_CHECK(is_device(current), op, ": expected tvarant tensors");
  const int64_t rows = current.numel();
  check_vector(current, rows, at::kLong, current, op, "current");
  check_vector(next, rows, at::kLong, current, op, "next");
  check_vector(slots, rows, at::kLong, current, op, "slots");
  const bool some = tokens.has_value() && tokens->defined();
  TORCH_CHECK(some == (lens.has_value() && lens->defined()), op, ": tokens and lens come together");
  if (some) {
    TORCH_CHECK(tokens->device() == current.device() && tokens->dim() == 2 &&
                    tokens->size(0) == rows && tokens->is_contiguous() &&
                    (tokens->scalar_type() == at::kLong || tokens->scalar_type() == at::kInt),
                op, ": tokens must be contiguous int32 or int64 [", rows, ", history], got ",
                tokens->sizes());
    check_vector(*lens, rows, at::kInt, current, op, "lens");
  }
  c10::DeviceGuard guard(current.device());
  const int64_t capacity = some ? tokens->size(1) : 0;
  TVR_TRY(tvr_advance_tokens(
      static_cast<int64_t*>(current.data_ptr()), static_cast<const int64_t*>(next.data_ptr()),
      static_cast<const int64_t*>(slots.data_ptr()), some ? tokens->data_ptr() : nullptr,
      some && tokens->scalar_type() == at::kLong ? 64 : 32, capacity,
      some ? static_cast<int32_t*>(lens->data_ptr()) : nullptr, rows, capacity,
      current_stream_handle()));
}

}  // namespace
}  // namespace tvarant::ops

TORCH_LIBRARY_FRAGMENT(tvarant, m) {
  m.def("page_plan(Tensor(a!) block_table, Tensor(b!) seq_lens, Tensor new_lens, "
        "Tensor(c!) free_pages, Tensor(d!) free_count, int page_size, int tokens, "
        "int tokens_per_request=0, int max_len=0) -> (Tensor, Tensor, Tensor)");
  m.def("paged_append_(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor k_new, Tensor v_new, "
        "Tensor slots) -> ()");
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, "
        "Tensor seq_lens, float scale, Tensor(a!) workspace) -> (Tensor, Tensor)");
  m.def("paged_attention_append(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_pages, "
        "Tensor(b!) v_pages, Tensor slots, Tensor block_table, Tensor seq_lens, float scale, "
        "Tensor(c!) workspace) -> (Tensor, Tensor)");
  m.def("paged_attention_workspace(int heads, int kv_heads, int head_dim) -> int",
        &tvarant::ops::paged_attention_workspace);
  m.def("adjust_logits(Tensor logits, Tensor? tokens=None, Tensor? prompt_lens=None, "
        "Tensor? total_lens=None, Tensor? repetition=None, Tensor? presence=None, "
        "Tensor? frequency=None, Tensor? bias_ids=None, Tensor? bias_values=None, "
        "Tensor? bias_counts=None, Tensor? masks=None, Tensor? mask_rows=None) -> Tensor");
  m.def("history_append_(Tensor(a!) tokens, Tensor(b!) lens, Tensor ids, Tensor? live=None) -> ()");
  m.def("advance_tokens_(Tensor(a!) current, Tensor next, Tensor slots, Tensor(b!)? tokens=None, "
        "Tensor(c!)? lens=None) -> ()");
}

TORCH_LIBRARY_IMPL(tvarant, PrivateUse1, m) {
  m.impl("page_plan", TORCH_FN(tvarant::ops::page_plan));
  m.impl("paged_append_", TORCH_FN(tvarant::ops::paged_append_));
  m.impl("paged_attention", TORCH_FN(tvarant::ops::paged_attention));
  m.impl("paged_attention_append", TORCH_FN(tvarant::ops::paged_attention_append));
  m.impl("adjust_logits", TORCH_FN(tvarant::ops::adjust_logits));
  m.impl("history_append_", TORCH_FN(tvarant::ops::history_append_));
  m.impl("advance_tokens_", TORCH_FN(tvarant::ops::advance_tokens_));
}
