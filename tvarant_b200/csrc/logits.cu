// Logits of a decode step adjusted before the next token is chosen
// (tvr_adjust_logits): penalties for tokens of the history, sparse biases,
// grammar masks; and the histories' growth by the chosen tokens
// (tvr_history_append).
#include "internal.h"

#include <cmath>
#include <cstring>

namespace tvr {
namespace {

// One pass over the logits: 4 bytes read and 4 written per logit, plus the
// row's history (4 or 8 bytes a token, read once per slice) and its mask bits.
// A CTA takes a slice of one row's vocabulary:
//   1. counts the row's history tokens that fall into the slice, in shared
//      memory (whole numbers: the order of the atomics does not matter); the
//      top bit says that the token is in the prompt;
//   2. streams the slice, applying penalties and the mask;
//   3. adds the slice's biases to what it wrote, each token's in list order:
//      the first entry of a token's id takes all of them.
constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;

struct LogitParams {
  const float* x;
  float* y;
  int64_t x_stride, y_stride;
  int vocab;
  int slice;
  tvr_logit_rules r;
  int* status;
};

__device__ __forceinline__ float penalise(float x, uint32_t c, float rep, float freq, float pres) {
  if (c == 0) return x;
  x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
  const uint32_t made = c & ~kPrompt;
  if (made != 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(made))), pres);
  return x;
}

__global__ void __launch_bounds__(kThreads)
    adjust_logits_kernel(const __grid_constant__ LogitParams p) {
  extern __shared__ uint32_t s_count[];
  const int row = blockIdx.y;
  const int v0 = blockIdx.x * p.slice, n = min(p.slice, p.vocab - v0);
  const float* x = p.x + row * p.x_stride + v0;
  float* y = p.y + row * p.y_stride + v0;
  const tvr_logit_rules& r = p.r;

  for (int i = threadIdx.x; i < p.slice; i += kThreads) s_count[i] = 0;
  __syncthreads();
  if (r.tokens != nullptr) {
    const int total =
        static_cast<int>(max(static_cast<int64_t>(0),
                             min(static_cast<int64_t>(r.total_lens[row]), r.tokens_stride)));
    const int prompt = r.prompt_lens != nullptr ? r.prompt_lens[row] : 0;
    for (int i = threadIdx.x; i < total; i += kThreads) {
      const int64_t at = row * r.tokens_stride + i;
      const int64_t t = (r.token_bits == 64 ? static_cast<const int64_t*>(r.tokens)[at]
                                            : static_cast<const int32_t*>(r.tokens)[at]) - v0;
      if (t < 0 || t >= n) continue;
      if (i < prompt) {
        atomicOr(&s_count[t], kPrompt);
      } else {
        atomicAdd(&s_count[t], 1u);
      }
    }
    __syncthreads();
  }
  const float rep = r.repetition != nullptr ? r.repetition[row] : 1.f;
  const float pres = r.presence != nullptr ? r.presence[row] : 0.f;
  const float freq = r.frequency != nullptr ? r.frequency[row] : 0.f;
  const uint32_t* mask = nullptr;
  if (r.masks != nullptr) {
    const int64_t m = r.mask_rows != nullptr ? r.mask_rows[row] : row;
    if (m >= r.n_masks) {
      if (threadIdx.x == 0 && blockIdx.x == 0 && p.status != nullptr) {
        atomicCAS(p.status, TVR_DEV_OK, TVR_DEV_BAD_INDEX);
      }
    } else if (m >= 0) {
      mask = r.masks + m * r.mask_stride;
    }
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float z = penalise(x[i], s_count[i], rep, freq, pres);
    const int v = v0 + i;
    if (mask != nullptr && ((mask[v >> 5] >> (v & 31)) & 1u) == 0) z = -INFINITY;
    y[i] = z;
  }
  if (r.bias_ids == nullptr) return;
  const int biases = static_cast<int>(
      r.bias_counts != nullptr
          ? max(static_cast<int64_t>(0),
                min(static_cast<int64_t>(r.bias_counts[row]), r.bias_stride))
          : r.bias_stride);
  const int32_t* ids = r.bias_ids + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  // the counters become "the first list entry of this token"
  __syncthreads();
  for (int i = threadIdx.x; i < biases; i += kThreads) {
    const int64_t t = static_cast<int64_t>(ids[i]) - v0;
    if (t >= 0 && t < n) s_count[t] = 0xffffffffu;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < biases; i += kThreads) {
    const int64_t t = static_cast<int64_t>(ids[i]) - v0;
    if (t >= 0 && t < n) atomicMin(&s_count[t], static_cast<uint32_t>(i));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < biases; i += kThreads) {
    const int64_t t = static_cast<int64_t>(ids[i]) - v0;
    if (t < 0 || t >= n || s_count[t] != static_cast<uint32_t>(i)) continue;
    const int v = static_cast<int>(t) + v0;
    if (mask != nullptr && ((mask[v >> 5] >> (v & 31)) & 1u) == 0) continue;
    float z = y[t];
    for (int j = i; j < biases; ++j) {
      if (ids[j] == v) z = __fadd_rn(z, values[j]);
    }
    y[t] = z;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    history_append_kernel(T* tokens, int64_t stride, int32_t* lens, const int64_t* ids,
                          const int32_t* live, int64_t rows, int64_t capacity) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (row >= rows || (live != nullptr && live[row] <= 0)) return;
  const int at = lens[row];
  if (at < 0 || at >= capacity) return;
  tokens[row * stride + at] = static_cast<T>(ids[row]);
  lens[row] = at + 1;
}

}  // namespace
}  // namespace tvr

using namespace tvr;

extern "C" int tvr_adjust_logits(const float* logits, int64_t logits_stride, float* out,
                                 int64_t out_stride, int64_t rows, int64_t vocab,
                                 const tvr_logit_rules* rules, void* stream) {
  TVR_CHECK(rows >= 0 && vocab >= 0, "adjust_logits: negative size");
  TVR_CHECK(rules != nullptr, "adjust_logits: null rules");
  if (rows == 0 || vocab == 0) return TVR_OK;
  TVR_CHECK(logits && out, "adjust_logits: null pointer");
  TVR_CHECK(rows <= 65535 && vocab <= 0x40000000, "adjust_logits: too many rows or tokens");
  TVR_CHECK(rows == 1 || (logits_stride >= vocab && out_stride >= vocab),
            "adjust_logits: a row stride is less than the vocabulary");
  TVR_CHECK(logits != out || rows == 1 || logits_stride == out_stride,
            "adjust_logits: in place with two strides");
  const tvr_logit_rules& r = *rules;
  if (r.tokens != nullptr) {
    TVR_CHECK(r.token_bits == 32 || r.token_bits == 64, "adjust_logits: token_bits %d", r.token_bits);
    TVR_CHECK(r.total_lens != nullptr, "adjust_logits: a history without lengths");
    TVR_CHECK(r.tokens_stride >= 0 && r.tokens_stride <= 0x7fffffff,
              "adjust_logits: history stride %lld", (long long)r.tokens_stride);
  }
  if (r.bias_ids != nullptr) {
    TVR_CHECK(r.bias_values != nullptr, "adjust_logits: bias ids without values");
    TVR_CHECK(r.bias_stride >= 0 && r.bias_stride <= 0x7fffffff, "adjust_logits: bias stride %lld",
              (long long)r.bias_stride);
  }
  if (r.masks != nullptr) {
    TVR_CHECK(r.mask_stride >= ceil_div(vocab, 32) || r.n_masks <= 1,
              "adjust_logits: a mask row of %lld words is less than the vocabulary",
              (long long)r.mask_stride);
    TVR_CHECK(r.mask_rows != nullptr || r.n_masks >= rows, "adjust_logits: fewer masks than rows");
  }
  LogitParams p;
  memset(&p, 0, sizeof(p));
  p.x = logits;
  p.y = out;
  p.x_stride = logits_stride;
  p.y_stride = out_stride;
  p.vocab = static_cast<int>(vocab);
  p.slice = 8192;
  p.r = r;
  p.status = device_status_ptr(current_device());
  const dim3 grid(static_cast<unsigned>(ceil_div(vocab, p.slice)), static_cast<unsigned>(rows));
  adjust_logits_kernel<<<grid, kThreads, p.slice * 4, as_stream(stream)>>>(p);
  TVR_LAUNCH_CHECK();
  return TVR_OK;
}

extern "C" int tvr_history_append(void* tokens, int token_bits, int64_t tokens_stride,
                                  int32_t* lens, const int64_t* ids, const int32_t* live,
                                  int64_t rows, int64_t capacity, void* stream) {
  TVR_CHECK(rows >= 0 && capacity >= 0, "history_append: negative size");
  TVR_CHECK(token_bits == 32 || token_bits == 64, "history_append: token_bits %d", token_bits);
  TVR_CHECK(capacity <= 0x7fffffff && rows <= 0x7fffffff, "history_append: size past 32 bits");
  if (rows == 0) return TVR_OK;
  TVR_CHECK(lens && ids && (tokens || capacity == 0), "history_append: null pointer");
  TVR_CHECK(rows == 1 || tokens_stride >= capacity,
            "history_append: the row stride is less than the capacity");
  const unsigned grid = static_cast<unsigned>(ceil_div(rows, kThreads));
  if (token_bits == 64) {
    history_append_kernel<int64_t><<<grid, kThreads, 0, as_stream(stream)>>>(
        static_cast<int64_t*>(tokens), tokens_stride, lens, ids, live, rows, capacity);
  } else {
    history_append_kernel<int32_t><<<grid, kThreads, 0, as_stream(stream)>>>(
        static_cast<int32_t*>(tokens), tokens_stride, lens, ids, live, rows, capacity);
  }
  TVR_LAUNCH_CHECK();
  return TVR_OK;
}
