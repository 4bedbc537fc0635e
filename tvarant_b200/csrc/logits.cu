// Logits of a decode step adjusted before the next token is chosen
// (tvr_adjust_logits): penalties for tokens of the history, sparse biases,
// grammar masks; and the histories' growth by the chosen tokens
// (tvr_history_append).
#include "tc_ptx.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

namespace tvr {
namespace {

// One pass over the logits: 4 bytes read and 4 written per logit, plus the
// row's history (4 or 8 bytes a token, read by every slice from L2) and its
// mask bits.  A CTA takes a slice of one row's vocabulary, of which a bulk copy
// brings the logits into shared memory while it
//   1. counts the row's history tokens that fall into the slice (whole
//      numbers: the order of the atomics does not matter) and marks the
//      slice's biased tokens, those with several biases in `twice`;
//   2. applies penalties and the mask;
//   3. adds the biases, several of one token by the warp of the first, in list
//      order; then a bulk copy takes the slice out.
// What bounds a long history is that each slice reads all of it.  Sharing it
// out over a cluster measured slower, in every form tried: atomics on one
// another's counters 262 us, against 158, for 400 rows of 129280 logits and
// 15000 tokens; sorting it by slices with atomics that return places, 590.
constexpr int kThreads = 512;
constexpr int kMinSlice = 4 * kThreads;
constexpr int kMaxSlice = 8192;
constexpr uint32_t kPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;
constexpr uint32_t kNone = 0xffffffffu;

struct LogitParams {
  const float* x;
  float* y;
  int64_t x_stride, y_stride;
  int vocab;
  int slice;  // a multiple of kMinSlice
  tvr_logit_rules r;
  int* status;
};

struct RowRules {
  float rep, inverse, freq, pres;
};

// Without branches: in a long history nearly every warp has a token of it.
__device__ __forceinline__ float adjust(float x, uint32_t c, bool allowed, const RowRules& r) {
  const float made = static_cast<float>(c & kCount);
  const float factor = x > 0.f ? r.inverse : r.rep;
  x = __fmul_rn(x, (c & (kPrompt | kCount)) != 0 ? factor : 1.f);
  x = __fsub_rn(x, made > 0.f ? __fmul_rn(r.freq, made) : 0.f);
  x = __fsub_rn(x, made > 0.f ? r.pres : 0.f);
  return allowed ? x : -INFINITY;
}

// f(token - v0) for the n tokens, as an unsigned number: what is outside a slice
// that begins at v0 is past its end.  Several loads of a thread are under way:
// one at a time is what bounds a long history (265 us, then 155 us, for 400
// rows of 129280 logits and 15000 tokens).
template <typename F>
__device__ __forceinline__ void scan_tokens(const int64_t* tokens, int n, int v0, const F& f) {
  for (int first = threadIdx.x; first < n; first += 8 * kThreads) {
    int64_t t[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const int i = first + b * kThreads;
      t[b] = i < n ? __ldg(tokens + i) - v0 : -1;
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      f(static_cast<uint64_t>(t[b]) < kNone ? static_cast<uint32_t>(t[b]) : kNone);
    }
  }
}
template <typename F>
__device__ __forceinline__ void scan_tokens(const int32_t* tokens, int n, int v0, const F& f) {
  const uint32_t base = static_cast<uint32_t>(v0);
  auto one = [&](int i) {
    if (i < n) f(static_cast<uint32_t>(__ldg(tokens + i)) - base);
  };
  // a few, fours on 16-byte boundaries, a few
  const int head = min(n, static_cast<int>((0 - (reinterpret_cast<uintptr_t>(tokens) >> 2)) & 3));
  const int quads = (n - head) / 4;
  const int4* const t4 = reinterpret_cast<const int4*>(tokens + head);
  for (int first = threadIdx.x; first < quads; first += 4 * kThreads) {
    int4 t[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int g = first + b * kThreads;
      t[b] = g < quads ? __ldg(t4 + g) : make_int4(-1, -1, -1, -1);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f(static_cast<uint32_t>(t[b].x) - base);
      f(static_cast<uint32_t>(t[b].y) - base);
      f(static_cast<uint32_t>(t[b].z) - base);
      f(static_cast<uint32_t>(t[b].w) - base);
    }
  }
  if (threadIdx.x < head) one(threadIdx.x);
  if (threadIdx.x < 4) one(head + 4 * quads + threadIdx.x);
}

// The counter of token t of a slice of n, where t < n.  Predicated: a branch
// around the atomic of each token costs twice its work.
__device__ __forceinline__ void count_one(uint32_t counters, uint32_t t, uint32_t n) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.lt.u32 p, %1, %2;\n\t"
      "@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(counters + 4 * t),
      "r"(t), "r"(n)
      : "memory");
}
__device__ __forceinline__ void mark_prompt(uint32_t counters, uint32_t t, uint32_t n) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.lt.u32 p, %1, %2;\n\t"
      "@p red.shared.or.b32 [%0], %3;\n\t}" ::"r"(counters + 4 * t),
      "r"(t), "r"(n), "r"(kPrompt)
      : "memory");
}

// Words of shared memory: counters, logits, mask words and `twice`.
inline int64_t smem_words(int64_t slice) { return 2 * (slice + 4) + (slice / 32 + 4) + slice / 32; }

// VECTOR: x and y lie alike on 16-byte boundaries.
template <bool VECTOR>
__global__ void __launch_bounds__(kThreads)
    adjust_logits_kernel(const __grid_constant__ LogitParams p) {
  extern __shared__ __align__(16) uint32_t s_words[];
  __shared__ uint64_t s_bar;
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int v0 = blockIdx.x * p.slice, n = min(p.slice, p.vocab - v0);
  const float* x = p.x + row * p.x_stride + v0;
  float* y = p.y + row * p.y_stride + v0;
  const tvr_logit_rules& r = p.r;

  // Token i of the slice is word i + shift of the counters and of the logits,
  // so that what is on a 16-byte boundary in memory is on one here.  Logits
  // [lead, lead + 4 groups) go by fours.
  const int shift = VECTOR ? static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3) : 0;
  const int lead = VECTOR ? min(n, (4 - shift) & 3) : n;
  const int groups = (n - lead) / 4;
  uint32_t* const count = s_words + shift;
  float* const z = reinterpret_cast<float*>(s_words + p.slice + 4) + shift;
  uint32_t* const allowed = s_words + 2 * (p.slice + 4);
  uint32_t* const twice = allowed + p.slice / 32 + 4;
  const uint32_t bar = tc::smem_u32(&s_bar);
  if (VECTOR && tid == 0) {
    tc::mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::mbar_expect_tx(bar, 16 * groups);
    if (groups > 0) {
      asm volatile(
          "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, "
          "[%3];" ::"r"(tc::smem_u32(z + lead)),
          "l"(x + lead), "r"(16 * groups), "r"(bar)
          : "memory");
    }
  }

  RowRules rules;
  rules.rep = r.repetition != nullptr ? r.repetition[row] : 1.f;
  rules.inverse = __fdiv_rn(1.f, rules.rep);
  rules.pres = r.presence != nullptr ? r.presence[row] : 0.f;
  rules.freq = r.frequency != nullptr ? r.frequency[row] : 0.f;
  const int64_t held = r.tokens != nullptr ? r.total_lens[row] : 0;
  const int prompt = r.tokens != nullptr && r.prompt_lens != nullptr ? r.prompt_lens[row] : 0;
  const int64_t biased =
      r.bias_ids == nullptr ? 0 : r.bias_counts != nullptr ? r.bias_counts[row] : r.bias_stride;
  int64_t m = r.masks == nullptr ? -1 : r.mask_rows != nullptr ? r.mask_rows[row] : row;
  if (m >= r.n_masks) {
    if (tid == 0 && blockIdx.x == 0 && p.status != nullptr) {
      atomicCAS(p.status, TVR_DEV_OK, TVR_DEV_BAD_INDEX);
    }
    m = -1;
  }
  const int total = static_cast<int>(max(int64_t(0), min(held, r.tokens_stride)));
  const int biases = static_cast<int>(max(int64_t(0), min(biased, r.bias_stride)));
  const int32_t* ids = r.bias_ids + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  const int32_t first_id = tid < biases ? ids[tid] : -1;  // this thread's first bias
  const float first_value = tid < biases ? values[tid] : 0.f;

  // v0 is a multiple of 32
  const uint32_t* mask = m >= 0 ? r.masks + m * r.mask_stride + v0 / 32 : nullptr;
  for (int i = tid; i < (n + 31) / 32; i += kThreads) allowed[i] = mask != nullptr ? mask[i] : ~0u;
  for (int i = tid; i < (p.slice + 4) / 4; i += kThreads) {
    reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
  }
  for (int i = tid; i < p.slice / 32; i += kThreads) twice[i] = 0;
  __syncthreads();
  if (total > 0) {
    // the prompt's part and what was generated; the marks and counts of a
    // token are in other bits, so their order does not matter
    const int64_t base = row * r.tokens_stride;
    const int made_from = max(0, min(prompt, total));
    const uint32_t counters = tc::smem_u32(count);
    const uint32_t nu = static_cast<uint32_t>(n);
    auto mark = [&](uint32_t t) { mark_prompt(counters, t, nu); };
    auto tally = [&](uint32_t t) { count_one(counters, t, nu); };
    if (r.token_bits == 64) {
      const int64_t* tokens = static_cast<const int64_t*>(r.tokens) + base;
      scan_tokens(tokens, made_from, v0, mark);
      scan_tokens(tokens + made_from, total - made_from, v0, tally);
    } else {
      const int32_t* tokens = static_cast<const int32_t*>(r.tokens) + base;
      scan_tokens(tokens, made_from, v0, mark);
      scan_tokens(tokens + made_from, total - made_from, v0, tally);
    }
  }
  for (int i = tid; i < biases; i += kThreads) {
    const int64_t t = static_cast<int64_t>(i == tid ? first_id : ids[i]) - v0;
    if (t < 0 || t >= n) continue;
    if ((atomicOr(&count[t], kBiased) & kBiased) != 0) atomicOr(&twice[t >> 5], 1u << (t & 31));
  }
  __syncthreads();

  auto allowed_at = [&](int i) { return ((allowed[i >> 5] >> (i & 31)) & 1u) != 0; };
  if (VECTOR) {
    if (!tc::mbar_wait(bar, 0, nullptr) && p.status != nullptr) {
      atomicCAS(p.status, TVR_DEV_OK, TVR_DEV_TIMEOUT_MMA);
    }
#pragma unroll 2
    for (int g = tid; g < groups; g += kThreads) {
      const int i = lead + 4 * g, at = i & 31;
      // the word after the last one is read, but not used
      const uint32_t bits =
          mask != nullptr ? __funnelshift_r(allowed[i >> 5], allowed[(i >> 5) + 1], at) & 15u : 15u;
      const uint4 c = *reinterpret_cast<const uint4*>(count + i);
      if (((c.x | c.y | c.z | c.w) & (kPrompt | kCount)) == 0 && bits == 15u) continue;
      float4 v = *reinterpret_cast<const float4*>(z + i);
      v.x = adjust(v.x, c.x, (bits & 1u) != 0, rules);
      v.y = adjust(v.y, c.y, (bits & 2u) != 0, rules);
      v.z = adjust(v.z, c.z, (bits & 4u) != 0, rules);
      v.w = adjust(v.w, c.w, (bits & 8u) != 0, rules);
      *reinterpret_cast<float4*>(z + i) = v;
    }
    if (tid < 4) {  // what is not on a boundary: the first, and the last, few
      const int rest = lead + 4 * groups + tid;
      if (tid < lead) z[tid] = adjust(x[tid], count[tid], allowed_at(tid), rules);
      if (rest < n) z[rest] = adjust(x[rest], count[rest], allowed_at(rest), rules);
    }
  } else {
    for (int i = tid; i < n; i += kThreads) z[i] = adjust(x[i], count[i], allowed_at(i), rules);
  }
  if (biases > 0) {
    __syncthreads();
    for (int base = tid - lane; base < biases; base += kThreads) {
      const int i = base + lane;
      const int id = i >= biases ? -1 : i == tid ? first_id : ids[i];
      const int64_t t = static_cast<int64_t>(id) - v0;
      const bool in = t >= 0 && t < n && allowed_at(static_cast<int>(t));
      const bool several = in && ((twice[t >> 5] >> (t & 31)) & 1u) != 0;
      if (in && !several) z[t] = __fadd_rn(z[t], i == tid ? first_value : values[i]);
      // a token of several entries: the warp looks for them, and the thread of
      // the first adds their values one by one
      for (uint32_t left = __ballot_sync(0xffffffffu, several); left != 0; left &= left - 1) {
        const int who = __ffs(left) - 1;
        const int32_t wanted = __shfl_sync(0xffffffffu, id, who);
        float sum = z[wanted - v0];
        bool mine = true;
        for (int j0 = 0; j0 < biases && mine; j0 += 32) {
          const int j = j0 + lane;
          const bool same = j < biases && ids[j] == wanted;
          const float v = same ? values[j] : 0.f;
          for (uint32_t hits = __ballot_sync(0xffffffffu, same); hits != 0 && mine;
               hits &= hits - 1) {
            const int at = __ffs(hits) - 1;
            mine = j0 + at >= base + who;  // an earlier entry: its thread does it
            sum = __fadd_rn(sum, __shfl_sync(0xffffffffu, v, at));
          }
        }
        __syncwarp();
        if (mine && lane == who) z[wanted - v0] = sum;
      }
    }
  }
  if (VECTOR) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (tid == 0 && groups > 0) {
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(y + lead),
                   "r"(tc::smem_u32(z + lead)), "r"(16 * groups)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    if (tid < 4) {
      const int rest = lead + 4 * groups + tid;
      if (tid < lead) y[tid] = z[tid];
      if (rest < n) y[rest] = z[rest];
    }
    // shared memory lasts until the copy has read it
    if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  } else {
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) y[i] = z[i];
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
  // Slices small enough for three CTAs an SM, so that their phases overlap; at
  // least one access a thread, at most what shared memory holds three times.
  const int dev = current_device();
  const int64_t share = ceil_div(rows * vocab, 3ll * sm_count(dev));
  p.slice = static_cast<int>(std::min<int64_t>(
      kMaxSlice, std::max<int64_t>(kMinSlice, ceil_div(share, kMinSlice) * kMinSlice)));
  p.r = r;
  p.status = device_status_ptr(dev);
  const dim3 grid(static_cast<unsigned>(ceil_div(vocab, p.slice)), static_cast<unsigned>(rows));
  const size_t smem = 4 * static_cast<size_t>(smem_words(p.slice));
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev & 63], [&]() {
    const int most = 4 * static_cast<int>(smem_words(kMaxSlice));
    attr_err[dev & 63] = cudaFuncSetAttribute(adjust_logits_kernel<true>,
                                              cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (attr_err[dev & 63] == cudaSuccess) {
      attr_err[dev & 63] = cudaFuncSetAttribute(adjust_logits_kernel<false>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    }
  });
  TVR_CUDA_TRY(attr_err[dev & 63]);
  // rows of any vocabulary may start anywhere, as long as both sides do so alike
  const auto place = [](const float* base, int64_t stride) {
    return ((reinterpret_cast<uintptr_t>(base) >> 2) & 3) << 2 | (stride & 3);
  };
  if (place(logits, logits_stride) == place(out, out_stride)) {
    adjust_logits_kernel<true><<<grid, kThreads, smem, as_stream(stream)>>>(p);
  } else {
    adjust_logits_kernel<false><<<grid, kThreads, smem, as_stream(stream)>>>(p);
  }
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
