// Logits of a decode step adjusted before the next token is chosen
// (tvr_adjust_logits): penalties for tokens of the history, sparse biases,
// grammar masks; the histories' growth by the chosen tokens
// (tvr_history_append), and their taking the place of the current ones
// (tvr_advance_tokens).
#include "tc_ptx.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

namespace tvr {
namespace {

// One pass over the logits: 4 bytes read and 4 written per logit, plus the
// row's history (4 or 8 bytes a token, read by every slice from L2) and its
// mask bits.  A CTA takes a slice of one row's vocabulary:
//   1. it counts the row's history tokens that fall into the slice, in shared
//      memory (whole numbers: the order of the atomics does not matter), and
//      marks the slice's biased tokens and those with several biases;
//   2. the slice passes through two buffers in shared memory, chunk by chunk:
//      a bulk copy brings the next one in and another takes the last one out
//      while a chunk's logits are penalised, masked and biased (several biases
//      of one token by the warp of the first, in list order).
// 400 rows of 129280 logits take 76 us without a history (5.4 TB/s) and 121 us
// with 15000 tokens, 150 biases and a mask each.  What bounds long histories is
// that each slice reads all of it: counters are 16 bits wide where no count can
// exceed 32767, which the array's width bounds, for slices four times as wide
// (32-bit counters, the same rows in an array of 131072: 168 us; with 1000
// tokens of history 106 and 128 us).  int64 tokens: 136 us.
// Sharing a history out over a cluster measured slower in every form tried:
// atomics on one another's counters 262 us, sorting it by slices with atomics
// that return places 590.
constexpr int kThreads = 512;
constexpr int kChunk = 4096;
constexpr int kMinSlice = 4 * kThreads;
constexpr int kMaxSliceWide = 8192;     // of 32-bit counters
constexpr int kMaxSliceNarrow = 32768;  // of 16-bit ones
constexpr int kNarrowHistory = 32767;
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

// Counters of a token: the top bit says that it is in the prompt, the others
// count it among the generated.
template <bool NARROW>
struct Counter {
  using Word = typename std::conditional<NARROW, uint16_t, uint32_t>::type;
  static constexpr uint32_t kPrompt = NARROW ? 0x8000u : 0x80000000u;
};

// Without branches: in a long history nearly every warp has a token of it.
template <bool NARROW>
__device__ __forceinline__ float adjust(float x, uint32_t c, bool allowed, const RowRules& r) {
  const float made = static_cast<float>(c & (Counter<NARROW>::kPrompt - 1));
  const float factor = x > 0.f ? r.inverse : r.rep;
  x = __fmul_rn(x, c != 0 ? factor : 1.f);
  x = __fsub_rn(x, made > 0.f ? __fmul_rn(r.freq, made) : 0.f);
  x = __fsub_rn(x, made > 0.f ? r.pres : 0.f);
  return allowed ? x : -INFINITY;
}

// f(token - v0) for the n tokens, as an unsigned number: what is outside a slice
// that begins at v0 is past its end.  Several loads of a thread are under way:
// one at a time is what would bound a long history (265 us, then 155 us, for
// 400 rows of 129280 logits and 15000 tokens).
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

// Adds `one` to, or sets in, the counter of token t of a slice of n, where
// t < n; a narrow counter is half of a word, which it cannot overflow.
// Predicated: a branch around the atomic of each token costs twice its work.
template <bool NARROW, bool MARK>
__device__ __forceinline__ void count(uint32_t counters, uint32_t t, uint32_t n) {
  const uint32_t one = MARK ? Counter<NARROW>::kPrompt : 1u;
  const uint32_t addr = counters + (NARROW ? 2 * (t & ~1u) : 4 * t);
  const uint32_t v = NARROW ? one << (16 * (t & 1)) : one;
  if constexpr (MARK) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.lt.u32 p, %1, %2;\n\t"
        "@p red.shared.or.b32 [%0], %3;\n\t}" ::"r"(addr),
        "r"(t), "r"(n), "r"(v)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.lt.u32 p, %1, %2;\n\t"
        "@p red.shared.add.u32 [%0], %3;\n\t}" ::"r"(addr),
        "r"(t), "r"(n), "r"(v)
        : "memory");
  }
}

// Words of shared memory: counters, two chunks, mask words and two bits a token.
inline int64_t smem_words(int64_t slice, bool narrow) {
  return (narrow ? slice / 2 : slice) + 4 + 2 * kChunk + (slice / 32 + 4) + 2 * (slice / 32);
}

// VECTOR: x and y lie alike on 16-byte boundaries.
template <bool VECTOR, bool NARROW>
__global__ void __launch_bounds__(kThreads)
    adjust_logits_kernel(const __grid_constant__ LogitParams p) {
  using Word = typename Counter<NARROW>::Word;
  extern __shared__ __align__(16) uint32_t s_words[];
  __shared__ uint64_t s_bar[2];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int v0 = blockIdx.x * p.slice, n = min(p.slice, p.vocab - v0);
  const float* x = p.x + row * p.x_stride + v0;
  float* y = p.y + row * p.y_stride + v0;
  const tvr_logit_rules& r = p.r;

  // Logits [lead, lead + 4 quads) go by fours, on 16-byte boundaries, and
  // through the chunks; the others (all of them, where x and y lie differently)
  // one by one.  Token i has counter i + shift, so that the counters of four
  // lie on a boundary as well.
  const int shift = VECTOR ? static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3) : 0;
  const int lead = VECTOR ? min(n, (4 - shift) & 3) : n;
  const int quads = VECTOR ? (n - lead) / 4 : 0, end = lead + 4 * quads;
  const int chunks = (4 * quads + kChunk - 1) / kChunk;
  const int counter_words = NARROW ? p.slice / 2 + 4 : p.slice + 4;
  Word* const counts = reinterpret_cast<Word*>(s_words) + shift;
  float* const z = reinterpret_cast<float*>(s_words + counter_words);
  uint32_t* const allowed = s_words + counter_words + 2 * kChunk;
  uint32_t* const biased = allowed + p.slice / 32 + 4;
  uint32_t* const twice = biased + p.slice / 32;
  auto floats_of = [&](int c) { return min(kChunk, 4 * quads - c * kChunk); };
  auto bring = [&](int c) {  // chunk c, by one thread
    const uint32_t bar = tc::smem_u32(&s_bar[c & 1]);
    tc::mbar_expect_tx(bar, 4 * floats_of(c));
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            tc::smem_u32(z + (c & 1) * kChunk)),
        "l"(x + lead + c * kChunk), "r"(4 * floats_of(c)), "r"(bar)
        : "memory");
  };
  if (tid == 0) {
    tc::mbar_init(tc::smem_u32(&s_bar[0]), 1);
    tc::mbar_init(tc::smem_u32(&s_bar[1]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (chunks > 0) bring(0);
  }

  RowRules rules;
  rules.rep = r.repetition != nullptr ? r.repetition[row] : 1.f;
  rules.inverse = __fdiv_rn(1.f, rules.rep);
  rules.pres = r.presence != nullptr ? r.presence[row] : 0.f;
  rules.freq = r.frequency != nullptr ? r.frequency[row] : 0.f;
  const int64_t held = r.tokens != nullptr ? r.total_lens[row] : 0;
  const int prompt = r.tokens != nullptr && r.prompt_lens != nullptr ? r.prompt_lens[row] : 0;
  const int64_t with_bias =
      r.bias_ids == nullptr ? 0 : r.bias_counts != nullptr ? r.bias_counts[row] : r.bias_stride;
  int64_t m = r.masks == nullptr ? -1 : r.mask_rows != nullptr ? r.mask_rows[row] : row;
  if (m >= r.n_masks) {
    if (tid == 0 && blockIdx.x == 0 && p.status != nullptr) {
      atomicCAS(p.status, TVR_DEV_OK, TVR_DEV_BAD_INDEX);
    }
    m = -1;
  }
  const int total = static_cast<int>(max(int64_t(0), min(held, r.tokens_stride)));
  const int biases = static_cast<int>(max(int64_t(0), min(with_bias, r.bias_stride)));
  const int32_t* ids = r.bias_ids + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  const int32_t first_id = tid < biases ? ids[tid] : -1;  // this thread's first bias
  const float first_value = tid < biases ? values[tid] : 0.f;

  // v0 is a multiple of 32
  const uint32_t* mask = m >= 0 ? r.masks + m * r.mask_stride + v0 / 32 : nullptr;
  for (int i = tid; i < (n + 31) / 32; i += kThreads) allowed[i] = mask != nullptr ? mask[i] : ~0u;
  for (int i = tid; i < counter_words / 4; i += kThreads) {
    reinterpret_cast<uint4*>(s_words)[i] = make_uint4(0, 0, 0, 0);
  }
  for (int i = tid; i < 2 * (p.slice / 32); i += kThreads) biased[i] = 0;  // and twice
  __syncthreads();
  if (total > 0) {
    // the prompt's part and what was generated; the marks and counts of a
    // token are in other bits, so their order does not matter
    const int64_t base = row * r.tokens_stride;
    const int made_from = max(0, min(prompt, total));
    const uint32_t counters = tc::smem_u32(s_words), at = static_cast<uint32_t>(shift);
    const uint32_t nu = static_cast<uint32_t>(n);
    // t + shift < n + shift, where t may be anything
    auto mark = [&](uint32_t t) { count<NARROW, true>(counters, t < nu ? t + at : kNone, nu + at); };
    auto tally = [&](uint32_t t) { count<NARROW, false>(counters, t < nu ? t + at : kNone, nu + at); };
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
    const uint32_t bit = 1u << (t & 31);
    if ((atomicOr(&biased[t >> 5], bit) & bit) != 0) atomicOr(&twice[t >> 5], bit);
  }
  __syncthreads();

  auto bit_of = [&](const uint32_t* bits, int i) { return ((bits[i >> 5] >> (i & 31)) & 1u) != 0; };
  // the logits outside the chunks; one of them with a bias looks for all of its
  // entries, in list order
  auto one = [&](int i) {
    const bool in = bit_of(allowed, i);
    float v = adjust<NARROW>(x[i], counts[i], in, rules);
    if (in && bit_of(biased, i)) {
      for (int j = 0; j < biases; ++j) {
        if (ids[j] == v0 + i) v = __fadd_rn(v, values[j]);
      }
    }
    y[i] = v;
  };
  for (int i = tid; i < lead; i += kThreads) one(i);
  if (end + tid < n) one(end + tid);

  for (int c = 0; c < chunks; ++c) {
    float* const zc = z + (c & 1) * kChunk;
    const int i0 = lead + c * kChunk, of_chunk = floats_of(c);
    if (tid == 0 && c + 1 < chunks) {
      // the other buffer's last chunk is on its way out
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      bring(c + 1);
    }
    if (!tc::mbar_wait(tc::smem_u32(&s_bar[c & 1]), (c >> 1) & 1, nullptr) && p.status != nullptr) {
      atomicCAS(p.status, TVR_DEV_OK, TVR_DEV_TIMEOUT_MMA);
    }
#pragma unroll 2
    for (int g = 4 * tid; g < of_chunk; g += 4 * kThreads) {
      const int i = i0 + g, at = i & 31;
      // the word after the last one is read, but not used
      const uint32_t bits =
          mask != nullptr ? __funnelshift_r(allowed[i >> 5], allowed[(i >> 5) + 1], at) & 15u : 15u;
      uint4 k;
      if constexpr (NARROW) {
        const uint2 two = *reinterpret_cast<const uint2*>(counts + i);
        k = make_uint4(two.x & 0xffffu, two.x >> 16, two.y & 0xffffu, two.y >> 16);
      } else {
        k = *reinterpret_cast<const uint4*>(counts + i);
      }
      if ((k.x | k.y | k.z | k.w) == 0 && bits == 15u) continue;
      float4 v = *reinterpret_cast<const float4*>(zc + g);
      v.x = adjust<NARROW>(v.x, k.x, (bits & 1u) != 0, rules);
      v.y = adjust<NARROW>(v.y, k.y, (bits & 2u) != 0, rules);
      v.z = adjust<NARROW>(v.z, k.z, (bits & 4u) != 0, rules);
      v.w = adjust<NARROW>(v.w, k.w, (bits & 8u) != 0, rules);
      *reinterpret_cast<float4*>(zc + g) = v;
    }
    if (biases > 0) {
      __syncthreads();
      for (int base = tid - lane; base < biases; base += kThreads) {
        const int i = base + lane;
        const int id = i >= biases ? -1 : i == tid ? first_id : ids[i];
        const int64_t t = static_cast<int64_t>(id) - v0;
        const bool in = t >= i0 && t < i0 + of_chunk && bit_of(allowed, static_cast<int>(t));
        const bool several = in && bit_of(twice, static_cast<int>(t));
        if (in && !several) {
          zc[t - i0] = __fadd_rn(zc[t - i0], i == tid ? first_value : values[i]);
        }
        // a token of several entries: the warp looks for them, and the thread
        // of the first adds their values one by one
        for (uint32_t left = __ballot_sync(0xffffffffu, several); left != 0; left &= left - 1) {
          const int who = __ffs(left) - 1;
          const int32_t wanted = __shfl_sync(0xffffffffu, id, who);
          float* const place = zc + (wanted - v0 - i0);
          float sum = *place;
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
          if (mine && lane == who) *place = sum;
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(y + i0),
                   "r"(tc::smem_u32(zc)), "r"(4 * of_chunk)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  // shared memory lasts until the copies have read it
  if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// A thread a row.  Rows count where live[row] > 0 or, with `slots`, where
// slots[row] >= 0; `current` (null: none) takes ids[row] as well.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    history_append_kernel(T* tokens, int64_t stride, int32_t* lens, const int64_t* ids,
                          const int32_t* live, const int64_t* slots, int64_t* current, int64_t rows,
                          int64_t capacity) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (row >= rows || (live != nullptr && live[row] <= 0)) return;
  if (slots != nullptr && slots[row] < 0) return;
  const int64_t id = ids[row];
  if (current != nullptr) current[row] = id;
  if (lens == nullptr) return;
  const int at = lens[row];
  if (at < 0 || at >= capacity) return;
  tokens[row * stride + at] = static_cast<T>(id);
  lens[row] = at + 1;
}

int append_history(const char* op, void* tokens, int token_bits, int64_t stride, int32_t* lens,
                   const int64_t* ids, const int32_t* live, const int64_t* slots,
                   int64_t* current, int64_t rows, int64_t capacity, void* stream) {
  TVR_CHECK(rows >= 0 && capacity >= 0, "%s: negative size", op);
  TVR_CHECK(token_bits == 32 || token_bits == 64, "%s: token_bits %d", op, token_bits);
  TVR_CHECK(capacity <= 0x7fffffff && rows <= 0x7fffffff, "%s: size past 32 bits", op);
  if (rows == 0) return TVR_OK;
  TVR_CHECK(ids && (lens || current) && (tokens || lens == nullptr || capacity == 0),
            "%s: null pointer", op);
  TVR_CHECK(lens == nullptr || rows == 1 || stride >= capacity,
            "%s: the row stride is less than the capacity", op);
  const unsigned grid = static_cast<unsigned>(ceil_div(rows, kThreads));
  if (token_bits == 64) {
    history_append_kernel<int64_t><<<grid, kThreads, 0, as_stream(stream)>>>(
        static_cast<int64_t*>(tokens), stride, lens, ids, live, slots, current, rows, capacity);
  } else {
    history_append_kernel<int32_t><<<grid, kThreads, 0, as_stream(stream)>>>(
        static_cast<int32_t*>(tokens), stride, lens, ids, live, slots, current, rows, capacity);
  }
  TVR_LAUNCH_CHECK();
  return TVR_OK;
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
  // least one access a thread, at most what leaves room for two CTAs; all of a
  // row's alike.
  const int dev = current_device();
  const int64_t share = ceil_div(rows * vocab, 3ll * sm_count(dev));
  const bool narrow = r.tokens == nullptr || r.tokens_stride <= kNarrowHistory;
  const int64_t most_slice = narrow ? kMaxSliceNarrow : kMaxSliceWide;
  const int64_t least = ceil_div(vocab, std::min(most_slice, std::max<int64_t>(kMinSlice, share)));
  p.slice = static_cast<int>(ceil_div(ceil_div(vocab, least), kMinSlice) * kMinSlice);
  p.r = r;
  p.status = device_status_ptr(dev);
  const dim3 grid(static_cast<unsigned>(ceil_div(vocab, p.slice)), static_cast<unsigned>(rows));
  const size_t smem = 4 * static_cast<size_t>(smem_words(p.slice, narrow));
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev & 63], [&]() {
    const int most = 4 * static_cast<int>(std::max(smem_words(kMaxSliceNarrow, true),
                                                   smem_words(kMaxSliceWide, false)));
    attr_err[dev & 63] = cudaSuccess;
    for (const void* kernel : {reinterpret_cast<const void*>(adjust_logits_kernel<true, true>),
                               reinterpret_cast<const void*>(adjust_logits_kernel<true, false>),
                               reinterpret_cast<const void*>(adjust_logits_kernel<false, true>),
                               reinterpret_cast<const void*>(adjust_logits_kernel<false, false>)}) {
      const cudaError_t e =
          cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e != cudaSuccess) attr_err[dev & 63] = e;
    }
  });
  TVR_CUDA_TRY(attr_err[dev & 63]);
  // rows of any vocabulary may start anywhere, as long as both sides do so alike
  const auto place = [](const float* base, int64_t stride) {
    return ((reinterpret_cast<uintptr_t>(base) >> 2) & 3) << 2 | (stride & 3);
  };
  const bool vector = place(logits, logits_stride) == place(out, out_stride);
  auto kernel = vector ? narrow ? adjust_logits_kernel<true, true> : adjust_logits_kernel<true, false>
                : narrow ? adjust_logits_kernel<false, true>
                         : adjust_logits_kernel<false, false>;
  kernel<<<grid, kThreads, smem, as_stream(stream)>>>(p);
  TVR_LAUNCH_CHECK();
  return TVR_OK;
}

extern "C" int tvr_history_append(void* tokens, int token_bits, int64_t tokens_stride,
                                  int32_t* lens, const int64_t* ids, const int32_t* live,
                                  int64_t rows, int64_t capacity, void* stream) {
  return append_history("history_append", tokens, token_bits, tokens_stride, lens, ids, live,
                        nullptr, nullptr, rows, capacity, stream);
}

extern "C" int tvr_advance_tokens(int64_t* current, const int64_t* next, const int64_t* slots,
                                  void* tokens, int token_bits, int64_t tokens_stride,
                                  int32_t* lens, int64_t rows, int64_t capacity, void* stream) {
  TVR_CHECK(rows <= 0 || (current && slots), "advance_tokens: null pointer");
  return append_history("advance_tokens", tokens, token_bits, tokens_stride, lens, next, nullptr,
                        slots, current, rows, capacity, stream);
}
