// The page plan of one serving step (tvr_page_plan) and the append of new
// keys and values to their pages (tvr_paged_append).
#include "paged_common.cuh"

#include "cluster.cuh"

#include <algorithm>
#include <climits>
#include <cstring>
#include <mutex>

namespace tvr {
namespace paged {
namespace {

// ---- page plan --------------------------------------------------------------
//
// With s_r positions held, n_r new ones, P positions a page:
//   held_r = ceil(s_r / P),  need_r = ceil((s_r + n_r) / P) - held_r,
//   released before r:  R_r = sum of held_q over the ended requests q < r,
//   taken before r:     N_r = sum of need_q over the requests q < r,
//   tokens before r:    T_r = sum of n_q over the requests q < r (n_q > 0).
// The stack after the releases has top = free + R_total entries; entry e is
// free_pages[e] for e < free, else the released page with number e - free.
// Allocation j takes entry top - 1 - j, so every page and every token's slot
// follows from the three prefix sums alone.
//
// One launch: every CTA computes the prefix sums of all requests in its shared
// memory (20 bytes a request), the grid's threads share out the new table
// entries, the pages pushed and the tokens; a search in a prefix sum finds the
// request.  Nothing that a thread reads from memory is written in the same call
// except, in place, the lengths and the count: then the grid is one cluster,
// and they are written after a cluster barrier that follows the sums.
// Bound by latencies: two rounds of loads, the sums and one search per output
// (1000 requests, 41 thousand tokens: 16 us on a cluster of 8 CTAs of 1024
// threads, 9 us on 148 of 256).  With few tokens one CTA also moves the pages of
// requests that end, 256 at a time (64 requests of 500 pages each: 67 us).
constexpr int kMaxRequests = 8192;
constexpr int kClusterCtas = 8;

struct PlanParams {
  int32_t* table;
  int64_t table_stride;
  int max_pages;
  int most;  // positions of a request
  int requests;
  int32_t* free_pages;
  int num_pages;
  FastDiv page;
  const int32_t* seq;
  const int32_t* grow;
  int32_t* seq_out;
  const int32_t* count;
  int32_t* count_out;
  int64_t* slots;
  int32_t* positions;
  int32_t* rows;
  int64_t tokens;
  int64_t per_request;
  int* status;
};

// The first index i in [0, n) with ends[i] > x (n if there is none).
template <typename T>
__device__ __forceinline__ int first_above(const T* ends, int n, T x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

struct Sums {
  int released, need;
  long long tokens;
};

__device__ __forceinline__ Sums add(const Sums& a, const Sums& b) {
  return {a.released + b.released, a.need + b.need, a.tokens + b.tokens};
}

__device__ __forceinline__ Sums shfl_up(const Sums& a, int d) {
  return {__shfl_up_sync(0xffffffffu, a.released, d), __shfl_up_sync(0xffffffffu, a.need, d),
          __shfl_up_sync(0xffffffffu, a.tokens, d)};
}

// THREADS a CTA.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) page_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ __align__(16) unsigned char plan_smem[];
  const int n = p.requests;
  long long* s_tokens = reinterpret_cast<long long*>(plan_smem);  // inclusive sums
  int* s_released = reinterpret_cast<int*>(s_tokens + n);
  int* s_need = s_released + n;
  int* s_seq = s_need + n;  // the length held; ~length for an ended request
  constexpr int WARPS = THREADS / 32;
  __shared__ Sums s_warp[WARPS];
  __shared__ int s_refused;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int free_count = max(0, min(p.num_pages, *p.count));
  auto pages_of = [&](long long positions) -> int {
    // positions < 2^31 + 2^31: a request that long is past any table
    if (positions > INT_MAX) return INT_MAX;
    return static_cast<int>(fast_div(static_cast<uint32_t>(positions) + p.page.d - 1, p.page));
  };

  // the prefix sums: each thread takes consecutive requests, adds them up, and
  // goes over them again with what lies before them
  const int per_thread = (n + THREADS - 1) / THREADS;
  const int r_begin = min(n, tid * per_thread), r_end = min(n, r_begin + per_thread);
  auto request = [&](int r, int& held_seq) -> Sums {
    Sums own = {0, 0, 0};
    const int seq = max(0, p.seq[r]), grow = p.grow[r];
    const int held = pages_of(seq);
    if (grow < 0) {
      own.released = min(held, p.max_pages);
      held_seq = ~seq;
    } else {
      const int want = pages_of(static_cast<long long>(seq) + grow);
      const bool room = p.per_request == 0 || grow <= p.per_request;
      own.need = room && static_cast<long long>(seq) + grow <= p.most ? want - held : 0;
      own.tokens = grow;
      held_seq = seq;
    }
    return own;
  };
  if (tid == 0) s_refused = 0;
  Sums mine = {0, 0, 0};
  for (int r = r_begin; r < r_end; ++r) {
    int held_seq;
    mine = add(mine, request(r, held_seq));
  }
  Sums sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Sums below = shfl_up(sum, d);
    if (lane >= d) sum = add(sum, below);
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  if (warp == 0 && lane < WARPS) {
    constexpr unsigned LANES = WARPS == 32 ? 0xffffffffu : (1u << (WARPS & 31)) - 1u;
    Sums w = s_warp[lane];
#pragma unroll
    for (int d = 1; d < WARPS; d <<= 1) {
      const Sums below = {__shfl_up_sync(LANES, w.released, d), __shfl_up_sync(LANES, w.need, d),
                          __shfl_up_sync(LANES, w.tokens, d)};
      if (lane >= d) w = add(w, below);
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const Sums before = s_warp[WARPS - 1];  // of all requests
  if (warp > 0) sum = add(sum, s_warp[warp - 1]);
  sum = {sum.released - mine.released, sum.need - mine.need, sum.tokens - mine.tokens};
  for (int r = r_begin; r < r_end; ++r) {
    int held_seq;
    sum = add(sum, request(r, held_seq));
    s_released[r] = sum.released;
    s_need[r] = sum.need;
    s_tokens[r] = sum.tokens;
    s_seq[r] = held_seq;
  }
  __syncthreads();
  const int top = free_count + before.released;
  // Admitted: a request that fits its positions and the token arrays, and
  // needs no page or ends within the stack.  The sums count every request that
  // fits its positions, so the first one past the stack refuses all that need a page
  // after it, and the first one past packed token arrays all that bring tokens.
  auto admitted = [&](int r) -> bool {
    const int seq = s_seq[r];
    if (seq < 0) return false;
    const long long first = r > 0 ? s_tokens[r - 1] : 0, grow = s_tokens[r] - first;
    if (seq + grow > p.most) return false;
    if (p.per_request > 0 ? grow > p.per_request : grow > 0 && s_tokens[r] > p.tokens) return false;
    const int need = s_need[r] - (r > 0 ? s_need[r - 1] : 0);
    return need == 0 || s_need[r] <= top;
  };
  // entry e of the stack after the releases
  auto entry = [&](int e) -> int {
    if (e < free_count) return p.free_pages[e];
    const int k = e - free_count;
    const int q = first_above(s_released, n, k);
    const int at = k - (q > 0 ? s_released[q - 1] : 0);
    return p.table[q * p.table_stride + at];
  };
  // pages taken: the needs are taken in order until one does not fit
  int cut = before.need <= top ? n : first_above(s_need, n, top);
  if (p.per_request == 0 && before.tokens > p.tokens) {
    cut = min(cut, first_above(s_tokens, n, static_cast<long long>(p.tokens)));
  }
  const int taken = cut > 0 ? s_need[cut - 1] : 0;

  const int64_t step = static_cast<int64_t>(gridDim.x) * THREADS;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * THREADS + tid;
  for (int64_t j = first; j < taken; j += step) {
    const int r = first_above(s_need, n, static_cast<int>(j));
    const int at = pages_of(s_seq[r]) + static_cast<int>(j) - (r > 0 ? s_need[r - 1] : 0);
    p.table[r * p.table_stride + at] = entry(top - 1 - static_cast<int>(j));
  }
  const int left = top - taken;  // entries of the stack after the step
  for (int64_t e = free_count + first; e < left; e += step) {
    if (e < p.num_pages) p.free_pages[e] = entry(static_cast<int>(e));
  }
  for (int64_t t = first; t < p.tokens; t += step) {
    int r;
    long long i;
    bool live;
    if (p.per_request > 0) {
      r = static_cast<int>(t / p.per_request);
      i = t - r * p.per_request;
      live = r < n && i < s_tokens[r] - (r > 0 ? s_tokens[r - 1] : 0);
    } else {
      r = first_above(s_tokens, n, static_cast<long long>(t));
      live = r < n;
      i = live ? t - (r > 0 ? s_tokens[r - 1] : 0) : 0;
    }
    int64_t slot = -1;
    int position = 0;
    if (live) {
      const int seq = s_seq[r];
      position = static_cast<int>(min(seq + i, static_cast<long long>(INT_MAX)));
      if (admitted(r)) {
        const int at = static_cast<int>(fast_div(static_cast<uint32_t>(position), p.page));
        const int held = pages_of(seq);
        const int id = at < held ? p.table[r * p.table_stride + at]
                                 : entry(top - 1 - (r > 0 ? s_need[r - 1] : 0) - (at - held));
        slot = static_cast<int64_t>(id) * p.page.d + (position - at * static_cast<int>(p.page.d));
      }
    }
    p.slots[t] = slot;
    if (p.positions != nullptr) p.positions[t] = position;
    if (p.rows != nullptr) p.rows[t] = live ? r : -1;
  }

  cluster_sync();  // in place: every CTA has read the lengths and the count
  if (blockIdx.x == 0) {
    for (int r = tid; r < n; r += THREADS) {
      const int seq = s_seq[r];
      const int grow = static_cast<int>(s_tokens[r] - (r > 0 ? s_tokens[r - 1] : 0));
      const bool in = admitted(r);
      if (seq >= 0 && !in) s_refused = 1;
      p.seq_out[r] = seq < 0 ? 0 : in ? seq + grow : seq;
    }
    if (tid == 0) *p.count_out = min(left, p.num_pages);
    __syncthreads();
    if (tid == 0 && s_refused != 0) report(p.status, TVR_DEV_CACHE_FULL);
  }
}

template <int THREADS>
int launch_plan(const PlanParams& p, unsigned ctas, unsigned cluster, cudaStream_t stream) {
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  const int dev = current_device();
  std::call_once(once[dev & 63], [&]() {
    attr_err[dev & 63] =
        cudaFuncSetAttribute(page_plan_kernel<THREADS>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRequests * 20);
  });
  TVR_CUDA_TRY(attr_err[dev & 63]);
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.requests) * 20;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  TVR_CUDA_TRY(cudaLaunchKernelEx(&cfg, page_plan_kernel<THREADS>, p));
  return TVR_OK;
}

// ---- append -------------------------------------------------------------------
//
// A copy with conversion: reads 4 bytes and writes 4 or 2 per value, bound by
// memory.  A thread moves VEC values, 16 bytes of a page row where the
// operands allow it (one value where they do not), kBatch of them under way;
// the threads of a token lie side by side (16385 tokens of 8 heads of 128 into
// bf16 pages: 33 us, 6.1 TB/s; one value a thread 201 us).
constexpr int kBatch = 2;

struct AppendParams {
  void* pages[2];
  const float* src[2];
  int64_t page_stride[2][3];  // page, head, position
  int64_t src_stride[2][2];   // token, head
  const int64_t* slots;
  int64_t n_slots;  // num_pages * page_size
  FastDiv page_size;
  int64_t items;
  FastDiv per_token, per_side, per_head;  // vectors of a token (K and V), of one side, of a head
  int* status;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendParams p) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
       first < p.items; first += kBatch * step) {
    float x[kBatch][VEC];
    T* dst[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t item = first + b * step;
      dst[b] = nullptr;
      if (item >= p.items) continue;
      const int64_t token = item <= UINT_MAX
                                ? fast_div(static_cast<uint32_t>(item), p.per_token)
                                : item / p.per_token.d;
      const uint32_t in_token = static_cast<uint32_t>(item - token * p.per_token.d);
      const uint32_t side = fast_div(in_token, p.per_side);
      const uint32_t in_side = in_token - side * p.per_side.d;
      const uint32_t head = fast_div(in_side, p.per_head);
      const uint32_t d = (in_side - head * p.per_head.d) * VEC;
      const float* src =
          p.src[side] + token * p.src_stride[side][0] + head * p.src_stride[side][1] + d;
      if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          const float4 v = __ldg(reinterpret_cast<const float4*>(src + i));
          x[b][i] = v.x;
          x[b][i + 1] = v.y;
          x[b][i + 2] = v.z;
          x[b][i + 3] = v.w;
        }
      } else {
        x[b][0] = __ldg(src);
      }
      const int64_t slot = __ldg(p.slots + token);
      if (slot < 0) continue;
      if (slot >= p.n_slots) {
        if (in_token == 0) report(p.status, TVR_DEV_BAD_INDEX);
        continue;
      }
      const int64_t page = slot <= UINT_MAX ? fast_div(static_cast<uint32_t>(slot), p.page_size)
                                            : slot / p.page_size.d;
      const int64_t at = slot - page * p.page_size.d;
      dst[b] = static_cast<T*>(p.pages[side]) + page * p.page_stride[side][0] +
               head * p.page_stride[side][1] + at * p.page_stride[side][2] + d;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (dst[b] == nullptr) continue;
      T t[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) from_f32(t[i], x[b][i]);
      if constexpr (VEC == 1) {
        *dst[b] = t[0];
      } else {
        uint4 v;
        memcpy(&v, t, 16);
        *reinterpret_cast<uint4*>(dst[b]) = v;
      }
    }
  }
}

template <typename T, int VEC>
int append(AppendParams& p, int64_t tokens, int64_t heads, int64_t dim, cudaStream_t stream) {
  const int64_t per_head = dim / VEC;
  p.per_head = make_fastdiv(static_cast<uint32_t>(per_head));
  p.per_side = make_fastdiv(static_cast<uint32_t>(per_head * heads));
  p.per_token = make_fastdiv(static_cast<uint32_t>(2 * per_head * heads));
  p.items = tokens * 2 * per_head * heads;
  paged_append_kernel<T, VEC>
      <<<elementwise_grid(ceil_div(p.items, kBatch), 256, current_device()), 256, 0, stream>>>(p);
  TVR_LAUNCH_CHECK();
  return TVR_OK;
}

template <typename T>
int append(AppendParams& p, int64_t tokens, int64_t heads, int64_t dim, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  bool whole = dim % VEC == 0;
  for (int side = 0; side < 2; ++side) {
    whole = whole && reinterpret_cast<uintptr_t>(p.pages[side]) % 16 == 0 &&
            reinterpret_cast<uintptr_t>(p.src[side]) % 16 == 0;
    for (int64_t st : p.page_stride[side]) whole = whole && st % VEC == 0;
    for (int64_t st : p.src_stride[side]) whole = whole && st % 4 == 0;
  }
  return whole ? append<T, VEC>(p, tokens, heads, dim, stream)
               : append<T, 1>(p, tokens, heads, dim, stream);
}

}  // namespace
}  // namespace paged
}  // namespace tvr

using namespace tvr;

extern "C" int tvr_page_plan(const tvr_page_pool* pool, const int32_t* seq_lens,
                             const int32_t* new_lens, int32_t* seq_lens_out,
                             const int32_t* free_count, int32_t* free_count_out, int64_t* slots,
                             int32_t* positions, int32_t* rows, int64_t tokens,
                             int64_t tokens_per_request, void* stream) {
  using namespace paged;
  TVR_CHECK(pool != nullptr, "page_plan: null pool");
  TVR_CHECK(pool->requests >= 0 && pool->max_pages >= 0 && pool->num_pages >= 0 && tokens >= 0 &&
                tokens_per_request >= 0 && pool->max_positions >= 0,
            "page_plan: negative size");
  TVR_CHECK(pool->page_size >= 1 && pool->page_size <= (1 << 20),
            "page_plan: page size %lld is not in 1..2^20", (long long)pool->page_size);
  TVR_CHECK(pool->max_pages <= 0x7fffffff / pool->page_size && pool->num_pages < 0x7fffffff &&
                tokens <= 0x7fffffff,
            "page_plan: too many pages or tokens");
  TVR_CHECK(pool->requests == 0 ||
                pool->max_pages <= (0x7fffffff - pool->num_pages) / pool->requests,
            "page_plan: too many pages in the tables");
  TVR_CHECK(pool->table_stride >= pool->max_pages || pool->requests <= 1,
            "page_plan: the table's row stride is less than max_pages");
  if (pool->requests > kMaxRequests) {
    return fail(TVR_ERR_UNSUPPORTED, "page_plan: %lld requests, at most %d",
                (long long)pool->requests, kMaxRequests);
  }
  TVR_CHECK(free_count && free_count_out, "page_plan: null free count");
  TVR_CHECK(pool->requests == 0 || (seq_lens && new_lens && seq_lens_out), "page_plan: null lengths");
  TVR_CHECK(pool->requests == 0 || pool->max_pages == 0 || pool->block_table,
            "page_plan: null block table");
  TVR_CHECK(pool->num_pages == 0 || pool->free_pages, "page_plan: null free pages");
  TVR_CHECK(tokens == 0 || slots, "page_plan: null slots");
  const int dev = current_device();
  PlanParams p = {};
  p.table = pool->block_table;
  p.table_stride = pool->table_stride;
  p.max_pages = static_cast<int>(pool->max_pages);
  p.most = static_cast<int>(pool->max_pages * pool->page_size);
  if (pool->max_positions > 0) p.most = static_cast<int>(std::min<int64_t>(p.most, pool->max_positions));
  p.requests = static_cast<int>(pool->requests);
  p.free_pages = pool->free_pages;
  p.num_pages = static_cast<int>(pool->num_pages);
  p.page = make_fastdiv(static_cast<uint32_t>(pool->page_size));
  p.seq = seq_lens;
  p.grow = new_lens;
  p.seq_out = seq_lens_out;
  p.count = free_count;
  p.count_out = free_count_out;
  p.slots = slots;
  p.positions = positions;
  p.rows = rows;
  p.tokens = tokens;
  p.per_request = tokens_per_request;
  p.status = device_status_ptr(dev);
  // In place: one CTA, or one cluster where there are more tokens than a few a
  // thread.  Otherwise a CTA for each 256 tokens, up to one an SM.
  const bool in_place = seq_lens_out == seq_lens || free_count_out == free_count;
  if (tokens <= 4 * 256) return launch_plan<256>(p, 1, 1, as_stream(stream));
  if (in_place) return launch_plan<1024>(p, kClusterCtas, kClusterCtas, as_stream(stream));
  const int64_t ctas = std::min<int64_t>(sm_count(dev), ceil_div(tokens, 256));
  return launch_plan<256>(p, static_cast<unsigned>(ctas), 1, as_stream(stream));
}

extern "C" int tvr_paged_append(const tvr_paged_kv* cache, const float* k_new, const float* v_new,
                                const int64_t* strides, const int64_t* slots, int64_t tokens,
                                void* stream) {
  using namespace paged;
  if (int rc = check_cache(cache, "paged_append")) return rc;
  TVR_CHECK(tokens >= 0, "paged_append: negative size");
  const int64_t heads = cache->kv_heads, dim = cache->head_dim;
  if (tokens == 0 || heads == 0 || dim == 0) return TVR_OK;
  TVR_CHECK(k_new && v_new && strides && slots, "paged_append: null pointer");
  TVR_CHECK(cache->num_pages == 0 || (cache->k_pages && cache->v_pages), "paged_append: null pages");
  TVR_CHECK(heads * dim <= 0x3fffffff, "paged_append: too many values a token");
  AppendParams p = {};
  p.pages[0] = cache->k_pages;
  p.pages[1] = cache->v_pages;
  p.src[0] = k_new;
  p.src[1] = v_new;
  for (int i = 0; i < 3; ++i) {
    p.page_stride[0][i] = cache->k_strides[i];
    p.page_stride[1][i] = cache->v_strides[i];
  }
  for (int i = 0; i < 2; ++i) {
    p.src_stride[0][i] = strides[i];
    p.src_stride[1][i] = strides[2 + i];
  }
  p.slots = slots;
  p.n_slots = cache->num_pages * cache->page_size;
  p.page_size = make_fastdiv(static_cast<uint32_t>(cache->page_size));
  p.status = device_status_ptr(current_device());
  switch (cache->page_type) {
    case TVR_PAGE_F32: return append<float>(p, tokens, heads, dim, as_stream(stream));
    case TVR_PAGE_F16: return append<__half>(p, tokens, heads, dim, as_stream(stream));
    default: return append<__nv_bfloat16>(p, tokens, heads, dim, as_stream(stream));
  }
}
