// Attention of one new token per request over its pages, with the append of
// that token's key and value in the same launch (tvr_paged_attention):
//   out[r, h] = softmax_j(scale q[r, h] . k[r, g, j]) v[r, g, j],  j < n_r,
// with g = h / (heads / kv_heads) and n_r = seq_lens[r] read on the device.
#include "paged_common.cuh"

#include <cfloat>
#include <cmath>

namespace tvr {
namespace paged {
namespace {

struct AttendParams {
  const float* q;
  const float* k_new;  // with v_new and slots, or all null
  const float* v_new;
  const int64_t* slots;
  void* k;
  void* v;
  const int32_t* table;
  const int32_t* lens;
  float* out;
  float* lse;
  int64_t table_stride;
  int64_t q_s[2], kn_s[2], vn_s[2], o_s[2];  // request, head
  int64_t k_s[3], v_s[3];                    // page, head, position
  int64_t n_slots;
  int max_keys;  // max_pages * page_size
  int num_pages;
  int heads, group, dim;
  FastDiv page;
  float scale_log2;
  int* status;
};

// ---- the general form ---------------------------------------------------------
//
// Any head dimension to 256, any strides and alignment: a CTA per query head,
// a warp per key, lane l holding dimensions l, l + 32, ...  The keys are dealt
// to the warps in turn; each warp keeps a running maximum and sum (exp2
// domain) and the CTA joins the warps at the end.  The maximum starts at
// -FLT_MAX, not -inf, so that a score of -inf gives a weight of 0 without a
// special case and a row of nothing but -inf gives 0 / 0, as the formula does.
constexpr int kGeneralWarps = 4;
constexpr int kMaxDim = 256;

template <typename T>
__global__ void __launch_bounds__(32 * kGeneralWarps)
    paged_attention_general_kernel(const __grid_constant__ AttendParams p) {
  constexpr int DL = kMaxDim / 32;
  __shared__ float s_m[kGeneralWarps], s_l[kGeneralWarps];
  __shared__ float s_o[kGeneralWarps][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = blockIdx.x / p.heads;
  const int h = static_cast<int>(blockIdx.x - r * p.heads), g = h / p.group;
  const int n = max(0, min(p.max_keys, p.lens[r]));
  const int64_t slot = p.slots != nullptr && n > 0 ? p.slots[r] : -1;
  const bool fresh = slot >= 0 && slot < p.n_slots;
  if (slot >= p.n_slots && threadIdx.x == 0) report(p.status, TVR_DEV_BAD_INDEX);

  float q[DL], o[DL];
#pragma unroll
  for (int i = 0; i < DL; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < p.dim ? p.q[r * p.q_s[0] + h * p.q_s[1] + d] : 0.f;
    o[i] = 0.f;
  }
  float m = -FLT_MAX, l = 0.f;
  for (int j = warp; j < n; j += kGeneralWarps) {
    float k[DL], v[DL];
    if (fresh && j == n - 1) {
      const float* kn = p.k_new + r * p.kn_s[0] + g * p.kn_s[1];
      const float* vn = p.v_new + r * p.vn_s[0] + g * p.vn_s[1];
      const int64_t page = slot / p.page.d, at = slot - page * p.page.d;
      T* kc = static_cast<T*>(p.k) + page * p.k_s[0] + g * p.k_s[1] + at * p.k_s[2];
      T* vc = static_cast<T*>(p.v) + page * p.v_s[0] + g * p.v_s[1] + at * p.v_s[2];
#pragma unroll
      for (int i = 0; i < DL; ++i) {
        const int d = lane + 32 * i;
        k[i] = v[i] = 0.f;
        if (d < p.dim) {
          T kt, vt;
          from_f32(kt, kn[d]);
          from_f32(vt, vn[d]);
          k[i] = to_f32(kt);
          v[i] = to_f32(vt);
          if (h == g * p.group) {
            kc[d] = kt;
            vc[d] = vt;
          }
        }
      }
    } else {
      const uint32_t at = fast_div(static_cast<uint32_t>(j), p.page);
      const int page = p.table[r * p.table_stride + at];
      if (page < 0 || page >= p.num_pages) {
        if (lane == 0) report(p.status, TVR_DEV_BAD_INDEX);
        continue;
      }
      const int in_page = j - static_cast<int>(at * p.page.d);
      const T* kc = static_cast<const T*>(p.k) + page * p.k_s[0] + g * p.k_s[1] + in_page * p.k_s[2];
      const T* vc = static_cast<const T*>(p.v) + page * p.v_s[0] + g * p.v_s[1] + in_page * p.v_s[2];
#pragma unroll
      for (int i = 0; i < DL; ++i) {
        const int d = lane + 32 * i;
        k[i] = d < p.dim ? to_f32(kc[d]) : 0.f;
        v[i] = d < p.dim ? to_f32(vc[d]) : 0.f;
      }
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < DL; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale_log2;
    const float top = fmaxf(m, s), keep = exp2f(m - top), w = exp2f(s - top);
    m = top;
    l = fmaf(l, keep, w);
#pragma unroll
    for (int i = 0; i < DL; ++i) o[i] = fmaf(w, v[i], o[i] * keep);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < DL; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -FLT_MAX, sum = 0.f;
  for (int w = 0; w < kGeneralWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kGeneralWarps; ++w) sum += s_l[w] * exp2f(s_m[w] - top);
  for (int d = threadIdx.x; d < p.dim; d += 32 * kGeneralWarps) {
    float acc = 0.f;
    for (int w = 0; w < kGeneralWarps; ++w) acc += s_o[w][d] * exp2f(s_m[w] - top);
    p.out[r * p.o_s[0] + h * p.o_s[1] + d] = n > 0 ? acc / sum : 0.f;
  }
  if (threadIdx.x == 0 && p.lse != nullptr) {
    p.lse[r * p.heads + h] = n > 0 ? top * 0.69314718055994531f + logf(sum) : -INFINITY;
  }
}

}  // namespace
}  // namespace paged
}  // namespace tvr

using namespace tvr;

extern "C" int tvr_paged_attention_workspace(int64_t heads, int64_t kv_heads, int64_t head_dim,
                                             int64_t* bytes) {
  TVR_CHECK(bytes != nullptr, "paged_attention_workspace: null pointer");
  TVR_CHECK(heads >= 0 && kv_heads >= 0 && head_dim >= 0 && heads <= 65535 && head_dim <= 65535,
            "paged_attention_workspace: bad size");
  *bytes = 0;
  return TVR_OK;
}

extern "C" int tvr_paged_attention(const tvr_paged_kv* cache, const float* q, const float* k_new,
                                   const float* v_new, const int64_t* slots,
                                   const int32_t* block_table, int64_t table_stride,
                                   int64_t max_pages, const int32_t* seq_lens, float* out,
                                   float* lse, int64_t requests, int64_t heads,
                                   const int64_t* strides, float scale, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  using namespace paged;
  (void)workspace;
  (void)workspace_bytes;
  if (int rc = check_cache(cache, "paged_attention")) return rc;
  TVR_CHECK(requests >= 0 && heads >= 0 && max_pages >= 0, "paged_attention: negative size");
  const int64_t dim = cache->head_dim;
  if (requests == 0 || heads == 0 || dim == 0) return TVR_OK;
  TVR_CHECK(cache->kv_heads >= 1 && heads % cache->kv_heads == 0,
            "paged_attention: %lld heads do not share %lld key heads evenly", (long long)heads,
            (long long)cache->kv_heads);
  TVR_CHECK(q && out && strides && seq_lens, "paged_attention: null pointer");
  TVR_CHECK(max_pages == 0 || (block_table && cache->k_pages && cache->v_pages),
            "paged_attention: null pages or block table");
  TVR_CHECK((k_new != nullptr) == (slots != nullptr) && (v_new != nullptr) == (slots != nullptr),
            "paged_attention: k_new, v_new and slots come together");
  TVR_CHECK(table_stride >= max_pages || requests == 1,
            "paged_attention: the table's row stride is less than max_pages");
  TVR_CHECK(max_pages <= 0x7fffffff / cache->page_size && requests * heads <= 0x7fffffff &&
                heads <= 65535,
            "paged_attention: too many positions or heads");
  TVR_CHECK(std::isfinite(scale), "paged_attention: the scale is not finite");
  if (dim > kMaxDim) {
    return fail(TVR_ERR_UNSUPPORTED, "paged_attention: head dimension %lld, at most %d",
                (long long)dim, kMaxDim);
  }
  AttendParams p = {};
  p.q = q;
  p.k_new = k_new;
  p.v_new = v_new;
  p.slots = slots;
  p.k = cache->k_pages;
  p.v = cache->v_pages;
  p.table = block_table;
  p.lens = seq_lens;
  p.out = out;
  p.lse = lse;
  p.table_stride = table_stride;
  for (int i = 0; i < 2; ++i) {
    p.q_s[i] = strides[i];
    p.kn_s[i] = strides[2 + i];
    p.vn_s[i] = strides[4 + i];
    p.o_s[i] = strides[6 + i];
  }
  for (int i = 0; i < 3; ++i) {
    p.k_s[i] = cache->k_strides[i];
    p.v_s[i] = cache->v_strides[i];
  }
  p.n_slots = cache->num_pages * cache->page_size;
  p.max_keys = static_cast<int>(max_pages * cache->page_size);
  p.num_pages = static_cast<int>(cache->num_pages);
  p.heads = static_cast<int>(heads);
  p.group = static_cast<int>(heads / cache->kv_heads);
  p.dim = static_cast<int>(dim);
  p.page = make_fastdiv(static_cast<uint32_t>(cache->page_size));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = device_status_ptr(current_device());
  const unsigned grid = static_cast<unsigned>(requests * heads);
  const cudaStream_t s = as_stream(stream);
  switch (cache->page_type) {
    case TVR_PAGE_F32:
      paged_attention_general_kernel<float><<<grid, 32 * kGeneralWarps, 0, s>>>(p);
      break;
    case TVR_PAGE_F16:
      paged_attention_general_kernel<__half><<<grid, 32 * kGeneralWarps, 0, s>>>(p);
      break;
    default:
      paged_attention_general_kernel<__nv_bfloat16><<<grid, 32 * kGeneralWarps, 0, s>>>(p);
  }
  TVR_LAUNCH_CHECK();
  return TVR_OK;
}
