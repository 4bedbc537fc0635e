// Shared by the kernels of the paged KV cache (include/tvarant.h): the page
// element types, their conversions, and bounds-checked page addressing.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"

#include "fastdiv.cuh"

namespace tvr {
namespace paged {

// fp32 -> page element, rounded to nearest even; page element -> fp32, exact.
__device__ __forceinline__ void from_f32(float& d, float x) { d = x; }
__device__ __forceinline__ void from_f32(__half& d, float x) { d = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float x) { d = __float2bfloat16_rn(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, TVR_DEV_OK, code);
}

inline int64_t type_size(int page_type) { return page_type == TVR_PAGE_F32 ? 4 : 2; }

// Checks of a tvr_paged_kv that every entry point makes.
inline int check_cache(const tvr_paged_kv* c, const char* op) {
  TVR_CHECK(c != nullptr, "%s: null cache", op);
  TVR_CHECK(c->page_type >= TVR_PAGE_F32 && c->page_type <= TVR_PAGE_BF16,
            "%s: unknown page type %d", op, c->page_type);
  TVR_CHECK(c->num_pages >= 0 && c->kv_heads >= 0 && c->head_dim >= 0, "%s: negative size", op);
  TVR_CHECK(c->page_size >= 1 && c->page_size <= (1 << 20), "%s: page size %lld is not in 1..2^20",
            op, (long long)c->page_size);
  TVR_CHECK(c->num_pages <= 0x7fffffff && c->kv_heads <= 65535 && c->head_dim <= 65535,
            "%s: too many pages, heads or dimensions", op);
  return TVR_OK;
}

}  // namespace paged
}  // namespace tvr
