// Attention of one new token per request over its pages, with the append of
// that token's key and value in the same launch (tvr_paged_attention):
//   out[r, h] = softmax_j(scale q[r, h] . k[r, g, j]) v[r, g, j],  j < n_r,
// with g = h / (heads / kv_heads) and n_r = seq_lens[r] read on the device.
#include "paged_common.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstring>
#include <mutex>
#include <type_traits>

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
// special case and a row of nothing but -inf gives 0 / 0, as the formula does;
// a row without any position that counts (length 0, or all of its page ids out
// of range) is told apart from it and gives zeros.
// Bound by latency, a key at a time (128 requests of 200 to 8000 keys, 12 heads
// of 64, fp32 pages: 1708 us; the streaming form below 257 us), so it takes only
// what the other cannot: rows that are not whole 16-byte chunks.
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
  bool counted = false;  // whether any position of this warp counts
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
    counted = true;
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
  const bool some = __syncthreads_or(counted) != 0;
  float top = -FLT_MAX, sum = 0.f;
  for (int w = 0; w < kGeneralWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kGeneralWarps; ++w) sum += s_l[w] * exp2f(s_m[w] - top);
  for (int d = threadIdx.x; d < p.dim; d += 32 * kGeneralWarps) {
    float acc = 0.f;
    for (int w = 0; w < kGeneralWarps; ++w) acc += s_o[w][d] * exp2f(s_m[w] - top);
    p.out[r * p.o_s[0] + h * p.o_s[1] + d] = some ? acc / sum : 0.f;
  }
  if (threadIdx.x == 0 && p.lse != nullptr) {
    p.lse[r * p.heads + h] = some ? top * 0.69314718055994531f + logf(sum) : -INFINITY;
  }
}

// ---- the streaming form -------------------------------------------------------
//
// Bound by the stream of keys and values (2 * head_dim elements a position and
// key head), so the work is cut by bytes, not by requests: every (request, key
// head) is cut into tiles of kTile positions, and CTA c of G takes the tiles
// [c N / G, (c + 1) N / G) of all N in the order request, key head, position.
// The lengths are read on the device; nothing of this is known to the host.
// A CTA walks through the segments of its range.  A segment that is all of its
// (request, key head) is written out; of any other the CTA leaves maximum, sum
// and unnormalised output in the workspace, and the last CTA to arrive at that
// (request, key head), told by a counter, joins the parts in the order of the
// CTAs: the result does not depend on which one was last.
//   128 requests of 200 to 8000 keys, 12 heads of 64, fp32: 257 us, 6.6 TB/s;
//   61 of 100 to 16000 keys, 64 heads of 128 on 8, f16: 144 us, 5.6 TB/s;
//   2 of 63000 and 100001 keys, 32 heads of 128 on 8, bf16: 121 us, 5.5 TB/s;
//   1 of 777 keys, 12 heads of 64, fp32: 8.6 us, which is latency.
// To begin a unit costs as much as some tiles; a unit's first tile counts for
// kSetup more when the work is cut, without which CTAs of many short units end
// last (kSetup 1: 273, 156 and 123 us for the first three).  A CTA takes kShare
// tiles at least: with half of it the single request above takes 10.5 us and one
// of 12000 keys and 16 heads in one unit 33.2 us instead of 32.4, with twice of
// it 9.3 and 41.5 us.  The last CTA joins up to kJoinAtOnce parts; of more,
// groups of kJoinGroup are joined first, by the last CTA of each (that request:
// 51 us when one CTA joins them all).
//
// In a CTA each warp streams its own kKeys positions of every tile through a
// ring of kStages stages in shared memory (16-byte cp.async; a warp waits for
// nobody else).  Bulk copies of whole rows carry the same bytes with fewer
// instructions, but a warp issues one in 80 cycles, 1300 to 2600 for a stage,
// which is what bounded short requests.  Positions past the length, and pages
// out of range, are filled with zeros instead of read, and their scores set to
// -inf, so that what the pages hold there (NaN, infinities) does not matter.
// The rows are padded so that the reads below are free of bank conflicts.
//
// The running maximum moves only when a score exceeds it by 8 (a factor 2^8 in
// the exp2 domain, exact after the division by the sum), so that the rescaling
// of the outputs is rare; it starts at -FLT_MAX as in the general form.
//
// MT = 0, one query head a key head: DP / 16 lanes share a position, 16
// dimensions each, fp32 FMAs.
//
// MT > 0, 8 MT query heads a key head: tensor cores (mma.sync with 16 rows,
// fp32 sums), which take operands of 8 or 11 bits.  A query or weight is
// therefore cut into terms that together carry 22 to 24 bits, each product of
// a term with a page element is exact, and only the terms' sums lose bits (the
// tensor core cuts them off: relative errors of outputs to 1.1e-6, for 1.5e-7
// to 2.1e-7 of MT = 0):
//   f16 pages:  x = hi + lo in f16, rows h and h + 8 of the 16.  f16 has little
//     range, so a head's query is scaled by a power of two to 2^13 and weights
//     by 2^7 (both are taken back exactly);
//   bf16 pages: x = hi + mid + lo in bf16, the third in a second product; with
//     at most four heads (PACKED) in rows h + 4 of the same one, for which a
//     head's scores are made in two lanes, 16 apart;
//   f32 pages:  x = hi + lo in tf32, and so are keys and values, their hi and
//     lo in a product each; of lo's 12 or 13 bits tf32 takes 11.
// A lane's scores are its own weights of the second product, and rows h and
// h + 8 of a sum are in one lane: nothing is exchanged between lanes.
constexpr int kMaxCtas = 640;  // bound on a launch's CTAs; sizes the workspace
constexpr int kCounterBytes = 8192;  // three counters a CTA
constexpr int kJoinAtOnce = 24, kJoinGroup = 16;
constexpr float kSlack = 8.f;
constexpr int kSetup = 3;

template <typename T, int DP, int MT, bool PACKED>
struct Stream {
  static constexpr int kElem = static_cast<int>(sizeof(T));
  static constexpr int kChunk = 16 / kElem;        // elements of a 16-byte chunk
  static constexpr int kRow = DP / kChunk;         // chunks of a row
  static constexpr int kRowBytes = DP * kElem;
  static constexpr bool kBf16 = MT > 0 && std::is_same<T, __nv_bfloat16>::value;
  // 4 KB a stage; for the tensor cores as many steps of 8 positions as make
  // 8 KB, 16 at most
  static constexpr int kKeys = MT == 0 ? 2048 / kRowBytes : kElem == 2 && DP <= 128 ? 16 : 8;
  static constexpr int kWarps = 4;
  static constexpr int kThreads = 32 * kWarps;
  // by registers: 16 a lane for the output of MT = 0, MT * DP / 2 for MT > 0;
  // and for 512-byte rows by shared memory
  static constexpr int kCtasPerSm = MT == 0            ? 4
                                    : kRowBytes > 512  ? 1
                                    : MT * DP <= 128 && kRowBytes <= 256 ? 3
                                                       : 2;
  // Row pitches.  MT = 0: the lanes of odd rows take their chunks in another
  // order, so that rows need no padding.  Tensor cores: 16-bit rows are read
  // eight at a time, a chunk each; f32 keys two rows of four chunks, f32 values
  // four even or odd rows of two.  The padding puts these on banks of their own.
  static constexpr int kPitchK = kRowBytes + (MT == 0 ? 0 : kElem == 4 ? 64 : 16);
  static constexpr int kPitchV = kRowBytes + (MT == 0 ? 0 : 16);
  static constexpr int kHalf = kKeys * kPitchK;  // keys, then values
  static constexpr int kStage = kHalf + kKeys * kPitchV;
  static constexpr int kTile = kWarps * kKeys;
  // the least that a CTA takes: parts of more heads are more to join
  static constexpr int kShare = MT == 0 ? 2 : 4;
  static constexpr int kHeads = MT == 0 ? 1 : PACKED ? 4 : 8 * MT;
  static_assert(!PACKED || (kBf16 && MT == 1), "packed rows");
  // query fragments of a k step of 16 (f32: 8): 16 bytes a lane, for bf16 8 more
  static constexpr int kSteps = kElem == 4 ? DP / 8 : DP / 16;
  static constexpr int kFrags = kBf16 && !PACKED ? 2 : 1;
  static constexpr int kQueryBytes = MT * kSteps * (kFrags == 2 ? 768 : 512);
  // MT = 0: the warps' parts, or the sums of eight groups of lanes that join a
  // unit's parts; MT > 0: in the ring
  static constexpr int kPartBytes = MT == 0 ? (DP == 64 ? 8 : 4) * DP * 4 : 0;
  // As many stages as an SM's shared memory (228 KB, one of it taken by each
  // CTA) holds, four at most; besides the ring there are the arrays declared in
  // the kernel.
  static constexpr int dynamic_bytes(int stages) {
    return kWarps * stages * kStage + kQueryBytes + kPartBytes;
  }
  static constexpr bool fits(int stages) {
    const int arrays = 128 + kWarps * (4 * stages + 12 * kHeads + 16) + 12 * kHeads +
                       4 * kWarps * (MT == 0 ? stages : stages - 1) * kKeys;
    return dynamic_bytes(stages) + arrays <= 228 * 1024 / kCtasPerSm - 1024;
  }
  static constexpr int kStages = fits(4) ? 4 : fits(3) ? 3 : fits(2) ? 2 : 1;
  static constexpr int kWarpRing = kStages * kStage;
  static constexpr int kSmem = dynamic_bytes(kStages);
  static_assert(kStages >= 2 && kKeys <= 16, "the ring");
  static_assert(MT == 0 || kStage >= kHeads * (DP + 8) * 4, "a part takes the place of a stage");
  // floats of one head's part: output, maximum, sum, whether a position counts
  static constexpr int kRecord = DP + 4;
};

struct StreamParams {
  AttendParams a;
  int requests;
  int key_heads;
  int subs;  // units of a key head: ceil(group / heads a unit)
  int* counters;
  float* parts;
};

using tc::smem_u32;

// 16 bytes from global to shared memory; or 16 zeros, with nothing read.
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16 : 0)
               : "memory");
}
// N bytes (4 or 8) from global to shared memory, waited for by cp.async.wait_all.
template <int N>
__device__ __forceinline__ void fetch_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(N)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ void lds64(uint32_t addr, uint32_t& x, uint32_t& y) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(addr));
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}

// dst[0 .. 3] = x f, in one store where dst allows it.
__device__ __forceinline__ void put_four(float* dst, const float4& x, float f) {
  const float4 y = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
  if ((reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
    *reinterpret_cast<float4*>(dst) = y;
  } else {
    dst[0] = y.x;
    dst[1] = y.y;
    dst[2] = y.z;
    dst[3] = y.w;
  }
}

// The elements of a chunk as fp32.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& c, float (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// fp32 values rounded to the page type, as a chunk.
template <typename T>
__device__ __forceinline__ uint4 pack(const float* src) {
  T t[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) from_f32(t[i], src[i]);
  uint4 c;
  memcpy(&c, t, 16);
  return c;
}

// x = hi + lo: hi carries the leading 11 bits (rounded), which tf32 holds.
__device__ __forceinline__ void split_rounded(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

// d = a b + c, all registers; FIRST: c is zero.
#define TVR_MMA(shape_types, a_list, b_list, ...)                                              \
  if constexpr (FIRST) {                                                                       \
    asm volatile("mma.sync.aligned." shape_types " {%0, %1, %2, %3}, " a_list ", " b_list      \
                 ", {%10, %10, %10, %10};"                                                     \
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                              \
                 : __VA_ARGS__, "f"(0.f));                                                     \
  } else {                                                                                     \
    asm volatile("mma.sync.aligned." shape_types " {%0, %1, %2, %3}, " a_list ", " b_list      \
                 ", {%0, %1, %2, %3};"                                                         \
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                              \
                 : __VA_ARGS__, "f"(0.f));                                                     \
  }

template <bool FIRST>
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  TVR_MMA("m16n8k8.row.col.f32.tf32.tf32.f32", "{%4, %5, %6, %7}", "{%8, %9}", "r"(a.x), "r"(a.y),
          "r"(a.z), "r"(a.w), "r"(b0), "r"(b1))
}

// 16-bit operands, 16 or 8 products a sum.
template <typename T, bool FIRST>
__device__ __forceinline__ void mma_k16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    TVR_MMA("m16n8k16.row.col.f32.f16.f16.f32", "{%4, %5, %6, %7}", "{%8, %9}", "r"(a.x), "r"(a.y),
            "r"(a.z), "r"(a.w), "r"(b0), "r"(b1))
  } else {
    TVR_MMA("m16n8k16.row.col.f32.bf16.bf16.f32", "{%4, %5, %6, %7}", "{%8, %9}", "r"(a.x),
            "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1))
  }
}
template <typename T, bool FIRST>
__device__ __forceinline__ void mma_k8(float (&c)[4], const uint4& a, uint32_t b0) {
  if constexpr (std::is_same<T, __half>::value) {
    TVR_MMA("m16n8k8.row.col.f32.f16.f16.f32", "{%4, %5}", "{%8}", "r"(a.x), "r"(a.y), "r"(0),
            "r"(0), "r"(b0), "r"(0))
  } else {
    TVR_MMA("m16n8k8.row.col.f32.bf16.bf16.f32", "{%4, %5}", "{%8}", "r"(a.x), "r"(a.y), "r"(0),
            "r"(0), "r"(b0), "r"(0))
  }
}
#undef TVR_MMA

// Four 8 x 8 matrices of 16-bit elements, lane l giving row l % 8 of matrix
// l / 8; lane 4 g + t gets elements (g, 2 t) and (g, 2 t + 1) of each, or of
// its transpose.
template <bool TRANSPOSED>
__device__ __forceinline__ uint4 ldmatrix4(uint32_t addr) {
  uint4 v;
  if constexpr (TRANSPOSED) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
  } else {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
  }
  return v;
}

// Two values rounded to T, packed; x and y become what the rounding left.
template <typename T>
__device__ __forceinline__ uint32_t take_term(float& x, float& y) {
  T t[2];
  from_f32(t[0], x);
  from_f32(t[1], y);
  x -= to_f32(t[0]);
  y -= to_f32(t[1]);
  uint32_t v;
  memcpy(&v, t, 4);
  return v;
}

template <typename T, int DP, int MT, bool PACKED>
__global__ void __launch_bounds__(Stream<T, DP, MT, PACKED>::kThreads,
                                  Stream<T, DP, MT, PACKED>::kCtasPerSm)
    paged_attention_stream_kernel(const __grid_constant__ StreamParams sp) {
  using S = Stream<T, DP, MT, PACKED>;
  constexpr int CH = S::kChunk, ROW = S::kRow, KEYS = S::kKeys, HEADS = S::kHeads;
  constexpr int WARPS = S::kWarps, THREADS = S::kThreads;
  constexpr unsigned FULL = 0xffffffffu;
  [[maybe_unused]] constexpr bool HALFS = std::is_same<T, __half>::value;
  const AttendParams& p = sp.a;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_scan[WARPS];
  __shared__ long long s_before;
  __shared__ int s_request, s_found, s_last;
  __shared__ uint32_t s_live[WARPS][S::kStages];
  __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS], s_f[WARPS][HEADS];
  __shared__ float s_top[HEADS], s_sum[HEADS], s_inverse[HEADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // ---- this CTA's range of tiles
  const int units = sp.key_heads * sp.subs;
  auto length = [&](int r) { return max(0, min(p.max_keys, p.lens[r])); };
  // An empty request has one tile, of no positions: somebody writes its row.
  // A unit's first tile counts for kSetup more, what it costs to begin one.
  auto tiles = [&](int n) { return max(1, (n + S::kTile - 1) / S::kTile) + kSetup; };
  // The first THREADS requests' inclusive sums are kept; further ones are only
  // summed, and scanned below where the range begins among them.
  auto scan = [&](long long x) -> long long {  // inclusive, over the CTA
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long below = __shfl_up_sync(FULL, x, d);
      if (lane >= d) x += below;
    }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS - 1; ++w) x += w < warp ? s_scan[w] : 0;
    return x;
  };
  const int my_length = tid < sp.requests ? length(tid) : 0;
  const int my_tiles = tid < sp.requests ? tiles(my_length) : 0;
  const long long my_end = scan(my_tiles);
  long long head_tiles = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) head_tiles += s_scan[w];
  total = head_tiles;
  if (sp.requests > THREADS) {
    long long own = 0;
    for (int q = THREADS + tid; q < sp.requests; q += THREADS) own += tiles(length(q));
    __syncthreads();
    own = scan(own);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += s_scan[w];
  }
  total *= units;
  const long long ctas = min(static_cast<long long>(gridDim.x), max(1ll, total / S::kShare));
  const long long cta = blockIdx.x;
  if (cta >= ctas) return;
  // tile x belongs to CTA ((x + 1) ctas - 1) / total; CTA c begins at c total / ctas
  auto divide = [](long long x, long long y) -> long long {  // x, y >= 0
    return ((x | y) >> 32) == 0 ? static_cast<uint32_t>(x) / static_cast<uint32_t>(y) : x / y;
  };
  long long u = divide(cta * total, ctas);
  const long long u_end = divide((cta + 1) * total, ctas);
  int r, n;
  {
    const long long target = divide(u, units);
    if (my_tiles > 0 && my_end > target && my_end - my_tiles <= target) {
      s_request = tid;
      s_found = my_length;
      s_before = my_end - my_tiles;
    }
    long long before = head_tiles;
    for (int base = THREADS; before <= target; base += THREADS) {
      __syncthreads();
      const int q = base + tid;
      const int of_q = q < sp.requests ? length(q) : 0;
      const int t = q < sp.requests ? tiles(of_q) : 0;
      const long long end = before + scan(t);
      if (q < sp.requests && end > target && end - t <= target) {
        s_request = q;
        s_found = of_q;
        s_before = end - t;
      }
#pragma unroll
      for (int w = 0; w < WARPS; ++w) before += s_scan[w];
    }
    __syncthreads();
    r = s_request;
    n = s_found;
  }
  int count = tiles(n);
  const long long in_request = u - s_before * units;
  int unit = static_cast<int>(divide(in_request, count));
  int t0 = static_cast<int>(in_request - static_cast<long long>(unit) * count);

  const uint32_t ring = smem_u32(smem) + warp * S::kWarpRing;
  const int cols = p.dim / CH;  // chunks of a row that exist
  // pages hold whole stages
  const bool aligned = (p.page.d & (KEYS - 1)) == 0 && cols == ROW;
  // The ring, over all segments: the stage to be filled, the stage to be read.
  int put = 0, get = 0;
  // Where a warp leaves its part of a segment: MT = 0, in a place of its own;
  // MT > 0, in the stage of its ring that is filled last.
  auto part_of = [&](int w) -> float* {
    if constexpr (MT == 0) {
      return reinterpret_cast<float*>(smem + WARPS * S::kWarpRing) + w * DP;
    } else {
      const int stage = put == 0 ? S::kStages - 1 : put - 1;
      return reinterpret_cast<float*>(smem + w * S::kWarpRing + stage * S::kStage);
    }
  };
  constexpr int PART = MT == 0 ? DP : DP + 8;  // floats from one head of a part to the next
  // Stages that are filled before the parts of the segment before are joined;
  // what that takes (length, slot, pages) is fetched during that segment.
  constexpr int EARLY = MT == 0 ? S::kStages : S::kStages - 1;
  __shared__ int s_pages[WARPS][EARLY][KEYS], s_length[WARPS];
  __shared__ int64_t s_slot[WARPS];

  // ---- the segment at hand: positions of (request r, unit), tiles real0 to
  // real1 without what stands for the setup; a range that ends there leaves the
  // unit to the next CTA
  int t1 = 0, real0 = 0, stages = 0, first = 0, fresh = -1, g = 0, sub = 0;
  int64_t slot = -1;
  auto slot_of = [&](int q) -> int64_t { return p.slots != nullptr ? p.slots[q] : -1; };
  // the rest of the segment's numbers; false if it has no tiles
  auto begin = [&]() -> bool {
    t1 = static_cast<int>(min(static_cast<long long>(count), t0 + (u_end - u)));
    real0 = max(0, t0 - kSetup);
    stages = t1 - kSetup - real0;
    first = real0 * S::kTile + warp * KEYS;  // the warp's first position of stage 0
    g = unit / sp.subs;
    sub = unit - g * sp.subs;
    fresh = n > 0 && slot >= 0 && slot < p.n_slots ? n - 1 : -1;
    if (n > 0 && slot >= p.n_slots && tid == 0) report(p.status, TVR_DEV_BAD_INDEX);
    return t1 > kSetup;
  };

  // ---- the ring: stage i holds this warp's positions of tile real0 + i
    // The lanes hold the pages of the rows l % KEYS, and copy the 16-byte chunks
    // 32 c + l of the keys and of the values.
    constexpr uint32_t ROWS_MASK = (1u << KEYS) - 1u;
    constexpr int STEPS = KEYS * ROW / 32;
    const int my_row = lane % KEYS;
    // The page of position j of request q, wherever the table has one: whether
    // the position counts is decided when its row is copied.
    auto page_at = [&](int q, int j) -> int {
      if (j >= p.max_keys) return -1;
      return p.table[q * p.table_stride + fast_div(static_cast<uint32_t>(j), p.page)];
    };
    auto page_of = [&](int i) -> int {
      return i < stages ? page_at(r, first + i * S::kTile + my_row) : -1;
    };
    int filled = 0;  // stages of the segment
    auto fill = [&](int page) {  // the next stage, row l % KEYS from `page`
      if (filled < stages) {
        const uint32_t kd = ring + put * S::kStage, vd = kd + S::kHalf;
        const int j0 = first + filled * S::kTile;
        const int new_row = fresh - j0;  // the row of the new position, if 0 <= it < KEYS
        const bool has_new = fresh >= 0 && new_row >= 0 && new_row < KEYS;
        const bool exists = static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages);
        const T* const kg = static_cast<const T*>(p.k) + g * p.k_s[1];
        const T* const vg = static_cast<const T*>(p.v) + g * p.v_s[1];
        if (aligned && j0 + KEYS <= n && !has_new && __all_sync(FULL, exists)) {
          // one page and all of its rows: the chunks are a constant step apart
          const int row0 = j0 - static_cast<int>(fast_div(static_cast<uint32_t>(j0), p.page) *
                                                 p.page.d) + (ROW <= 32 ? lane / ROW : 0);
          const int col = ROW <= 32 ? lane % ROW : lane;
          const T* ks = kg + page * p.k_s[0] + row0 * p.k_s[2] + col * CH;
          const T* vs = vg + page * p.v_s[0] + row0 * p.v_s[2] + col * CH;
          const uint32_t kc = kd + (ROW <= 32 ? lane / ROW : 0) * S::kPitchK + col * 16;
          const uint32_t vc = vd + (ROW <= 32 ? lane / ROW : 0) * S::kPitchV + col * 16;
          if constexpr (ROW <= 32) {
            const int64_t kn = (32 / ROW) * p.k_s[2], vn = (32 / ROW) * p.v_s[2];
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
              copy_async(kc + c * (32 / ROW) * S::kPitchK, ks);
              copy_async(vc + c * (32 / ROW) * S::kPitchV, vs);
              ks += kn;
              vs += vn;
            }
          } else {
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
              copy_async(kc + (c / 2) * S::kPitchK + (c % 2) * 512, ks + (c % 2) * 32 * CH);
              copy_async(vc + (c / 2) * S::kPitchV + (c % 2) * 512, vs + (c % 2) * 32 * CH);
              if (c % 2 == 1) {
                ks += p.k_s[2];
                vs += p.v_s[2];
              }
            }
          }
          if (lane == 0) s_live[warp][put] = ROWS_MASK;
        } else {
          // row by row: zeros for what does not count, nothing for the new row
          const int j = j0 + my_row;
          const bool counts = j < n && j != fresh;
          if (counts && !exists) report(p.status, TVR_DEV_BAD_INDEX);
          const uint32_t read = __ballot_sync(FULL, counts && exists) & ROWS_MASK;
          if (lane == 0) s_live[warp][put] = read | (has_new ? 1u << new_row : 0u);
          const int in_page =
              j - static_cast<int>(fast_div(static_cast<uint32_t>(j), p.page) * p.page.d);
          const int64_t ko = page * p.k_s[0] + in_page * p.k_s[2];
          const int64_t vo = page * p.v_s[0] + in_page * p.v_s[2];
#pragma unroll 1
          for (int c = 0; c < STEPS; ++c) {
            const int row = (c * 32 + lane) / ROW, col = (c * 32 + lane) % ROW;
            const int64_t ks = __shfl_sync(FULL, ko, row), vs = __shfl_sync(FULL, vo, row);
            const bool live = ((read >> row) & 1u) != 0 && col < cols;
            if (has_new && row == new_row && col < cols) continue;
            copy_async_or_zero(kd + row * S::kPitchK + col * 16, live ? kg + ks + col * CH : kg,
                               live);
            copy_async_or_zero(vd + row * S::kPitchV + col * 16, live ? vg + vs + col * CH : vg,
                               live);
          }
        }
        put = put + 1 == S::kStages ? 0 : put + 1;
        ++filled;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");  // a stage, or nothing
    };
    // The new position, if stage i (the one to be read) has it: from k_new and
    // v_new into its row and its slot, while the stage's copies are under way.
    auto place_new = [&](int i) {
      const int row = fresh - (first + i * S::kTile);
      if (fresh < 0 || row < 0 || row >= KEYS) return;
      const uint32_t stage = ring + get * S::kStage;
      const float* kn = p.k_new + r * p.kn_s[0] + g * p.kn_s[1];
      const float* vn = p.v_new + r * p.vn_s[0] + g * p.vn_s[1];
      const int64_t page = divide(slot, p.page.d), at = slot - page * p.page.d;
      T* kc = static_cast<T*>(p.k) + page * p.k_s[0] + g * p.k_s[1] + at * p.k_s[2];
      T* vc = static_cast<T*>(p.v) + page * p.v_s[0] + g * p.v_s[1] + at * p.v_s[2];
      for (int col = lane; col < cols; col += 32) {
        const uint4 kx = pack<T>(kn + col * CH), vx = pack<T>(vn + col * CH);
        if (sub == 0) {
          *reinterpret_cast<uint4*>(kc + col * CH) = kx;
          *reinterpret_cast<uint4*>(vc + col * CH) = vx;
        }
        sts128(stage + row * S::kPitchK + col * 16, kx);
        sts128(stage + S::kHalf + row * S::kPitchV + col * 16, vx);
      }
    };
    // Waits for the stage to be read.
    auto ready = [&]() {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
      __syncwarp();
    };
    auto advance = [&]() {
      __syncwarp();
      get = get + 1 == S::kStages ? 0 : get + 1;
    };
  // the first segment
  slot = slot_of(r);
  int ahead[EARLY + 1];  // pages of the stages to be filled next
#pragma unroll
  for (int i = 0; i <= EARLY; ++i) {
    ahead[i] = page_at(r, max(0, t0 - kSetup) * S::kTile + warp * KEYS + i * S::kTile + my_row);
  }
  if (!begin()) return;
#pragma unroll
  for (int i = 0; i < EARLY; ++i) fill(ahead[i]);
  int next_page = ahead[EARLY];

  for (bool more = true; more;) {
    if constexpr (MT > 0) {
      const int page = next_page;
      next_page = page_of(filled + 1);
      fill(page);
    }
    const int h0 = g * p.group + sub * HEADS;
    const int heads = min(HEADS, p.group - sub * HEADS);
    bool counted = false;  // whether any position of this warp's counts
    // the segment after this one begins a unit, if there is one
    const bool follow = u + (t1 - t0) < u_end;
    const int n_unit = unit + 1 < units ? unit + 1 : 0, n_request = r + (unit + 1 < units ? 0 : 1);
    if (follow) {
#pragma unroll
      for (int i = 0; i < EARLY; ++i) {
        const int j = warp * KEYS + i * S::kTile + lane;
        if (lane < KEYS && j < p.max_keys) {
          fetch_async<4>(&s_pages[warp][i][lane],
                         p.table + n_request * p.table_stride +
                             fast_div(static_cast<uint32_t>(j), p.page));
        }
      }
      if (lane == 0) {
        fetch_async<4>(&s_length[warp], p.lens + n_request);
        if (p.slots != nullptr) fetch_async<8>(&s_slot[warp], p.slots + n_request);
      }
    }

    if constexpr (MT == 0) {
      constexpr int L = DP / 16, NC = 16 / CH, STEP = 32 / L;
      const int lead = lane & (L - 1);
      // chunk c of this lane, in the order that it reads them
      const int turn = L < 8 ? (lane / L) & 1 : 0;
      auto chunk = [&](int c) { return (c ^ turn) * L + lead; };
      float q[NC][CH], o[NC][CH];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = chunk(c) * CH;
        const float* src = p.q + r * p.q_s[0] + h0 * p.q_s[1] + d;
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          q[c][e] = d < p.dim ? src[e] * p.scale_log2 : 0.f;
          o[c][e] = 0.f;
        }
      }
      float m = -FLT_MAX, l = 0.f;  // m: one for the warp
      for (int i = 0; i < stages; ++i) {
        place_new(i);
        ready();
        const uint32_t kd = ring + get * S::kStage, vd = kd + S::kHalf;
        const uint32_t live = s_live[warp][get];
        counted |= live != 0;
#pragma unroll
        for (int it = 0; it < KEYS / STEP; ++it) {
          const int row = it * STEP + lane / L;
          const uint32_t rk = kd + row * S::kPitchK, rv = vd + row * S::kPitchV;
          float s = 0.f;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            float k[CH];
            unpack<T>(lds128(rk + chunk(c) * 16), k);
#pragma unroll
            for (int e = 0; e < CH; ++e) s = fmaf(q[c][e], k[e], s);
          }
#pragma unroll
          for (int x = 1; x < L; x <<= 1) s += __shfl_xor_sync(FULL, s, x);
          s = ((live >> row) & 1u) != 0 ? s : -INFINITY;
          if (__any_sync(FULL, s > m + kSlack)) {
            float top = s;
#pragma unroll
            for (int x = L; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, x));
            top = fmaxf(top, m);
            const float keep = exp2f(m - top);
            m = top;
            l *= keep;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
              for (int e = 0; e < CH; ++e) o[c][e] *= keep;
            }
          }
          const float w = exp2f(s - m);
          l += w;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            float v[CH];
            unpack<T>(lds128(rv + chunk(c) * 16), v);
#pragma unroll
            for (int e = 0; e < CH; ++e) o[c][e] = fmaf(w, v[e], o[c][e]);
          }
        }
        advance();
        const int page = next_page;
        next_page = page_of(filled + 1);
        fill(page);
      }
      // the rows' sums, lanes of even and odd rows apart as their orders differ
      constexpr int TURNED = L < 8 ? 2 * L : L;
#pragma unroll
      for (int x = TURNED; x < 32; x <<= 1) {
        l += __shfl_xor_sync(FULL, l, x);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
          for (int e = 0; e < CH; ++e) o[c][e] += __shfl_xor_sync(FULL, o[c][e], x);
        }
      }
      if constexpr (L < 8) {
        l += __shfl_xor_sync(FULL, l, L);
        // chunk c of an even row's lane is chunk c ^ 1 of an odd row's
#pragma unroll
        for (int c = 0; c < NC; c += 2) {
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            const float a = __shfl_xor_sync(FULL, o[c][e], L);
            const float b = __shfl_xor_sync(FULL, o[c + 1][e], L);
            o[c][e] += b;
            o[c + 1][e] += a;
          }
        }
      }
      if (lane < L) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
          for (int e = 0; e < CH; ++e) part_of(warp)[chunk(c) * CH + e] = o[c][e];
        }
      }
      if (lane == 0) {
        s_m[warp][0] = m;
        s_l[warp][0] = l;
      }
    } else {
      // lane = 4 grp + thr: rows grp and grp + 8 of a fragment (head grp's terms)
      constexpr int KS = S::kSteps, NT = KEYS / 8, MTR = MT > 0 ? MT : 1, XT = DP / 8;
      constexpr float LIFT = HALFS ? 7.f : 0.f;
      const int grp = lane >> 2, thr = lane & 3;
      const uint32_t query0 = smem_u32(smem + WARPS * S::kWarpRing), query = query0 + lane * 16;
      const uint32_t third = query + MTR * KS * 512 - lane * 8;  // bf16: the third terms

      // ---- the query's fragments, shared by the warps
      // DP / 8 lanes a head, eight dimensions each
      for (int x = tid; x < HEADS * (DP / 8); x += THREADS) {
        const int h = x / (DP / 8), j = x % (DP / 8);
        const float* src = p.q + r * p.q_s[0] + (h0 + h) * p.q_s[1] + 8 * j;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = h < heads && 8 * j + e < p.dim ? src[e] * p.scale_log2 : 0.f;
        }
        if constexpr (HALFS) {
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
          for (int d = 1; d < DP / 8; d <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, d));
          // 2^(13 - exponent of top): down to 2^-114, up to 2^100 (smaller
          // queries make scores that are zero to fp32's last bit all the same)
          const int e2 = static_cast<int>((__float_as_uint(top) >> 23) & 255u);
          const int lift = e2 == 0 || e2 == 255 ? 0 : min(100, 13 - (e2 - 127));
          const float up = __uint_as_float(static_cast<uint32_t>(127 + lift) << 23);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= up;
          if (j == 0) s_top[h] = __uint_as_float(static_cast<uint32_t>(127 - lift) << 23);
        }
        const int mt = h / 8;
        const uint32_t row = static_cast<uint32_t>(h % 8) * 4;  // its first lane
        if constexpr (sizeof(T) == 4) {
          // step 2 c + e takes, of chunk 4 c + thr, element 2 e as product thr
          // and element 2 e + 1 as product thr + 4
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int chunk = 2 * j + (y >> 1), ks = 2 * (chunk >> 2) + (y & 1);
            uint4 f;
            split_rounded(v[2 * y], f.x, f.y);
            split_rounded(v[2 * y + 1], f.z, f.w);
            sts128(query0 + (mt * KS + ks) * 512 + (row + (chunk & 3)) * 16, f);
          }
        } else {
          // step ks takes dimensions 16 ks + 2 thr and the next one as products
          // 2 thr and 2 thr + 1, and those 8 further as 2 thr + 8 and 2 thr + 9
          const int ks = mt * KS + (j >> 1);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint32_t hi = take_term<T>(v[2 * y], v[2 * y + 1]);
            const uint32_t mid = take_term<T>(v[2 * y], v[2 * y + 1]);
            const uint32_t at = query0 + ks * 512 + (row + y) * 16 + (j & 1) * 8;
            sts64(at, hi, mid);
            if constexpr (PACKED) sts64(at + 256, take_term<T>(v[2 * y], v[2 * y + 1]), 0);
            if constexpr (S::kFrags == 2) {
              const uint32_t lo = take_term<T>(v[2 * y], v[2 * y + 1]);
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(query0 + MTR * KS * 512 + ks * 256 +
                                                          (row + y) * 8 + (j & 1) * 4),
                           "r"(lo)
                           : "memory");
            }
          }
        }
      }
      __syncthreads();
      float unscale[MTR];  // f16: takes the scaling of head mt * 8 + grp back
#pragma unroll
      for (int mt = 0; mt < MTR; ++mt) unscale[mt] = HALFS ? s_top[mt * 8 + grp] : 1.f;

      float o[MTR][XT][4], m[MTR], l[MTR];
#pragma unroll
      for (int mt = 0; mt < MTR; ++mt) {
        m[mt] = -FLT_MAX;
        l[mt] = 0.f;
#pragma unroll
        for (int x = 0; x < XT; ++x) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][x][e] = 0.f;
        }
      }
      for (int i = 0; i < stages; ++i) {
        place_new(i);
        ready();
        const uint32_t kd = ring + get * S::kStage, vd = kd + S::kHalf;
        const uint32_t live = s_live[warp][get];
        counted |= live != 0;

        // ---- scores
        constexpr int CHAINS = sizeof(T) == 4 ? 2 : 1;
        float s[MTR][NT][CHAINS][4];
#pragma unroll
        for (int mt = 0; mt < MTR; ++mt) {
#pragma unroll
          for (int x = 0; x < NT * CHAINS * 4; ++x) s[mt][x / (CHAINS * 4)][x / 4 % CHAINS][x % 4] = 0.f;
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < ROW / 4; ++c) {
            float k[CH];
            unpack<T>(lds128(kd + grp * S::kPitchK + (4 * c + thr) * 16), k);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t k0, k1, r0, r1;
              split_rounded(k[2 * e], k0, r0);
              split_rounded(k[2 * e + 1], k1, r1);
#pragma unroll
              for (int mt = 0; mt < MTR; ++mt) {
                const uint4 a = lds128(query + (mt * KS + 2 * c + e) * 512);
                mma_tf32<false>(s[mt][0][e], a, r0, r1);
                mma_tf32<false>(s[mt][0][e], a, k0, k1);
              }
            }
          }
        } else {
          const uint32_t rk = kd + (lane & 7) * S::kPitchK + (lane >> 3) * 16;
#pragma unroll
          for (int c = 0; c < KS / 2; ++c) {  // 32 dimensions
            uint4 k[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              k[nt] = ldmatrix4<false>(rk + nt * 8 * S::kPitchK + c * 64);
            }
#pragma unroll
            for (int mt = 0; mt < MTR; ++mt) {
#pragma unroll
              for (int f = 0; f < S::kFrags; ++f) {
                const int x = mt * KS + 2 * c;
                uint4 a = make_uint4(0, 0, 0, 0), b = a;
                if (f == 0) {
                  a = lds128(query + x * 512);
                  b = lds128(query + x * 512 + 512);
                } else {
                  lds64(third + x * 256, a.x, a.z);
                  lds64(third + x * 256 + 256, b.x, b.z);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_k16<T, false>(s[mt][nt][0], a, k[nt].x, k[nt].y);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_k16<T, false>(s[mt][nt][0], b, k[nt].z, k[nt].w);
              }
            }
          }
        }
        // of head grp at positions 8 nt + 2 thr and the next one: the sum of
        // the two rows of that head
        float z[MTR][NT][2];
        bool over = false;
#pragma unroll
        for (int mt = 0; mt < MTR; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float hi = s[mt][nt][0][e], lo = s[mt][nt][0][e + 2];
              if constexpr (CHAINS == 2) {
                hi += s[mt][nt][1][e];
                lo += s[mt][nt][1][e + 2];
              }
              float v = hi + lo;
              if constexpr (HALFS) v *= unscale[mt];
              if constexpr (PACKED) v += __shfl_xor_sync(FULL, v, 16);
              const bool in = ((live >> (nt * 8 + 2 * thr + e)) & 1u) != 0;
              z[mt][nt][e] = in ? v : -INFINITY;
              // of the difference, which is what the weight is made of: past
              // 2^25, m + 15 may round up to m + 16, and an f16 weight of 2^16
              // is an infinity
              over |= z[mt][nt][e] - m[mt] > LIFT + kSlack;
            }
          }
        }
        // m is the running maximum less LIFT: weights end below 2^(LIFT + 8)
        if (__any_sync(FULL, over)) {
#pragma unroll
          for (int mt = 0; mt < MTR; ++mt) {
            float top = z[mt][0][0];
#pragma unroll
            for (int x = 1; x < 2 * NT; ++x) top = fmaxf(top, z[mt][x >> 1][x & 1]);
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
            top = fmaxf(m[mt], top - LIFT);
            const float keep = exp2f(m[mt] - top);
            m[mt] = top;
            l[mt] *= keep;
#pragma unroll
            for (int x = 0; x < XT; ++x) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[mt][x][e] *= keep;
            }
          }
        }

        // ---- weights, as fragments: positions 2 thr and 2 thr + 1 of each 8
        float w[MTR][NT][2];
#pragma unroll
        for (int mt = 0; mt < MTR; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            w[mt][nt][0] = exp2f(z[mt][nt][0] - m[mt]);
            w[mt][nt][1] = exp2f(z[mt][nt][1] - m[mt]);
            l[mt] += w[mt][nt][0] + w[mt][nt][1];
          }
        }
        // ---- outputs.  The stage's products are summed on their own and then
        // added in fp32: the tensor core cuts its running sum off below, which
        // would show in a sum over many stages.
        if constexpr (sizeof(T) == 4) {
          uint4 a[MTR];
#pragma unroll
          for (int mt = 0; mt < MTR; ++mt) {
            split_rounded(w[mt][0][0], a[mt].x, a[mt].y);
            split_rounded(w[mt][0][1], a[mt].z, a[mt].w);
          }
          // product thr is position 2 thr, product thr + 4 the next one; tile
          // c * 4 + e takes, of chunk 8 c + grp, element e
          const uint32_t rv = vd + 2 * thr * S::kPitchV + grp * 16;
#pragma unroll
          for (int c = 0; c < ROW / 8; ++c) {
            float v0[CH], v1[CH];
            unpack<T>(lds128(rv + c * 128), v0);
            unpack<T>(lds128(rv + S::kPitchV + c * 128), v1);
#pragma unroll
            for (int e = 0; e < CH; ++e) {
              uint32_t x0, y0, x1, y1;
              split_rounded(v0[e], x0, y0);
              split_rounded(v1[e], x1, y1);
#pragma unroll
              for (int mt = 0; mt < MTR; ++mt) {
                float t[4];
                mma_tf32<true>(t, a[mt], y0, y1);
                mma_tf32<false>(t, a[mt], x0, x1);
#pragma unroll
                for (int x = 0; x < 4; ++x) o[mt][c * CH + e][x] += t[x];
              }
            }
          }
        } else {
          uint4 a[MTR][S::kFrags];
#pragma unroll
          for (int mt = 0; mt < MTR; ++mt) {
            a[mt][0].x = take_term<T>(w[mt][0][0], w[mt][0][1]);
            a[mt][0].y = take_term<T>(w[mt][0][0], w[mt][0][1]);
            if constexpr (S::kBf16) {
              const uint32_t lo = take_term<T>(w[mt][0][0], w[mt][0][1]);
              if constexpr (PACKED) {
                if (grp >= 4) {
                  a[mt][0].x = lo;
                  a[mt][0].y = 0;
                }
              } else {
                a[mt][S::kFrags - 1].x = lo;
                a[mt][S::kFrags - 1].y = 0;
              }
            }
            if constexpr (NT == 2) {
              a[mt][0].z = take_term<T>(w[mt][NT - 1][0], w[mt][NT - 1][1]);
              a[mt][0].w = take_term<T>(w[mt][NT - 1][0], w[mt][NT - 1][1]);
              if constexpr (S::kBf16) {
                const uint32_t lo = take_term<T>(w[mt][NT - 1][0], w[mt][NT - 1][1]);
                if constexpr (PACKED) {
                  if (grp >= 4) {
                    a[mt][0].z = lo;
                    a[mt][0].w = 0;
                  }
                } else {
                  a[mt][S::kFrags - 1].z = lo;
                  a[mt][S::kFrags - 1].w = 0;
                }
              }
            }
          }
          // NT = 2: of 16 dimensions, positions 0-7 and 8-15 of the first eight,
          // then of the next; NT = 1: eight positions of 32 dimensions
          const uint32_t rv =
              NT == 2 ? vd + (lane & 15) * S::kPitchV + (lane >> 4) * 16
                      : vd + (lane & 7) * S::kPitchV + (lane >> 3) * 16;
          constexpr int TILES = NT == 2 ? 2 : 4;
#pragma unroll
          for (int c = 0; c < XT / TILES; ++c) {
            const uint4 v = ldmatrix4<true>(rv + c * TILES * 16);
            const uint32_t vb[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < TILES; ++x) {
#pragma unroll
              for (int mt = 0; mt < MTR; ++mt) {
                float t[4];
                if constexpr (NT == 2) {
                  mma_k16<T, true>(t, a[mt][S::kFrags - 1], vb[(2 * x) & 3], vb[(2 * x + 1) & 3]);
                  if constexpr (S::kFrags == 2) {
                    mma_k16<T, false>(t, a[mt][0], vb[(2 * x) & 3], vb[(2 * x + 1) & 3]);
                  }
                } else {
                  mma_k8<T, true>(t, a[mt][S::kFrags - 1], vb[x]);
                  if constexpr (S::kFrags == 2) mma_k8<T, false>(t, a[mt][0], vb[x]);
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) o[mt][c * TILES + x][y] += t[y];
              }
            }
          }
        }
        advance();
        const int page = next_page;
        next_page = page_of(filled + 1);
        fill(page);
      }
      // the ring is drained: every copy into it has been waited for
#pragma unroll
      for (int mt = 0; mt < MTR; ++mt) {
        l[mt] += __shfl_xor_sync(FULL, l[mt], 1);
        l[mt] += __shfl_xor_sync(FULL, l[mt], 2);
        const bool mine = !PACKED || grp < 4;
        if (thr == 0 && mine) {
          s_m[warp][mt * 8 + grp] = m[mt];
          s_l[warp][mt * 8 + grp] = l[mt];
        }
        float* row = part_of(warp) + (mt * 8 + grp) * PART;
#pragma unroll
        for (int x = 0; x < XT; ++x) {
          // the columns 2 thr and 2 thr + 1 of tile x
          const int d = sizeof(T) == 4 ? (8 * (x / CH) + 2 * thr) * CH + x % CH : 8 * x + 2 * thr;
          float o0 = o[mt][x][0] + o[mt][x][2], o1 = o[mt][x][1] + o[mt][x][3];
          if constexpr (PACKED) {
            o0 += __shfl_xor_sync(FULL, o0, 16);
            o1 += __shfl_xor_sync(FULL, o1, 16);
          }
          if (mine) {
            if constexpr (sizeof(T) == 4) {
              row[d] = o0;
              row[d + CH] = o1;
            } else {
              *reinterpret_cast<float2*>(row + d) = make_float2(o0, o1);
            }
          }
        }
      }
    }

    // ---- on to the next segment, whose copies are under way while the parts
    // of this one are joined
    const int d_r = r, d_count = count;
    const bool whole = real0 == 0 && t1 == count;
    const int real_from = real0;
    const long long u_unit = u - t0;  // the unit's first tile
    constexpr int kPartStep = MT == 0 ? DP : S::kWarpRing / 4;  // floats between warps' parts
    float* const parts = part_of(0);
    more = follow;
    if (follow) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      u += t1 - t0;
      t0 = 0;
      r = n_request;
      unit = n_unit;
      n = max(0, min(p.max_keys, s_length[warp]));
      count = tiles(n);
      slot = p.slots != nullptr ? s_slot[warp] : -1;
      filled = 0;
      more = begin();
      if (more) {
        next_page = page_of(EARLY);
#pragma unroll
        for (int i = 0; i < EARLY; ++i) fill(s_pages[warp][i][my_row]);
      }
    }

    // ---- the warps' parts into one
    const bool empty = __syncthreads_or(counted) == 0;
    if (tid < HEADS) {
      float top = -FLT_MAX, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w][tid]);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = exp2f(s_m[w][tid] - top);
        s_f[w][tid] = f;
        sum += s_l[w][tid] * f;
      }
      s_top[tid] = top;
      s_sum[tid] = sum;
      s_inverse[tid] = 1.f / sum;
    }
    __syncthreads();
    float* const out = p.out + d_r * p.o_s[0] + h0 * p.o_s[1];
    float* const lse =
        p.lse != nullptr ? p.lse + static_cast<int64_t>(d_r) * p.heads + h0 : nullptr;
    float* const part =
        sp.parts + ((2 * cta + (real_from == 0 ? 1 : 0)) * HEADS) * S::kRecord;
    for (int x = tid; x < heads * (DP / 4); x += THREADS) {
      const int h = x / (DP / 4), d = 4 * (x % (DP / 4));
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float4 o = *reinterpret_cast<const float4*>(parts + w * kPartStep + h * PART + d);
        const float f = s_f[w][h];
        acc.x = fmaf(o.x, f, acc.x);
        acc.y = fmaf(o.y, f, acc.y);
        acc.z = fmaf(o.z, f, acc.z);
        acc.w = fmaf(o.w, f, acc.w);
      }
      if (!whole) {
        *reinterpret_cast<float4*>(part + h * S::kRecord + d) = acc;
      } else if (d < p.dim) {  // a whole number of fours
        put_four(out + h * p.o_s[1] + d, acc, empty ? 0.f : s_inverse[h]);
      }
    }
    if (tid < heads) {
      if (!whole) {
        part[tid * S::kRecord + DP] = s_top[tid];
        part[tid * S::kRecord + DP + 1] = s_sum[tid];
        part[tid * S::kRecord + DP + 2] = empty ? 0.f : 1.f;
      } else if (lse != nullptr) {
        lse[tid] = empty ? -INFINITY : s_top[tid] * 0.69314718055994531f + logf(s_sum[tid]);
      }
    }
    if (!whole) {
      const long long c0 = divide((u_unit + kSetup + 1) * ctas - 1, total);
      const long long c1 = divide((u_unit + d_count) * ctas - 1, total);
      const int n_parts = static_cast<int>(c1 - c0) + 1;
      // part i of the unit: of CTA c0 its last segment, of the others their first
      auto record = [&](int i) -> float* {
        return sp.parts + ((2 * (c0 + i) + (i == 0 ? 1 : 0)) * HEADS) * S::kRecord;
      };
      // Whether this CTA is the last of `arrivals`.  One thread's fence, after
      // the barrier, orders the CTA's stores before the count, and the count
      // before the CTA's loads.
      auto last_of = [&](int* counter, int arrivals) -> bool {
        __syncthreads();
        if (tid == 0) {
          __threadfence();
          s_last = atomicAdd(counter, 1) == arrivals - 1 ? 1 : 0;
          __threadfence();
          if (s_last != 0) *counter = 0;  // nobody else arrives
        }
        __syncthreads();
        return s_last != 0;
      };
      // Joins `count` parts from part `from` on, every `every`th: into the
      // outputs, or into the first of them.
      auto join = [&](int from, int every, int count, bool into_outputs) {
        // maximum and sum of each head: thread t takes head t % HEADS of every
        // (THREADS / HEADS)th part
        auto merge = [](float& top, float& sum, float m, float l) {
          const float to = fmaxf(top, m);
          sum = sum * exp2f(top - to) + l * exp2f(m - to);
          top = to;
        };
        float top = -FLT_MAX, sum = 0.f, some = 0.f;
        if (tid % HEADS < heads) {
#pragma unroll 4
          for (int x = tid; x < count * HEADS; x += THREADS) {
            const float4 mls = __ldcg(reinterpret_cast<const float4*>(
                record(from + x / HEADS * every) + x % HEADS * S::kRecord + DP));
            merge(top, sum, mls.x, mls.y);
            some = fmaxf(some, mls.z);
          }
        }
#pragma unroll
        for (int x = HEADS; x < 32; x <<= 1) {
          const float m = __shfl_xor_sync(FULL, top, x), l = __shfl_xor_sync(FULL, sum, x);
          merge(top, sum, m, l);
        }
        if (lane < HEADS) {
          s_m[warp][lane] = top;
          s_l[warp][lane] = sum;
        }
        const bool none = __syncthreads_or(some != 0.f) == 0;
        if (tid < heads) {
          top = s_m[0][tid];
          sum = s_l[0][tid];
#pragma unroll
          for (int w = 1; w < WARPS; ++w) merge(top, sum, s_m[w][tid], s_l[w][tid]);
          s_top[tid] = top;
          s_sum[tid] = sum;
          s_inverse[tid] = none ? 0.f : 1.f / sum;
          if (into_outputs && lse != nullptr) {
            lse[tid] = none ? -INFINITY : top * 0.69314718055994531f + logf(sum);
          }
        }
        __syncthreads();
        // LANES lanes read a part's outputs, 16 bytes each and VECS of them;
        // the GROUPS of lanes take the parts in turn, and leave their sums where
        // the warps' parts were
        constexpr int QUADS = HEADS * DP / 4, LANES = QUADS < 32 ? QUADS : 32;
        constexpr int VECS = QUADS / LANES, GROUPS = THREADS / LANES;
        static_assert(GROUPS == WARPS || (MT == 0 && GROUPS * DP * 4 <= S::kPartBytes),
                      "room for the groups' sums");
        const int group = tid / LANES, quad = tid % LANES;
        auto sums_of = [&](int y) -> float* { return parts + y * kPartStep; };
        float acc[VECS][4];
#pragma unroll
        for (int v = 0; v < VECS; ++v) acc[v][0] = acc[v][1] = acc[v][2] = acc[v][3] = 0.f;
#pragma unroll 2
        for (int i = group; i < count; i += GROUPS) {
          const float* rec = record(from + i * every);
#pragma unroll
          for (int v = 0; v < VECS; ++v) {
            const int x = (v * LANES + quad) * 4, h = x / DP;
            if (h < heads) {
              const float4 o = __ldcg(reinterpret_cast<const float4*>(rec + x + h * 4));
              const float f = exp2f(__ldcg(rec + h * S::kRecord + DP) - s_top[h]);
              acc[v][0] = fmaf(o.x, f, acc[v][0]);
              acc[v][1] = fmaf(o.y, f, acc[v][1]);
              acc[v][2] = fmaf(o.z, f, acc[v][2]);
              acc[v][3] = fmaf(o.w, f, acc[v][3]);
            }
          }
        }
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
          *reinterpret_cast<float4*>(sums_of(group) + (v * LANES + quad) * 4) =
              make_float4(acc[v][0], acc[v][1], acc[v][2], acc[v][3]);
        }
        __syncthreads();
        float* const into = record(from);
        for (int x = tid; x < heads * (DP / 4); x += THREADS) {
          const int h = x / (DP / 4), d = 4 * (x % (DP / 4));
          float4 sums = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int y = 0; y < GROUPS; ++y) {
            const float4 o = *reinterpret_cast<const float4*>(sums_of(y) + h * DP + d);
            sums.x += o.x;
            sums.y += o.y;
            sums.z += o.z;
            sums.w += o.w;
          }
          if (!into_outputs) {
            *reinterpret_cast<float4*>(into + h * S::kRecord + d) = sums;
          } else if (d < p.dim) {
            put_four(out + h * p.o_s[1] + d, sums, s_inverse[h]);
          }
        }
        if (!into_outputs && tid < heads) {
          *reinterpret_cast<float4*>(into + tid * S::kRecord + DP) =
              make_float4(s_top[tid], s_sum[tid], none ? 0.f : 1.f, 0.f);
        }
      };
      if (n_parts <= kJoinAtOnce) {
        if (last_of(sp.counters + c0, n_parts)) join(0, 1, n_parts, true);
      } else {
        // many parts: the last CTA of each kJoinGroup joins theirs, the last of
        // these what they made of them
        const int mine = static_cast<int>(cta - c0), begin_at = mine / kJoinGroup * kJoinGroup;
        const int members = min(kJoinGroup, n_parts - begin_at);
        const int groups = (n_parts + kJoinGroup - 1) / kJoinGroup;
        // counters of the first group and of a later one, which may begin with
        // the last part of this unit where the next unit's first group does
        int* const counter =
            sp.counters + (begin_at == 0 ? kMaxCtas + c0 : 2 * kMaxCtas + c0 + begin_at);
        if (last_of(counter, members)) {
          join(begin_at, 1, members, false);
          if (last_of(sp.counters + c0, groups)) join(0, kJoinGroup, groups, true);
        }
      }
    }
    __syncthreads();  // the shared parts are free for the next segment
  }
}

struct StreamPlan {
  int dp = 0;     // padded head dimension
  int mt = 0;     // row blocks
  int heads = 1;  // query heads of a unit
  int subs = 1;   // units of a key head
};

// More than 8 heads on a key head make units of 16 (MT = 2, for which 256
// dimensions leave no registers), so that keys and values are read once; but
// where most units are cut into parts, units of 8: a part costs by its heads, and
// the second unit's reads come from L2.  Equal at 64 (request, key head) pairs:
// 16 heads of 128 a key head, f16, 1000 to 8000 keys, 16 pairs 34.5 us with 16
// and 26.5 us with 8, 64 pairs 41 and 41 us, 128 pairs 61 and 74 us.  The lengths
// are not known here; short requests are cut less and lose by it: 80 pairs of 100
// to 1000 keys, fp32, 26.7 us with 16 and 24.9 us with 8 (64 dimensions 19.7 and
// 17.0), f16 of 64 dimensions 13.2 and 12.5.
constexpr int64_t kWidePairs = 64;

StreamPlan stream_plan(int page_type, int64_t pairs, int64_t group, int64_t dim) {
  StreamPlan s;
  s.dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  s.mt = group == 1 ? 0 : group <= 8 || s.dp == 256 || pairs < kWidePairs ? 1 : 2;
  s.heads = s.mt == 0 ? 1 : page_type == TVR_PAGE_BF16 && group <= 4 ? 4 : 8 * s.mt;
  s.subs = static_cast<int>(ceil_div(group, s.heads));
  return s;
}

int64_t workspace_bytes_of(int heads, int dp) {
  return kCounterBytes + 4ll * 2 * kMaxCtas * heads * (dp + 4);
}

template <typename T, int DP, int MT, bool PACKED>
int launch_stream(const StreamParams& sp, cudaStream_t stream) {
  using S = Stream<T, DP, MT, PACKED>;
  auto kernel = paged_attention_stream_kernel<T, DP, MT, PACKED>;
  const int dev = current_device();
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  std::call_once(once[dev & 63], [&]() {
    attr_err[dev & 63] =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  });
  TVR_CUDA_TRY(attr_err[dev & 63]);
  const int ctas = S::kCtasPerSm * std::min(kMaxCtas / 4, sm_count(dev));
  kernel<<<ctas, S::kThreads, S::kSmem, stream>>>(sp);
  TVR_LAUNCH_CHECK();
  return TVR_OK;
}

template <typename T, int DP>
int launch_stream(const StreamPlan& s, const StreamParams& sp, cudaStream_t stream) {
  if (s.mt == 0) return launch_stream<T, DP, 0, false>(sp, stream);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    if (s.heads == 4) return launch_stream<T, DP, 1, true>(sp, stream);
  }
  if constexpr (DP < 256) {
    if (s.mt == 2) return launch_stream<T, DP, 2, false>(sp, stream);
  }
  return launch_stream<T, DP, 1, false>(sp, stream);
}

template <typename T>
int launch_stream(const StreamPlan& s, const StreamParams& sp, cudaStream_t stream) {
  if (s.dp == 64) return launch_stream<T, 64>(s, sp, stream);
  if (s.dp == 128) return launch_stream<T, 128>(s, sp, stream);
  return launch_stream<T, 256>(s, sp, stream);
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
  TVR_CHECK(kv_heads == 0 || heads % kv_heads == 0,
            "paged_attention_workspace: heads do not share the key heads evenly");
  *bytes = 0;
  if (heads > 0 && kv_heads > 0 && head_dim > 0 && head_dim <= paged::kMaxDim) {
    // whatever the pages' type and the requests: the largest units
    const paged::StreamPlan s =
        paged::stream_plan(TVR_PAGE_F32, paged::kWidePairs, heads / kv_heads, head_dim);
    *bytes = paged::workspace_bytes_of(s.heads, s.dp);
  }
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
  TVR_CHECK(max_pages <= 0x7ffff000 / cache->page_size && requests * heads <= 0x7fffffff &&
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
  const cudaStream_t s = as_stream(stream);
  // The streaming form moves 16-byte chunks: rows a whole number of them, on
  // 16-byte boundaries.
  const int64_t chunk = 16 / type_size(cache->page_type);
  auto aligned = [](const void* base, const int64_t* st, int n_strides, int64_t unit) {
    bool ok = (reinterpret_cast<uintptr_t>(base) & 15u) == 0;
    for (int i = 0; i < n_strides; ++i) ok = ok && st[i] % unit == 0;
    return ok;
  };
  if (dim % chunk == 0 && aligned(p.k, p.k_s, 3, chunk) && aligned(p.v, p.v_s, 3, chunk)) {
    StreamParams sp = {};
    sp.a = p;
    sp.requests = static_cast<int>(requests);
    sp.key_heads = static_cast<int>(cache->kv_heads);
    const StreamPlan plan =
        stream_plan(cache->page_type, requests * cache->kv_heads, p.group, dim);
    const int64_t need = workspace_bytes_of(plan.heads, plan.dp);
    sp.subs = plan.subs;
    TVR_CHECK(workspace != nullptr && workspace_bytes >= need,
              "paged_attention: a workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
              (long long)need);
    TVR_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0,
              "paged_attention: the workspace is not 16-byte aligned");
    sp.counters = static_cast<int*>(workspace);
    sp.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    switch (cache->page_type) {
      case TVR_PAGE_F32: return launch_stream<float>(plan, sp, s);
      case TVR_PAGE_F16: return launch_stream<__half>(plan, sp, s);
      default: return launch_stream<__nv_bfloat16>(plan, sp, s);
    }
  }
  const unsigned grid = static_cast<unsigned>(requests * heads);
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
