// What the paged-cache kernels share: the cache and batch as the device sees them, bounds
// on what only the device can read, and the interval of keys that a row sees.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "ptx.cuh"

namespace snl {

constexpr int kPagedBadIndex = 4;  // bit 2 of the error word

struct PagedView {
  uint16_t* k;
  uint16_t* v;
  float* weight;
  uint64_t ps, hs, ss;  // strides of page, head, slot in elements
  const int32_t* table;
  const int32_t* start;
  const int32_t* len;
  uint32_t n_pages, shift, n_kv, n_seqs, n_rows, table_stride;
  int32_t max_len;  // min(max_len, slots of table_stride pages)
  int* err;
};

__device__ __forceinline__ void report_index(int* err) { atomicOr(err, kPagedBadIndex); }

// Length of sequence b, in [0, max_len]; n is what the batch says.
__device__ __forceinline__ int32_t paged_length(const PagedView& c, int32_t n) {
  if (n >= 0 && n <= c.max_len) return n;
  report_index(c.err);
  return n < 0 ? 0 : c.max_len;
}
__device__ __forceinline__ int32_t paged_len(const PagedView& c, uint32_t b) { return paged_length(c, __ldg(c.len + b)); }

// Page of slot t (t in [0, max_len)) of sequence b, or -1 for a number outside the cache.
__device__ __forceinline__ int32_t paged_page(const PagedView& c, uint32_t b, uint32_t t) {
  const int32_t p = __ldg(c.table + (uint64_t)b * c.table_stride + (t >> c.shift));
  if (p >= 0 && p < (int32_t)c.n_pages) return p;
  report_index(c.err);
  return -1;
}
__device__ __forceinline__ uint64_t paged_at(const PagedView& c, int32_t page, uint32_t head, uint32_t t) {
  return (uint64_t)page * c.ps + (uint64_t)head * c.hs + (uint64_t)(t & ((1u << c.shift) - 1)) * c.ss;
}
__device__ __forceinline__ uint64_t paged_weight_at(const PagedView& c, int32_t page, uint32_t head, uint32_t t) {
  return (((uint64_t)page * c.n_kv + head) << c.shift) + (t & ((1u << c.shift) - 1));
}

// Rows [r0, r1) of a sequence, within [0, n_rows].
__device__ __forceinline__ int2 paged_rows(const PagedView& c, int32_t r0, int32_t r1) {
  if (r0 < 0 || r1 < r0 || r1 > (int32_t)c.n_rows) {
    report_index(c.err);
    return make_int2(0, 0);
  }
  return make_int2(r0, r1);
}
__device__ __forceinline__ int2 paged_rows(const PagedView& c, uint32_t b) {
  return paged_rows(c, __ldg(c.start + b), __ldg(c.start + b + 1));
}

// The sequence that owns row r: the last b with start[b] <= r. All lanes of the warp call
// it with the same r; each step looks at 32 boundaries at once.
__device__ __forceinline__ uint32_t paged_seq(const PagedView& c, uint32_t r, uint32_t lane) {
  uint32_t lo = 0, hi = c.n_seqs;  // start[lo] <= r; the answer is in [lo, hi)
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + 31) / 32;
    const uint32_t at = lo + lane * step;
    const bool le = at < hi && (at == lo || (uint32_t)__ldg(c.start + at) <= r);
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, le));  // a prefix of the lanes: start does not fall
    const uint32_t below = lo + (max(n, 1u) - 1) * step;
    hi = min(hi, below + step);
    lo = below;
  }
  return lo;
}

// The masks of attend and weigh, and the interval [x, y) of keys that row r at slot t sees.
struct PagedMask {
  const float* slopes;
  const int32_t* first;
  const int32_t* last;
  int32_t window;  // 0: none
  float scale, cap;
};
__device__ __forceinline__ int2 paged_interval(const PagedMask& m, int32_t first, int32_t last, int32_t t, int32_t len) {
  int32_t lo = first;
  if (m.window) lo = max(lo, t + 1 - m.window);
  lo = max(lo, 0);
  int32_t hi = t + 1;
  if (m.last) hi = max(hi, last);
  hi = min(hi, len);
  return t >= 0 && lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
}
__device__ __forceinline__ int2 paged_keys(const PagedMask& m, uint32_t r, int32_t t, int32_t len) {
  return paged_interval(m, m.first ? __ldg(m.first + r) : 0, m.last ? __ldg(m.last + r) : 0, t, len);
}

template <typename T>
struct Half2Of;
template <>
struct Half2Of<__half> {
  using type = __half2;
};
template <>
struct Half2Of<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// N contiguous elements (N = 4 or 8) of type SNL_T_* at element offset `at`, as floats.
template <int N>
__device__ __forceinline__ void load_as_float(const void* p, uint64_t at, uint32_t type, float* v) {
  if (type == SNL_T_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + i);
      v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
    return;
  }
  uint32_t w[N / 2];
  const uint16_t* s = static_cast<const uint16_t*>(p) + at;
  if constexpr (N == 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(s);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(s);
    w[0] = x.x, w[1] = x.y;
  }
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    const float2 f = type == SNL_T_F16 ? unpack2(w[i], __half()) : unpack2(w[i], __nv_bfloat16());
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
template <int N>
__device__ __forceinline__ void store_from_float(void* p, uint64_t at, uint32_t type, const float* v) {
  if (type == SNL_T_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(static_cast<float*>(p) + at + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    return;
  }
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; i++)
    w[i] = type == SNL_T_F16 ? pack2(v[2 * i], v[2 * i + 1], __half()) : pack2(v[2 * i], v[2 * i + 1], __nv_bfloat16());
  uint16_t* d = static_cast<uint16_t*>(p) + at;
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
  else
    *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
}

// Host side: the checks that every call makes.
int paged_check(const char* what, const snl_paged_cache* c, const snl_paged_batch* b, PagedView* v);
int paged_check_attn(const char* what, const snl_paged_cache& c, const snl_paged_batch& b, const snl_paged_attn_p* p,
                     PagedMask* m);
inline bool paged_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Strides of rows and heads of a tensor of `type`: multiples of 16 bytes.
inline bool paged_strides(uint32_t type, uint64_t row, uint64_t head) {
  const uint64_t m = type == SNL_T_F32 ? 4 : 8;
  return row % m == 0 && head % m == 0;
}
// Rows or heads of an output that would be written over one another (an expanded view's).
inline bool paged_overlap(uint64_t n, uint64_t stride, uint32_t head_dim) { return n > 1 && stride < head_dim; }

}  // namespace snl
