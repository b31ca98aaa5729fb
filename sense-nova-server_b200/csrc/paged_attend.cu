// Attention over the paged cache (snl_paged_attend) and the accumulated attention weights
// of its slots (snl_paged_weigh).
#include <algorithm>
#include <string>

#include "paged.cuh"

namespace snl {
namespace {

struct AttendArgs {
  PagedView c;
  PagedMask m;
  snl_paged_attn_p p;
  const uint16_t* q;
  const void* gate;
  void* out;
  float* lse;
  const float* lse_in;
  float decay;
};

constexpr float kLog2e = 1.4426950408889634f;

// Score in units of log2 from the raw product: cap, then the distance bias.
__device__ __forceinline__ float paged_score(const PagedMask& m, float qk, float slope, int32_t t, int32_t key) {
  float s = qk * m.scale;
  if (m.cap > 0.f) s = m.cap * tanhf(s / m.cap);
  return (s - slope * fabsf((float)(t - key))) * kLog2e;
}

constexpr uint32_t kWarps = 8;

// One warp per (row, head), one key at a time.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) attend_simple_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t item = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const uint32_t r = (uint32_t)(item / a.p.n_heads), h = (uint32_t)(item % a.p.n_heads);
  if (r >= a.c.n_rows) return;
  const uint32_t type = std::is_same<T, __half>::value ? SNL_T_F16 : SNL_T_BF16;
  const uint32_t kh = h / (a.p.n_heads / a.c.n_kv);
  const uint32_t b = paged_seq(a.c, r, lane);
  const int2 rr = paged_rows(a.c, b);
  const int32_t len = paged_len(a.c, b), t = len - (rr.y - (int32_t)r);
  const int2 keys = (int32_t)r < rr.x || (int32_t)r >= rr.y ? make_int2(0, 0) : paged_keys(a.m, r, t, len);
  const float slope = a.m.slopes ? __ldg(a.m.slopes + h) : 0.f;
  float q[E], o[E];
  load_as_float<E>(a.q, r * a.p.q_row + h * a.p.q_head + lane * E, type, q);
#pragma unroll
  for (int i = 0; i < E; i++) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int32_t key = keys.x; key < keys.y; key++) {
    const int32_t page = paged_page(a.c, b, key);
    if (page < 0) continue;
    float x[E], s = 0.f;
    load_as_float<E>(a.c.k, paged_at(a.c, page, kh, key) + lane * E, type, x);
#pragma unroll
    for (int i = 0; i < E; i++) s = fmaf(q[i], x[i], s);
    s = paged_score(a.m, warp_sum(s), slope, t, key);
    const float top = fmaxf(m, s);
    if (m == -INFINITY && s == -INFINITY) continue;
    const float old = exp2f(m - top), p = exp2f(s - top);
    m = top;
    l = fmaf(l, old, p);
    load_as_float<E>(a.c.v, paged_at(a.c, page, kh, key) + lane * E, type, x);
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = fmaf(o[i], old, p * x[i]);
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  float g[E];
  if (a.gate) load_as_float<E>(a.gate, r * a.p.gate_row + h * a.p.gate_head + lane * E, a.p.gate_type, g);
#pragma unroll
  for (int i = 0; i < E; i++) o[i] *= a.gate ? inv * sigmoidf_(g[i]) : inv;
  store_from_float<E>(a.out, r * a.p.out_row + h * a.p.out_head + lane * E, a.p.out_type, o);
  if (a.lse && lane == 0)
    a.lse[(uint64_t)r * a.p.n_heads + h] = l > 0.f || l != l ? (m + log2f(l)) / kLog2e : -INFINITY;
}

// One warp per (slot, KV head, sequence), one row and head at a time.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) weigh_simple_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const uint32_t type = std::is_same<T, __half>::value ? SNL_T_F16 : SNL_T_BF16;
  const uint32_t lane = threadIdx.x & 31, kh = blockIdx.y, b = blockIdx.z;
  const int32_t key = (int32_t)(blockIdx.x * kWarps + (threadIdx.x >> 5)), len = paged_len(a.c, b);
  if (key >= len) return;
  const int32_t page = paged_page(a.c, b, key);
  if (page < 0) return;
  const int2 rr = paged_rows(a.c, b);
  const uint32_t group = a.p.n_heads / a.c.n_kv;
  float x[E], sum = 0.f;
  load_as_float<E>(a.c.k, paged_at(a.c, page, kh, key) + lane * E, type, x);
  for (int32_t r = rr.x; r < rr.y; r++) {
    const int32_t t = len - (rr.y - r);
    const int2 keys = paged_keys(a.m, r, t, len);
    if (key < keys.x || key >= keys.y) continue;
    for (uint32_t g = 0; g < group; g++) {
      const uint32_t h = kh * group + g;
      float q[E], s = 0.f;
      load_as_float<E>(a.q, r * a.p.q_row + h * a.p.q_head + lane * E, type, q);
#pragma unroll
      for (int i = 0; i < E; i++) s = fmaf(q[i], x[i], s);
      s = paged_score(a.m, warp_sum(s), a.m.slopes ? __ldg(a.m.slopes + h) : 0.f, t, key);
      sum += exp2f(s - a.lse_in[(uint64_t)r * a.p.n_heads + h] * kLog2e);
    }
  }
  if (lane == 0) {
    float* w = a.c.weight + paged_weight_at(a.c, page, kh, key);
    const bool old = a.decay != 0.f && key < len - (rr.y - rr.x);
    *w = old ? fmaf(*w, a.decay, sum) : sum;
  }
}

}  // namespace
}  // namespace snl

using namespace snl;

#define SNL_BY_TYPE(kern, what, grid, block, smem, s, ...)                                                     \
  do {                                                                                                         \
    if (c->type == SNL_T_F16 && c->head_dim == 256)                                                            \
      SNL_PDL_LAUNCH(what, (kern<__half, 256>), grid, block, smem, s, __VA_ARGS__);                            \
    else if (c->type == SNL_T_F16)                                                                             \
      SNL_PDL_LAUNCH(what, (kern<__half, 128>), grid, block, smem, s, __VA_ARGS__);                            \
    else if (c->head_dim == 256)                                                                               \
      SNL_PDL_LAUNCH(what, (kern<__nv_bfloat16, 256>), grid, block, smem, s, __VA_ARGS__);                     \
    else                                                                                                       \
      SNL_PDL_LAUNCH(what, (kern<__nv_bfloat16, 128>), grid, block, smem, s, __VA_ARGS__);                     \
  } while (0)

extern "C" size_t snl_paged_attend_workspace(const snl_paged_cache* c, const snl_paged_batch* b, uint32_t n_heads) {
  return c && b && n_heads ? 16 : 0;
}

extern "C" int snl_paged_attend(const snl_paged_cache* c, const snl_paged_batch* b, const snl_paged_attn_p* p,
                                const void* q, const void* gate, void* out, float* lse, void* work, size_t work_bytes,
                                void* stream) {
  const std::string w = "snl_paged_attend";
  AttendArgs a{};
  SNL_TRY(paged_check("snl_paged_attend", c, b, &a.c));
  if (!p || (b->n_rows && (!q || !out))) return fail(SNL_E_INVALID, w + ": null argument");
  SNL_TRY(paged_check_attn("snl_paged_attend", *c, *b, p, &a.m));
  if (p->out_type > SNL_T_BF16 || (gate && p->gate_type > SNL_T_BF16)) return fail(SNL_E_INVALID, w + ": unknown type");
  if (!paged_aligned(q) || !paged_aligned(gate) || !paged_aligned(out) || !paged_aligned(work) ||
      !paged_strides(p->out_type, p->out_row, p->out_head) ||
      (gate && !paged_strides(p->gate_type, p->gate_row, p->gate_head)))
    return fail(SNL_E_INVALID, w + ": rows must be aligned to 16 bytes");
  if (work_bytes < snl_paged_attend_workspace(c, b, p->n_heads)) return fail(SNL_E_INVALID, w + ": work is too small");
  if (!work) return fail(SNL_E_INVALID, w + ": null argument");
  if (b->n_rows == 0 || b->n_seqs == 0) return SNL_OK;
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.gate = gate;
  a.out = out;
  a.lse = lse;
  SNL_TRY(paged_error_word(&a.c.err));
  const uint64_t items = (uint64_t)b->n_rows * p->n_heads;
  if (items > (1ull << 33)) return fail(SNL_E_UNSUPPORTED, w + ": too many rows");
  SNL_BY_TYPE(attend_simple_kernel, "attend_simple_kernel", dim3((unsigned)((items + kWarps - 1) / kWarps)),
              dim3(kWarps * 32), (size_t)0, (cudaStream_t)stream, a);
  return SNL_OK;
}

extern "C" int snl_paged_weigh(const snl_paged_cache* c, const snl_paged_batch* b, const snl_paged_attn_p* p,
                               const void* q, const float* lse, float decay, void* stream) {
  const std::string w = "snl_paged_weigh";
  AttendArgs a{};
  SNL_TRY(paged_check("snl_paged_weigh", c, b, &a.c));
  if (b->n_rows && (!q || !lse)) return fail(SNL_E_INVALID, w + ": null argument");
  SNL_TRY(paged_check_attn("snl_paged_weigh", *c, *b, p, &a.m));
  if (!c->weight) return fail(SNL_E_INVALID, w + ": the cache has no weights");
  if (!(decay >= 0.f) || decay > 3e38f) return fail(SNL_E_INVALID, w + ": decay must be finite and not negative");
  if (!paged_aligned(q)) return fail(SNL_E_INVALID, w + ": q rows must be aligned to 16 bytes");
  if (b->n_seqs == 0 || a.c.max_len == 0) return SNL_OK;
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.lse_in = lse;
  SNL_TRY(paged_error_word(&a.c.err));
  a.decay = decay;
  SNL_BY_TYPE(weigh_simple_kernel, "weigh_simple_kernel",
              dim3((unsigned)((a.c.max_len + kWarps - 1) / kWarps), c->n_kv, b->n_seqs), dim3(kWarps * 32), (size_t)0,
              (cudaStream_t)stream, a);
  return SNL_OK;
}
