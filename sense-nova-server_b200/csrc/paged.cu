// The paged key/value cache: rotary table, append, evict, and the checks of every call.
// attend and weigh are in paged_attend.cu.
#include <algorithm>
#include <string>

#include "paged.cuh"

namespace snl {
namespace {

// ---- rotary table ------------------------------------------------------------------------

// Angles in 64 bits: at position 2^18 a 32-bit product pos * inv_freq is off by 0.01.
__global__ void rope_table_kernel(double theta, uint32_t rot, uint32_t n_pos, float2* __restrict__ out) {
  const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t half = rot / 2;
  if (i >= (uint64_t)n_pos * half) return;
  const double a = (double)(i / half) * pow(theta, -2.0 * (double)(i % half) / (double)rot);
  double s, c;
  sincos(a, &s, &c);
  out[i] = make_float2((float)c, (float)s);
}

// ---- append ------------------------------------------------------------------------------

struct AppendArgs {
  PagedView c;
  snl_paged_append_p p;
  const void* q;
  const void* k;
  const void* v;
  const float* q_norm;
  const float* k_norm;
  const uint4* pos;
  const float2* rope;
  uint16_t* q_out;
  uint32_t cache_type;
};

constexpr uint32_t kAppendWarps = 8;

// One warp per (row, head): queries, then keys, then values. A lane holds D / 32
// neighbouring elements; the turn reads its partner element from the warp's row in shared
// memory, so any even rot_dim and either pairing work.
template <int D>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int E = D / 32;
  __shared__ __align__(16) float rows[kAppendWarps][D];
  pdl_trigger();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t heads = a.p.n_heads + 2 * a.c.n_kv;
  const uint64_t item = (uint64_t)blockIdx.x * kAppendWarps + warp;
  const uint32_t r = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
  pdl_wait();
  if (r >= a.c.n_rows) return;
  const bool is_q = h < a.p.n_heads, is_k = !is_q && h < a.p.n_heads + a.c.n_kv;
  const uint32_t kh = is_k ? h - a.p.n_heads : h - a.p.n_heads - a.c.n_kv;
  float x[E];
  if (is_q) load_as_float<E>(a.q, r * a.p.q_row + h * a.p.q_head + lane * E, a.p.in_type, x);
  else if (is_k) load_as_float<E>(a.k, r * a.p.k_row + kh * a.p.k_head + lane * E, a.p.in_type, x);
  else load_as_float<E>(a.v, r * a.p.v_row + kh * a.p.v_head + lane * E, a.p.in_type, x);

  uint16_t* dst = a.q_out + r * a.p.out_row + h * a.p.out_head;
  if (!is_q) {
    const uint32_t b = paged_seq(a.c, r, lane);
    const int2 rr = paged_rows(a.c, b);
    const int32_t len = paged_len(a.c, b), t = len - (rr.y - (int32_t)r);
    if ((int32_t)r < rr.x || (int32_t)r >= rr.y || t < 0 || t >= len) {
      if (lane == 0) report_index(a.c.err);
      return;
    }
    const int32_t page = paged_page(a.c, b, t);
    if (page < 0) return;
    dst = (is_k ? a.c.k : a.c.v) + paged_at(a.c, page, kh, t);
  }
  if (is_q || is_k) {
    const float* norm = is_q ? a.q_norm : a.k_norm;
    if (norm) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; i++) s = fmaf(x[i], x[i], s);
      const float inv = rsqrtf(warp_sum(s) / (float)D + a.p.eps);
      float w[E];
      load_as_float<E>(norm, lane * E, SNL_T_F32, w);
#pragma unroll
      for (int i = 0; i < E; i++) x[i] = x[i] * inv * (1.0f + w[i]);
    }
    if (a.p.rot_dim) {
#pragma unroll
      for (int i = 0; i < E; i += 4)
        *reinterpret_cast<float4*>(&rows[warp][lane * E + i]) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      __syncwarp();
      const uint4 pos = __ldg(a.pos + r);
      const uint32_t half = a.p.rot_dim / 2;
#pragma unroll
      for (int i = 0; i < E; i++) {
        const uint32_t e = lane * E + i;
        if (e >= a.p.rot_dim) continue;
        const bool adj = a.p.pairs == SNL_ROPE_ADJACENT;
        const uint32_t f = adj ? e / 2 : e % half;
        const bool second = adj ? (e & 1) : e >= half;
        const uint32_t other = adj ? (e ^ 1) : second ? e - half : e + half;
        uint32_t at = pos.x;
        if (a.p.axes == SNL_ROPE_SECTIONS)
          at = f < a.p.sections[0] ? pos.x : f < a.p.sections[0] + a.p.sections[1] ? pos.y : pos.z;
        else if (a.p.axes == SNL_ROPE_INTERLEAVED)
          at = f % 3 == 1 && f < 3 * a.p.sections[1] ? pos.y : f % 3 == 2 && f < 3 * a.p.sections[2] ? pos.z : pos.x;
        if (at >= a.p.n_pos) {
          report_index(a.c.err);
          at = 0;
        }
        const float2 cs = __ldg(a.rope + (uint64_t)at * half + f);
        const float o = rows[warp][other];
        x[i] = second ? fmaf(x[i], cs.x, o * cs.y) : fmaf(x[i], cs.x, -o * cs.y);
      }
    }
  }
  store_from_float<E>(dst, lane * E, a.cache_type, x);
}

// ---- evict -------------------------------------------------------------------------------

struct EvictArgs {
  PagedView c;
  snl_paged_evict_p p;
  int32_t* kept;
  const int32_t* into;
  int32_t* new_len;
  uint32_t head_dim;
};

// Order-preserving map of a weight to an unsigned key: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr uint32_t kSelectThreads = 1024;

// One CTA per (KV head, sequence): the n-th largest key of the candidates by four 8-bit
// radix passes, then the kept slots in slot order.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ uint32_t hist[256], warp_n[32], s_prefix, s_need;
  pdl_trigger();
  pdl_wait();
  const uint32_t kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t len = paged_len(a.c, b), budget = (int32_t)a.p.budget;
  int32_t* kept = a.kept + ((uint64_t)b * a.c.n_kv + kh) * a.p.budget;
  if (len <= budget) {
    for (int32_t i = tid; i < budget; i += kSelectThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int32_t t0 = (int32_t)a.p.sink, t1 = len - (int32_t)a.p.recent;  // the candidates
  auto key_of = [&](int32_t t) -> uint32_t {
    const int32_t page = paged_page(a.c, b, t);
    return page < 0 ? 0u : weight_key(a.c.weight[paged_weight_at(a.c, page, kh, t)]);
  };
  if (tid == 0) {
    s_prefix = 0;
    s_need = a.p.budget - a.p.sink - a.p.recent;
  }
  __syncthreads();
  const bool any = s_need != 0;
  for (int shift = 24; any && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    for (int32_t t = t0 + tid; t < t1; t += kSelectThreads) {
      const uint32_t key = key_of(t);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t need = s_need, d = 255;
      while (d > 0 && hist[d] < need) need -= hist[d--];
      s_need = need;  // of those that share the prefix so far
      s_prefix = prefix | (d << shift);
    }
    __syncthreads();
  }
  const uint32_t cut = s_prefix;
  uint32_t ties = any ? s_need : 0, n = 0;  // ties still to take; kept so far
  for (int32_t base = 0; base < len; base += kSelectThreads) {
    const int32_t t = base + tid;
    const bool must = t < len && (t < t0 || t >= t1), cand = t < len && !must;
    const uint32_t key = cand && any ? key_of(t) : 0u;
    const bool tie = cand && any && key == cut;
    uint32_t ahead = __popc(__ballot_sync(0xffffffffu, tie) & ((1u << lane) - 1));
    if (lane == 0) warp_n[warp] = 0;
    const uint32_t wt = __popc(__ballot_sync(0xffffffffu, tie));
    __syncwarp();
    if (lane == 0) warp_n[warp] = wt;
    __syncthreads();
    uint32_t all = 0;
    for (uint32_t w = 0; w < 32; w++) {
      if (w < warp) ahead += warp_n[w];
      all += warp_n[w];
    }
    const bool keep = must || (cand && any && key > cut) || (tie && ahead < ties);
    ties -= min(ties, all);
    __syncthreads();
    const uint32_t bal = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_n[warp] = __popc(bal);
    __syncthreads();
    uint32_t at = n + __popc(bal & ((1u << lane) - 1));
    for (uint32_t w = 0; w < 32; w++) {
      if (w < warp) at += warp_n[w];
      n += warp_n[w];
    }
    if (keep && at < a.p.budget) kept[at] = t;
    __syncthreads();
  }
}

constexpr uint32_t kMoveThreads = 256, kMoveRows = 8 * 32;  // rows of one step: 8 per group of 8 threads

// Moves kept slots to their new places. A CTA takes 128 bytes of every row (8 threads to a
// row) of k or v, or the weights; in place it walks the rows in order, so that a place is
// overwritten only after its slot was read: kept slots never move up. With new pages the
// steps are independent and blockIdx.z counts them too.
template <bool IN_PLACE>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs a,
                                                                  uint32_t steps) {
  pdl_trigger();
  pdl_wait();
  const uint32_t slices = a.head_dim * 2 / 128;  // of k, then as many of v, then the weights
  const uint32_t slice = blockIdx.x, kh = blockIdx.y, b = blockIdx.z / steps, step0 = blockIdx.z % steps;
  const uint32_t tid = threadIdx.x;
  const int32_t* kept = a.kept + ((uint64_t)b * a.c.n_kv + kh) * a.p.budget;
  if (slice == 2 * slices && kh == 0 && step0 == 0 && tid == 0) a.new_len[b] = min(paged_len(a.c, b), (int32_t)a.p.budget);
  const int32_t* to = IN_PLACE ? a.c.table + (uint64_t)b * a.c.table_stride : a.into + (uint64_t)b * a.p.into_stride;
  auto place = [&](uint32_t i) -> int32_t {
    const int32_t p = __ldg(to + (i >> a.c.shift));
    if (p >= 0 && p < (int32_t)a.c.n_pages) return p;
    report_index(a.c.err);
    return -1;
  };
  for (uint32_t r0 = step0 * kMoveRows; r0 < a.p.budget; r0 += steps * kMoveRows) {
    if (kept[r0] < 0) break;  // the same for the whole CTA: nothing is kept from here on
    if (slice == 2 * slices) {
      const uint32_t i = r0 + tid;
      const int32_t t = i < a.p.budget ? kept[i] : -1;
      const int32_t from = t >= 0 ? paged_page(a.c, b, t) : -1, dst = t >= 0 ? place(i) : -1;
      const bool ok = from >= 0 && dst >= 0;
      float w = 0.f;
      if (ok) w = a.c.weight[paged_weight_at(a.c, from, kh, t)];
      if (IN_PLACE) __syncthreads();
      if (ok) a.c.weight[paged_weight_at(a.c, dst, kh, i)] = w;
      if (IN_PLACE) __syncthreads();
      continue;
    }
    uint16_t* pool = slice < slices ? a.c.k : a.c.v;
    const uint32_t col = (slice % slices) * 64 + (tid % 8) * 8;
    uint4 x[8];
    bool ok[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t i = r0 + j * 32 + tid / 8;
      const int32_t t = i < a.p.budget ? kept[i] : -1;
      const int32_t from = t >= 0 && !(IN_PLACE && t == (int32_t)i) ? paged_page(a.c, b, t) : -1;
      ok[j] = from >= 0;
      if (ok[j]) x[j] = *reinterpret_cast<const uint4*>(pool + paged_at(a.c, from, kh, t) + col);
    }
    if (IN_PLACE) __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t i = r0 + j * 32 + tid / 8;
      const int32_t dst = ok[j] ? place(i) : -1;
      if (dst >= 0) *reinterpret_cast<uint4*>(pool + paged_at(a.c, dst, kh, i) + col) = x[j];
    }
    if (IN_PLACE) __syncthreads();
  }
}

uint32_t log2_of(uint32_t v) {
  uint32_t s = 0;
  while ((1u << s) < v) s++;
  return s;
}

}  // namespace

int paged_check(const char* what, const snl_paged_cache* c, const snl_paged_batch* b, PagedView* v) {
  const std::string w = what;
  if (!c || !b) return fail(SNL_E_INVALID, w + ": null argument");
  if (!c->k || !c->v || !b->table || !b->start || !b->len) return fail(SNL_E_INVALID, w + ": null array");
  if (c->type != SNL_T_F16 && c->type != SNL_T_BF16) return fail(SNL_E_UNSUPPORTED, w + ": the cache is f16 or bf16");
  if (c->head_dim != 128 && c->head_dim != 256) return fail(SNL_E_UNSUPPORTED, w + ": head_dim must be 128 or 256");
  if (c->page_size < 8 || (c->page_size & (c->page_size - 1)))
    return fail(SNL_E_UNSUPPORTED, w + ": page_size must be a power of two of at least 8");
  if (c->n_kv == 0 || c->n_kv > 65535u || c->n_pages == 0 || c->n_pages > 0x7fffffffu)
    return fail(SNL_E_INVALID, w + ": empty cache");
  if (b->n_seqs > 65535u) return fail(SNL_E_UNSUPPORTED, w + ": more than 65535 sequences");
  if (b->n_rows > (1u << 24)) return fail(SNL_E_UNSUPPORTED, w + ": more than 2^24 rows");
  if (b->table_stride == 0 && b->n_seqs) return fail(SNL_E_INVALID, w + ": empty table rows");
  if (!paged_aligned(c->k) || !paged_aligned(c->v) || c->page_stride % 8 || c->head_stride % 8 || c->slot_stride % 8)
    return fail(SNL_E_INVALID, w + ": pages must be aligned to 16 bytes");
  if (c->slot_stride < c->head_dim || (c->n_kv > 1 && c->head_stride < c->head_dim) ||
      (c->n_pages > 1 && c->page_stride < c->head_dim))
    return fail(SNL_E_INVALID, w + ": page strides overlap");
  v->k = static_cast<uint16_t*>(c->k);
  v->v = static_cast<uint16_t*>(c->v);
  v->weight = c->weight;
  v->ps = c->page_stride;
  v->hs = c->head_stride;
  v->ss = c->slot_stride;
  v->table = b->table;
  v->start = b->start;
  v->len = b->len;
  v->n_pages = c->n_pages;
  v->shift = log2_of(c->page_size);
  v->n_kv = c->n_kv;
  v->n_seqs = b->n_seqs;
  v->n_rows = b->n_rows;
  v->table_stride = b->table_stride;
  const uint64_t slots = (uint64_t)b->table_stride * c->page_size;
  v->max_len = (int32_t)std::min<uint64_t>({(uint64_t)b->max_len, slots, (uint64_t)(1u << 30)});
  return SNL_OK;
}

int paged_check_attn(const char* what, const snl_paged_cache& c, const snl_paged_batch& b, const snl_paged_attn_p* p,
                     PagedMask* m) {
  const std::string w = what;
  if (!p) return fail(SNL_E_INVALID, w + ": null argument");
  if (p->n_heads == 0 || p->n_heads % c.n_kv || p->n_heads / c.n_kv > 64)
    return fail(SNL_E_UNSUPPORTED, w + ": n_heads must be 1 to 64 times n_kv");
  if (!(p->scale == p->scale) || p->scale > 3e38f || p->scale < -3e38f || !(p->cap >= 0.f) || p->cap > 3e38f)
    return fail(SNL_E_INVALID, w + ": scale must be finite, cap finite and not negative");
  if (!paged_strides(c.type, p->q_row, p->q_head)) return fail(SNL_E_INVALID, w + ": q rows must be aligned to 16 bytes");
  m->slopes = p->slopes;
  m->first = p->first;
  m->last = p->last;
  m->window = (int32_t)std::min<uint32_t>(p->window, 1u << 30);
  m->scale = p->scale;
  m->cap = p->cap;
  return SNL_OK;
}

}  // namespace snl

using namespace snl;

extern "C" int snl_rope_table(double theta, uint32_t rot_dim, uint32_t n_pos, float* table, void* stream) {
  if (!table) return fail(SNL_E_INVALID, "snl_rope_table: null argument");
  if (!(theta > 0) || rot_dim == 0 || rot_dim % 2 || rot_dim > 256)
    return fail(SNL_E_INVALID, "snl_rope_table: theta must be positive, rot_dim even and at most 256");
  const uint64_t n = (uint64_t)n_pos * (rot_dim / 2);
  if (n == 0) return SNL_OK;
  if (n > (1ull << 38)) return fail(SNL_E_UNSUPPORTED, "snl_rope_table: too many positions");
  rope_table_kernel<<<(unsigned)((n + 255) / 256), 256, 0, (cudaStream_t)stream>>>(theta, rot_dim, n_pos,
                                                                                 reinterpret_cast<float2*>(table));
  SNL_LAUNCH_CHECK("rope_table");
  return SNL_OK;
}

extern "C" int snl_paged_append(const snl_paged_cache* c, const snl_paged_batch* b, const snl_paged_append_p* p,
                                const void* q, const void* k, const void* v, const float* q_norm, const float* k_norm,
                                const uint32_t* pos, const float* rope, void* q_out, void* stream) {
  const std::string w = "snl_paged_append";
  AppendArgs a{};
  SNL_TRY(paged_check("snl_paged_append", c, b, &a.c));
  if (!p || (b->n_rows && (!k || !v))) return fail(SNL_E_INVALID, w + ": null argument");
  if (b->n_rows == 0) return SNL_OK;
  if ((p->n_heads != 0) != (q != nullptr) || (q != nullptr) != (q_out != nullptr))
    return fail(SNL_E_INVALID, w + ": q and q_out are given with n_heads, or none of them");
  if (p->in_type != SNL_T_F32 && p->in_type != c->type)
    return fail(SNL_E_UNSUPPORTED, w + ": q, k and v are f32 or of the cache's type");
  if (p->rot_dim % 2 || p->rot_dim > c->head_dim) return fail(SNL_E_UNSUPPORTED, w + ": invalid rotary dim");
  if (p->rot_dim && (!pos || !rope || p->n_pos == 0)) return fail(SNL_E_INVALID, w + ": null positions or rotary table");
  if (p->axes > SNL_ROPE_INTERLEAVED || p->pairs > SNL_ROPE_ADJACENT)
    return fail(SNL_E_INVALID, w + ": unknown rotary layout");
  if (p->axes == SNL_ROPE_SECTIONS &&
      (uint64_t)p->sections[0] + p->sections[1] + p->sections[2] != p->rot_dim / 2)
    return fail(SNL_E_INVALID, w + ": the sections must add up to rot_dim / 2");
  if (p->axes == SNL_ROPE_INTERLEAVED && (p->sections[1] > 256 || p->sections[2] > 256))
    return fail(SNL_E_INVALID, w + ": sections out of range");
  if (!paged_aligned(q) || !paged_aligned(k) || !paged_aligned(v) || !paged_aligned(q_out) || !paged_aligned(pos) ||
      !paged_aligned(q_norm) || !paged_aligned(k_norm) || !paged_strides(p->in_type, p->q_row, p->q_head) ||
      !paged_strides(p->in_type, p->k_row, p->k_head) || !paged_strides(p->in_type, p->v_row, p->v_head) ||
      !paged_strides(c->type, p->out_row, p->out_head) || (reinterpret_cast<uintptr_t>(rope) & 7))
    return fail(SNL_E_INVALID, w + ": rows must be aligned to 16 bytes");
  if (b->n_seqs == 0) return SNL_OK;
  a.p = *p;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.pos = reinterpret_cast<const uint4*>(pos);
  a.rope = reinterpret_cast<const float2*>(rope);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.cache_type = c->type;
  SNL_TRY(paged_error_word(&a.c.err));
  const uint64_t items = (uint64_t)b->n_rows * (p->n_heads + 2 * c->n_kv);
  if (items > (1ull << 33)) return fail(SNL_E_UNSUPPORTED, w + ": too many rows");
  const dim3 grid((unsigned)((items + kAppendWarps - 1) / kAppendWarps));
  if (c->head_dim == 256)
    SNL_PDL_LAUNCH("append_kernel", append_kernel<256>, grid, dim3(kAppendWarps * 32), (size_t)0, (cudaStream_t)stream, a);
  else
    SNL_PDL_LAUNCH("append_kernel", append_kernel<128>, grid, dim3(kAppendWarps * 32), (size_t)0, (cudaStream_t)stream, a);
  return SNL_OK;
}

extern "C" int snl_paged_evict(const snl_paged_cache* c, const snl_paged_batch* b, const snl_paged_evict_p* p,
                               int32_t* kept, const int32_t* into, int32_t* new_len, void* stream) {
  const std::string w = "snl_paged_evict";
  EvictArgs a{};
  SNL_TRY(paged_check("snl_paged_evict", c, b, &a.c));
  if (!p) return fail(SNL_E_INVALID, w + ": null argument");
  if (!c->weight) return fail(SNL_E_INVALID, w + ": the cache has no weights");
  if (p->budget == 0 || p->budget > (1u << 30) || (uint64_t)p->sink + p->recent > p->budget)
    return fail(SNL_E_INVALID, w + ": budget must be positive and hold sink + recent slots");
  if (!kept || !new_len) return fail(SNL_E_INVALID, w + ": null argument");
  if (into && (uint64_t)p->into_stride * c->page_size < std::min<uint64_t>(p->budget, (uint64_t)a.c.max_len))
    return fail(SNL_E_INVALID, w + ": the new pages do not hold the budget");
  if (b->n_seqs == 0) return SNL_OK;
  a.p = *p;
  a.kept = kept;
  a.into = into;
  a.new_len = new_len;
  a.head_dim = c->head_dim;
  SNL_TRY(paged_error_word(&a.c.err));
  const cudaStream_t s = (cudaStream_t)stream;
  SNL_PDL_LAUNCH("evict_select_kernel", evict_select_kernel, dim3(c->n_kv, b->n_seqs), dim3(kSelectThreads), (size_t)0, s, a);
  const uint32_t slices = 2 * (c->head_dim * 2 / 128) + 1;
  const uint32_t all = (uint32_t)std::min<uint64_t>(p->budget, (uint64_t)std::max(a.c.max_len, 1));
  uint32_t steps = into ? (all + kMoveRows - 1) / kMoveRows : 1;
  steps = std::min<uint32_t>(steps, std::max(1u, 65535u / b->n_seqs));
  const dim3 grid(slices, c->n_kv, b->n_seqs * steps);
  if (into)
    SNL_PDL_LAUNCH("evict_move_kernel", evict_move_kernel<false>, grid, dim3(kMoveThreads), (size_t)0, s, a, steps);
  else
    SNL_PDL_LAUNCH("evict_move_kernel", evict_move_kernel<true>, grid, dim3(kMoveThreads), (size_t)0, s, a, steps);
  return SNL_OK;
}
