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
// How a row's elements find their partners: in the lane, a fixed number of lanes away, or
// through shared memory (halves that do not end with a lane).
enum { kTurnNone, kTurnLane, kTurnShuffle, kTurnShared };

// One warp takes `span` of a row's heads (queries, then keys, then values), four at a time: the
// row's slot, the turn's (cos, sin) and the norm's weights are looked up once for them. A
// lane holds D / 32 neighbouring elements.
template <int D, int TURN>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(const __grid_constant__ AppendArgs a, uint32_t span) {
  constexpr int E = D / 32;
  __shared__ __align__(16) float rows[TURN == kTurnShared ? kAppendWarps : 1][TURN == kTurnShared ? D : 1];
  pdl_trigger();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t nq = a.p.n_heads, heads = nq + 2 * a.c.n_kv, pieces = (heads + span - 1) / span;
  const uint64_t item = (uint64_t)blockIdx.x * kAppendWarps + warp;
  const uint32_t r = (uint32_t)(item / pieces), h0 = (uint32_t)(item % pieces) * span, h1 = min(h0 + span, heads);
  pdl_wait();
  if (r >= a.c.n_rows) return;

  // The slot, for keys and values.
  int32_t page = -1, t = 0;
  if (h1 > nq) {
    const uint32_t b = paged_seq(a.c, r, lane);
    const int2 rr = paged_rows(a.c, b);
    const int32_t len = paged_len(a.c, b);
    t = len - (rr.y - (int32_t)r);
    if ((int32_t)r < rr.x || (int32_t)r >= rr.y || t < 0 || t >= len) report_index(a.c.err);
    else page = paged_page(a.c, b, t);
  }
  // y = x cos + partner * sin, the sign of the sine by the place in the pair.
  float cs[E], sn[E];
  bool turned[E];
  const uint32_t half = a.p.rot_dim / 2;
  const bool adj = a.p.pairs == SNL_ROPE_ADJACENT;
  if constexpr (TURN != kTurnNone) {
    const uint4 pos = __ldg(a.pos + r);
#pragma unroll
    for (int i = 0; i < E; i++) {
      const uint32_t e = lane * E + i;
      turned[i] = e < a.p.rot_dim;
      cs[i] = 1.f, sn[i] = 0.f;
      if (!turned[i]) continue;
      const bool second = adj ? (e & 1) : e >= half;
      const uint32_t f = adj ? e / 2 : second ? e - half : e;
      uint32_t at = pos.x;
      if (a.p.axes == SNL_ROPE_SECTIONS)
        at = f < a.p.sections[0] ? pos.x : f < a.p.sections[0] + a.p.sections[1] ? pos.y : pos.z;
      else if (a.p.axes == SNL_ROPE_INTERLEAVED)
        at = f % 3 == 1 && f < 3 * a.p.sections[1] ? pos.y : f % 3 == 2 && f < 3 * a.p.sections[2] ? pos.z : pos.x;
      if (at >= a.p.n_pos) {
        report_index(a.c.err);
        at = 0;
      }
      const float2 v = __ldg(a.rope + (uint64_t)at * half + f);
      cs[i] = v.x;
      sn[i] = second ? v.y : -v.y;
    }
  }
  float wq[E], wk[E];
#pragma unroll
  for (int i = 0; i < E; i++) wq[i] = wk[i] = 0.f;
  if (a.q_norm && h0 < nq) load_as_float<E>(a.q_norm, lane * E, SNL_T_F32, wq);
  if (a.k_norm && h1 > nq) load_as_float<E>(a.k_norm, lane * E, SNL_T_F32, wk);

  for (uint32_t hb = h0; hb < h1; hb += 4) {
    float x[4][E];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t h = hb + u;
      if (h >= h1) continue;
      if (h < nq) load_as_float<E>(a.q, (uint64_t)r * a.p.q_row + (uint64_t)h * a.p.q_head + lane * E, a.p.in_type, x[u]);
      else if (h < nq + a.c.n_kv)
        load_as_float<E>(a.k, (uint64_t)r * a.p.k_row + (uint64_t)(h - nq) * a.p.k_head + lane * E, a.p.in_type, x[u]);
      else
        load_as_float<E>(a.v, (uint64_t)r * a.p.v_row + (uint64_t)(h - nq - a.c.n_kv) * a.p.v_head + lane * E, a.p.in_type, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t h = hb + u;
      if (h >= h1) break;
      const bool is_q = h < nq, is_v = h >= nq + a.c.n_kv;
      if (!is_v) {
        if (is_q ? a.q_norm : a.k_norm) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < E; i++) s = fmaf(x[u][i], x[u][i], s);
          const float inv = rsqrtf(warp_sum(s) / (float)D + a.p.eps);
#pragma unroll
          for (int i = 0; i < E; i++) x[u][i] = x[u][i] * inv * (1.0f + (is_q ? wq[i] : wk[i]));
        }
        if constexpr (TURN != kTurnNone) {
          float o[E];
          if constexpr (TURN == kTurnLane) {
#pragma unroll
            for (int i = 0; i < E; i++) o[i] = x[u][i ^ 1];
          } else if constexpr (TURN == kTurnShuffle) {
            const uint32_t away = half / E, from = lane < away ? lane + away : lane - away;
#pragma unroll
            for (int i = 0; i < E; i++) o[i] = __shfl_sync(0xffffffffu, x[u][i], from & 31);
          } else {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < E; i += 4)
              *reinterpret_cast<float4*>(&rows[warp][lane * E + i]) = make_float4(x[u][i], x[u][i + 1], x[u][i + 2], x[u][i + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < E; i++) {
              const uint32_t e = lane * E + i;
              o[i] = rows[warp][e < half ? e + half : e < a.p.rot_dim ? e - half : e];
            }
          }
#pragma unroll
          for (int i = 0; i < E; i++)
            if (turned[i]) x[u][i] = fmaf(x[u][i], cs[i], o[i] * sn[i]);
        }
      }
      uint16_t* dst;
      if (is_q) {
        dst = a.q_out + (uint64_t)r * a.p.out_row + (uint64_t)h * a.p.out_head;
      } else {
        if (page < 0) continue;
        dst = (is_v ? a.c.v : a.c.k) + paged_at(a.c, page, is_v ? h - nq - a.c.n_kv : h - nq, t);
      }
      store_from_float<E>(dst, lane * E, a.cache_type, x[u]);
    }
  }
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

constexpr uint32_t kSelectThreads = 1024, kSelectKeys = 4 * kSelectThreads;
constexpr uint32_t kSelectHeld = 48 * 1024;  // candidates whose keys are held in shared memory (192 KB)

// Sums of v over the threads before this one, and over all of them.
__device__ __forceinline__ uint32_t select_scan(uint32_t v, uint32_t* sh, uint32_t& all) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= (uint32_t)o) s += x;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = s;
  __syncthreads();
  uint32_t w = sh[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= (uint32_t)o) w += x;
  }
  all = __shfl_sync(0xffffffffu, w, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
  return s - v + (warp ? before : 0);
}

// One CTA per (KV head, sequence): the n-th largest key of the candidates by four 8-bit radix
// passes (equal digits of a warp are counted by one addition: weights crowd in few
// exponents), then the kept slots in slot order, 4096 at a time. A thread takes four
// neighbouring slots, which lie in one page. The weights are read once where their keys fit
// shared memory.
template <bool HELD>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t held[];
  __shared__ uint32_t hist[256], warp_n[32], s_digit, s_need;
  pdl_trigger();
  pdl_wait();
  const uint32_t kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int32_t len = paged_len(a.c, b), budget = (int32_t)a.p.budget;
  int32_t* kept = a.kept + ((uint64_t)b * a.c.n_kv + kh) * a.p.budget;
  if (len <= budget) {
    for (int32_t i = tid; i < budget; i += kSelectThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int32_t t0 = (int32_t)a.p.sink, t1 = len - (int32_t)a.p.recent;  // the candidates
  // Keys of slots t to t + 3 (t a multiple of 4): 0 for what is no candidate, which no weight maps to.
  auto fetch = [&](int32_t t) -> uint4 {
    uint4 k = make_uint4(0, 0, 0, 0);
    if (t + 3 < t0 || t >= t1) return k;
    const int32_t page = paged_page(a.c, b, t);
    if (page < 0) return k;
    const float4 w = *reinterpret_cast<const float4*>(a.c.weight + paged_weight_at(a.c, page, kh, t));
    if (t >= t0 && t < t1) k.x = weight_key(w.x);
    if (t + 1 >= t0 && t + 1 < t1) k.y = weight_key(w.y);
    if (t + 2 >= t0 && t + 2 < t1) k.z = weight_key(w.z);
    if (t + 3 >= t0 && t + 3 < t1) k.w = weight_key(w.w);
    return k;
  };
  auto keys_at = [&](int32_t t) -> uint4 { return HELD ? *reinterpret_cast<const uint4*>(held + t) : fetch(t); };
  const uint32_t take = a.p.budget - a.p.sink - a.p.recent;
  uint32_t cut = 0, need = take;  // the keys' common prefix so far, and how many of it are taken
  for (int shift = 24; take && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int32_t base = 0; base < len; base += kSelectKeys) {
      const int32_t t = base + 4 * (int32_t)tid;
      uint4 k = make_uint4(0, 0, 0, 0);
      if (t < len) {
        if (HELD && shift == 24) *reinterpret_cast<uint4*>(held + t) = k = fetch(t);
        else k = keys_at(t);
      }
      const uint32_t ks[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const bool in = ks[e] && (shift == 24 || ks[e] >> (shift + 8) == cut >> (shift + 8));
        const uint32_t d = in ? (ks[e] >> shift) & 255 : 256;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (in && lane == (uint32_t)__ffs(same) - 1) atomicAdd(&hist[d], __popc(same));
      }
    }
    __syncthreads();
    if (tid < 32) {  // the digit at which the sum from the top reaches `need`: 8 digits a lane
      uint32_t n[8], s = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) s += n[e] = hist[255 - 8 * lane - e];
      uint32_t upto = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= (uint32_t)o) upto += x;
      }
      uint32_t before = upto - s;
      if (before < need && upto >= need) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if (before < need && before + n[e] >= need) {
            s_digit = 255 - 8 * lane - e;
            s_need = need - before;
          }
          before += n[e];
        }
      }
    }
    __syncthreads();
    cut |= s_digit << shift;
    need = s_need;
  }
  // Kept: what must be, what lies above the cut, and of its equals the first `need`.
  uint32_t sure = 0, ties = 0;  // before this stretch
  for (int32_t base = 0; base < len; base += kSelectKeys) {
    const int32_t t = base + 4 * (int32_t)tid;
    const uint4 k = take && t < len ? keys_at(t) : make_uint4(0, 0, 0, 0);
    const uint32_t ks[4] = {k.x, k.y, k.z, k.w};
    uint32_t mine = 0;  // sure ones, ties << 16
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool must = t + e < len && (t + e < t0 || t + e >= t1);
      mine += must || (take && ks[e] > cut) ? 1u : take && ks[e] == cut ? 1u << 16 : 0u;
    }
    uint32_t all;
    const uint32_t before = select_scan(mine, warp_n, all);
    uint32_t s = sure + (before & 0xFFFF), q = ties + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool must = t + e < len && (t + e < t0 || t + e >= t1);
      const bool is_sure = must || (take && ks[e] > cut), tie = !is_sure && take && ks[e] == cut;
      const uint32_t at = s + min(q, need);
      if ((is_sure || (tie && q < need)) && at < a.p.budget) kept[at] = t + e;
      s += is_sure;
      q += tie;
    }
    sure += all & 0xFFFF;
    ties += all >> 16;
  }
}

constexpr uint32_t kMoveThreads = 256, kMoveRows = 8 * 32;  // rows of one step: 8 per group of 8 threads

// Moves kept slots to their new places within the batch's own pages. A CTA takes 128 bytes of
// every row (8 threads to a row) of k or v, or the weights, and walks the rows in order, so
// that a place is overwritten only after its slot was read: kept slots never move up.
__global__ void __launch_bounds__(kMoveThreads) evict_shift_kernel(const __grid_constant__ EvictArgs a) {
  pdl_trigger();
  pdl_wait();
  const uint32_t slices = a.head_dim * 2 / 128;  // of k, then as many of v, then the weights
  const uint32_t slice = blockIdx.x, kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int32_t* kept = a.kept + ((uint64_t)b * a.c.n_kv + kh) * a.p.budget;
  if (slice == 2 * slices && kh == 0 && tid == 0) a.new_len[b] = min(paged_len(a.c, b), (int32_t)a.p.budget);
  for (uint32_t r0 = 0; r0 < a.p.budget; r0 += kMoveRows) {
    if (kept[r0] < 0) break;  // the same for the whole CTA: nothing is kept from here on
    if (slice == 2 * slices) {
      const uint32_t i = r0 + tid;
      const int32_t t = i < a.p.budget && kept[i] < a.c.max_len ? kept[i] : -1;
      const int32_t from = t >= 0 ? paged_page(a.c, b, t) : -1, dst = t >= 0 ? paged_page(a.c, b, i) : -1;
      const bool ok = from >= 0 && dst >= 0;
      float w = 0.f;
      if (ok) w = a.c.weight[paged_weight_at(a.c, from, kh, t)];
      __syncthreads();
      if (ok) a.c.weight[paged_weight_at(a.c, dst, kh, i)] = w;
      __syncthreads();
      continue;
    }
    uint16_t* pool = slice < slices ? a.c.k : a.c.v;
    const uint32_t col = (slice % slices) * 64 + (tid % 8) * 8;
    uint4 x[8];
    bool ok[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t i = r0 + j * 32 + tid / 8;
      const int32_t t = i < a.p.budget && kept[i] < a.c.max_len ? kept[i] : -1;
      const int32_t from = t >= 0 && t != (int32_t)i ? paged_page(a.c, b, t) : -1;
      ok[j] = from >= 0;
      if (ok[j]) x[j] = *reinterpret_cast<const uint4*>(pool + paged_at(a.c, from, kh, t) + col);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t i = r0 + j * 32 + tid / 8;
      const int32_t dst = ok[j] ? paged_page(a.c, b, i) : -1;
      if (dst >= 0) *reinterpret_cast<uint4*>(pool + paged_at(a.c, dst, kh, i) + col) = x[j];
    }
    __syncthreads();
  }
}

constexpr uint32_t kCopyRows = 32;  // kept slots of a CTA: 4 of each warp, k and v

// Copies kept slots to new pages: every slot on its own, whole rows of k and v by a warp each,
// all of a warp's loads before its stores.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) evict_copy_kernel(const __grid_constant__ EvictArgs a, uint32_t steps) {
  constexpr uint32_t L = D * 2 / 16, R = 32 / L;  // lanes of a row; rows of a warp's load
  __shared__ uint64_t from_sh[kCopyRows], to_sh[kCopyRows];
  pdl_trigger();
  pdl_wait();
  const uint32_t kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t* kept = a.kept + ((uint64_t)b * a.c.n_kv + kh) * a.p.budget;
  if (blockIdx.x == 0 && kh == 0 && tid == 0) a.new_len[b] = min(paged_len(a.c, b), (int32_t)a.p.budget);
  constexpr uint64_t none = ~0ull;
  for (uint32_t r0 = blockIdx.x * kCopyRows; r0 < a.p.budget; r0 += steps * kCopyRows) {
    if (kept[r0] < 0) break;
    if (tid < kCopyRows) {
      const uint32_t i = r0 + tid;
      const int32_t t = i < a.p.budget && kept[i] < a.c.max_len ? kept[i] : -1;  // (unset where a page was bad)
      uint64_t from = none, to = none;
      if (t >= 0) {
        const int32_t p = paged_page(a.c, b, t), n = __ldg(a.into + (uint64_t)b * a.p.into_stride + (i >> a.c.shift));
        if (n < 0 || n >= (int32_t)a.c.n_pages) report_index(a.c.err);
        else if (p >= 0) {
          from = paged_at(a.c, p, kh, t);
          to = paged_at(a.c, n, kh, i);
          a.c.weight[paged_weight_at(a.c, n, kh, i)] = a.c.weight[paged_weight_at(a.c, p, kh, t)];
        }
      }
      from_sh[tid] = from;
      to_sh[tid] = to;
    }
    __syncthreads();
    constexpr uint32_t N = kCopyRows / 8 / R;  // loads of k, and of v
    uint4 x[2 * N];
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
      const uint64_t from = from_sh[warp * (kCopyRows / 8) + j * R + lane / L];
      if (from == none) continue;
      x[2 * j] = ld_stream16(a.c.k + from + lane % L * 8);
      x[2 * j + 1] = ld_stream16(a.c.v + from + lane % L * 8);
    }
#pragma unroll
    for (uint32_t j = 0; j < N; j++) {
      const uint64_t to = to_sh[warp * (kCopyRows / 8) + j * R + lane / L];
      if (to == none) continue;
      *reinterpret_cast<uint4*>(a.c.k + to + lane % L * 8) = x[2 * j];
      *reinterpret_cast<uint4*>(a.c.v + to + lane % L * 8) = x[2 * j + 1];
    }
    __syncthreads();
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
  // Heads of one warp: many rows share the row's look-ups among 8 heads, few rows spread theirs
  // over the SMs (8 rows of 24 heads: 3 each).
  const uint32_t heads = p->n_heads + 2 * c->n_kv;
  const uint64_t all = (uint64_t)b->n_rows * heads, warps = (uint64_t)std::max(1, sm_count()) * kAppendWarps * 4;
  const uint32_t span = (uint32_t)std::min<uint64_t>(8, std::max<uint64_t>(1, all / warps));
  const uint64_t items = (uint64_t)b->n_rows * ((heads + span - 1) / span);
  if (items > (1ull << 33)) return fail(SNL_E_UNSUPPORTED, w + ": too many rows");
  const uint32_t e = c->head_dim / 32;
  const int turn = !p->rot_dim ? kTurnNone : p->pairs == SNL_ROPE_ADJACENT ? kTurnLane
                   : p->rot_dim / 2 % e == 0 && p->rot_dim / 2 / e <= 16 ? kTurnShuffle : kTurnShared;
  auto go = [&](auto kern) -> int {
    SNL_PDL_LAUNCH("append_kernel", kern, dim3((unsigned)((items + kAppendWarps - 1) / kAppendWarps)), dim3(kAppendWarps * 32),
                   (size_t)0, (cudaStream_t)stream, a, span);
    return SNL_OK;
  };
  auto by_turn = [&](auto d) -> int {
    constexpr int D = decltype(d)::value;
    return turn == kTurnNone      ? go(append_kernel<D, kTurnNone>)
           : turn == kTurnLane    ? go(append_kernel<D, kTurnLane>)
           : turn == kTurnShuffle ? go(append_kernel<D, kTurnShuffle>)
                                  : go(append_kernel<D, kTurnShared>);
  };
  return c->head_dim == 256 ? by_turn(std::integral_constant<int, 256>()) : by_turn(std::integral_constant<int, 128>());
}

extern "C" int snl_paged_evict(const snl_paged_cache* c, const snl_paged_batch* b, const snl_paged_evict_p* p,
                               int32_t* kept, const int32_t* into, int32_t* new_len, void* stream) {
  const std::string w = "snl_paged_evict";
  EvictArgs a{};
  SNL_TRY(paged_check("snl_paged_evict", c, b, &a.c));
  if (!p) return fail(SNL_E_INVALID, w + ": null argument");
  if (!c->weight) return fail(SNL_E_INVALID, w + ": the cache has no weights");
  if (!paged_aligned(c->weight)) return fail(SNL_E_INVALID, w + ": the weights must be aligned to 16 bytes");
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
  const dim3 sel(c->n_kv, b->n_seqs);
  if ((uint32_t)a.c.max_len <= kSelectHeld) {
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr[dev]) {
      SNL_CUDA_TRY(cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(kSelectHeld * sizeof(uint32_t))));
      if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    const size_t smem = ((size_t)a.c.max_len + 3) / 4 * 16;
    SNL_PDL_LAUNCH("evict_select_kernel", evict_select_kernel<true>, sel, dim3(kSelectThreads), smem, s, a);
  } else {
    SNL_PDL_LAUNCH("evict_select_kernel", evict_select_kernel<false>, sel, dim3(kSelectThreads), (size_t)0, s, a);
  }
  if (!into) {
    SNL_PDL_LAUNCH("evict_shift_kernel", evict_shift_kernel, dim3(2 * (c->head_dim * 2 / 128) + 1, c->n_kv, b->n_seqs),
                   dim3(kMoveThreads), (size_t)0, s, a);
    return SNL_OK;
  }
  const uint32_t most = (uint32_t)std::min<uint64_t>(p->budget, (uint64_t)std::max(a.c.max_len, 1));
  const uint32_t steps = (most + kCopyRows - 1) / kCopyRows;
  const dim3 grid(steps, c->n_kv, b->n_seqs);
  if (c->head_dim == 256)
    SNL_PDL_LAUNCH("evict_copy_kernel", evict_copy_kernel<256>, grid, dim3(kMoveThreads), (size_t)0, s, a, steps);
  else
    SNL_PDL_LAUNCH("evict_copy_kernel", evict_copy_kernel<128>, grid, dim3(kMoveThreads), (size_t)0, s, a, steps);
  return SNL_OK;
}
