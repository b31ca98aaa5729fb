// The paged key/value cache: rotary table, append, evict, and the checks of every call.
// attend is in paged_attend.cu and paged_attend_rows.cu, weigh in paged_weigh.cu.
#include <algorithm>
#include <string>

#include "paged_tc.cuh"

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
constexpr int append_heads(int d) { return 1024 / d; }  // heads of a warp
// How a row's elements find their partners: in the lane, a fixed number of lanes away, or
// through shared memory (where a part of a lane's elements turns).
enum { kTurnNone, kTurnLane, kTurnShuffle, kTurnShared };

// One warp takes up to NH query, key or value heads of a row: the row's slot, the turn's (cos,
// sin) and the norm's weights are looked up once for them, while all their elements are on
// the way. A lane holds D / 32 neighbouring elements. Two chunks of up to 4096 rows of 16 + 8
// heads: 43 us (184 MB, 4.3 TB/s, 0.66 of a copy's rate; 116 us with a warp for each head,
// whose look-ups were most of its instructions), 8192 rows in f32 61 us (302 MB, 5.0 TB/s); 8 rows
// are one launch's latency.
template <int D, int TURN, bool IN32>
__global__ void __launch_bounds__(kAppendWarps * 32, IN32 ? 3 : 4) append_kernel(const __grid_constant__ AppendArgs a, uint32_t span) {
  constexpr int E = D / 32, NH = append_heads(D), W = E * (IN32 ? 4 : 2) / 4;  // words of a lane's elements
  __shared__ __align__(16) float rows[TURN == kTurnShared ? kAppendWarps : 1][TURN == kTurnShared ? D : 1];
  pdl_trigger();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t pq = (a.p.n_heads + span - 1) / span, pk = (a.c.n_kv + span - 1) / span, piece = blockIdx.y;
  const uint32_t r = blockIdx.x * kAppendWarps + warp;
  const int what = piece < pq ? 0 : piece < pq + pk ? 1 : 2;  // queries, keys, values
  const uint32_t h0 = (piece - (what == 0 ? 0 : what == 1 ? pq : pq + pk)) * span;
  const int n = (int)min(span, (what ? a.c.n_kv : a.p.n_heads) - h0);
  pdl_wait();
  if (r >= a.c.n_rows) return;

  const uint64_t step = what == 0 ? a.p.q_head : what == 1 ? a.p.k_head : a.p.v_head;  // elements between heads
  const uint8_t* src = static_cast<const uint8_t*>(what == 0 ? a.q : what == 1 ? a.k : a.v) +
                       ((uint64_t)r * (what == 0 ? a.p.q_row : what == 1 ? a.p.k_row : a.p.v_row) + h0 * step + lane * E) *
                           (IN32 ? 4 : 2);
  uint32_t raw[NH][W];
#pragma unroll
  for (int u = 0; u < NH; u++) {
    if (u >= n) continue;
    if constexpr (W == 2) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(src));
      raw[u][0] = x.x, raw[u][1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const uint4 x = ld_stream16(src + 4 * i);
        raw[u][i] = x.x, raw[u][i + 1] = x.y, raw[u][i + 2] = x.z, raw[u][i + 3] = x.w;
      }
    }
    src += step * (IN32 ? 4 : 2);
  }

  uint16_t* dst = a.q_out + (uint64_t)r * a.p.out_row + h0 * a.p.out_head + lane * E;
  uint64_t to = a.p.out_head;
  if (what) {  // the row's slot
    const uint32_t b = paged_seq(a.c, r, lane);
    const int2 rr = paged_rows(a.c, b);
    const int32_t len = paged_len(a.c, b), t = len - (rr.y - (int32_t)r);
    if ((int32_t)r < rr.x || (int32_t)r >= rr.y || t < 0 || t >= len) {
      report_index(a.c.err);
      return;
    }
    const int32_t page = paged_page(a.c, b, t);
    if (page < 0) return;
    dst = (what == 1 ? a.c.k : a.c.v) + paged_at(a.c, page, h0, t) + lane * E;
    to = a.c.hs;
  }
  // y = x cos + partner * sin, the sign of the sine by the place in the pair.
  float cs[E], sn[E];
  const bool turns = TURN != kTurnNone && what < 2 && lane * E < a.p.rot_dim;  // some of the lane's elements
  const uint32_t half = a.p.rot_dim / 2;
  if (turns) {
    const uint4 pos = __ldg(a.pos + r);
    if (max(pos.x, a.p.axes == SNL_ROPE_ONE ? 0u : max(pos.y, pos.z)) >= a.p.n_pos) report_index(a.c.err);
    const uint32_t last = a.p.n_pos - 1, px = min(pos.x, last), py = min(pos.y, last), pz = min(pos.z, last);
    const uint32_t e0 = lane * E, s0 = a.p.sections[0], s1 = s0 + a.p.sections[1];
    const bool adj = TURN == kTurnLane || (TURN == kTurnShared && a.p.pairs == SNL_ROPE_ADJACENT);
    const bool upper = TURN == kTurnShuffle && e0 >= half;  // the lane holds second places
#pragma unroll
    for (int i = 0; i < E; i++) {
      uint32_t f;
      bool second;
      if constexpr (TURN == kTurnShuffle) {
        f = e0 - (upper ? half : 0) + i, second = upper;
      } else if constexpr (TURN == kTurnLane) {
        f = e0 / 2 + i / 2, second = i & 1;
      } else {
        cs[i] = 1.f, sn[i] = 0.f;
        if (e0 + i >= a.p.rot_dim) continue;
        second = adj ? (i & 1) : e0 + i >= half;
        f = adj ? (e0 + i) / 2 : second ? e0 + i - half : e0 + i;
      }
      uint32_t at = px;
      if (a.p.axes == SNL_ROPE_SECTIONS) {
        at = f < s0 ? px : f < s1 ? py : pz;
      } else if (a.p.axes == SNL_ROPE_INTERLEAVED) {
        const uint32_t m = f % 3;
        at = m == 1 && f < 3 * a.p.sections[1] ? py : m == 2 && f < 3 * a.p.sections[2] ? pz : px;
      }
      const float2 v = __ldg(a.rope + (uint64_t)at * half + f);
      cs[i] = v.x;
      sn[i] = second ? v.y : -v.y;
    }
  }
  const float* weights = what == 0 ? a.q_norm : what == 1 ? a.k_norm : nullptr;
  float norm[E];
  if (weights) {
    load_as_float<E>(weights, lane * E, SNL_T_F32, norm);
#pragma unroll
    for (int i = 0; i < E; i++) norm[i] += 1.0f;
  }

  auto head = [&](int u) {
    float x[E];
    if constexpr (IN32) {
#pragma unroll
      for (int i = 0; i < E; i++) x[i] = __uint_as_float(raw[u][i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const float2 f = a.cache_type == SNL_T_F16 ? unpack2(raw[u][i / 2], __half()) : unpack2(raw[u][i / 2], __nv_bfloat16());
        x[i] = f.x, x[i + 1] = f.y;
      }
    }
    if (weights) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < E; i++) s = fmaf(x[i], x[i], s);
      const float inv = rsqrtf(warp_sum(s) / (float)D + a.p.eps);
#pragma unroll
      for (int i = 0; i < E; i++) x[i] = x[i] * inv * norm[i];
    }
    if (TURN != kTurnNone && what < 2) {
      float o[E];
      if constexpr (TURN == kTurnLane) {
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = x[i ^ 1];
      } else if constexpr (TURN == kTurnShuffle) {
        const uint32_t away = half / E, from = lane < away ? lane + away : lane - away;
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = __shfl_sync(0xffffffffu, x[i], from & 31);
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < E; i += 4)
          *reinterpret_cast<float4*>(&rows[warp][lane * E + i]) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < E; i++) {
          const uint32_t e = lane * E + i;
          o[i] = rows[warp][e >= a.p.rot_dim ? e : a.p.pairs == SNL_ROPE_ADJACENT ? e ^ 1 : e < half ? e + half : e - half];
        }
      }
      if (turns) {
#pragma unroll
        for (int i = 0; i < E; i++)
          if (TURN != kTurnShared || lane * E + i < a.p.rot_dim) x[i] = fmaf(x[i], cs[i], o[i] * sn[i]);
      }
    }
    store_from_float<E>(dst + u * to, 0, a.cache_type, x);
  };
  if (n == NH) {  // without a way out between them the heads' sums and turns overlap
#pragma unroll
    for (int u = 0; u < NH; u++) head(u);
  } else {
#pragma unroll
    for (int u = 0; u < NH; u++) {
      if (u >= n) break;
      head(u);
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
  uint32_t head_dim, cluster;  // CTAs that select from one list
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

// One CTA, or a cluster of them, per (KV head, sequence): the n-th largest key of the candidates by four 8-bit radix
// passes (weights crowd in few exponents: eight counts of each digit, by lane, on banks of
// their own), then the kept slots in slot order, 4096 at a time. A thread takes four
// neighbouring slots, which lie in one page. The weights are read once where their keys fit
// shared memory. 32 lists of up to 16384 weights take 16 us by clusters of 4 (22 by one CTA each),
// the copy of their 4096 kept slots 43 us (269 MB in all).
template <bool HELD, bool MANY>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t held[];
  __shared__ uint32_t hist[8][260], sums[2][256], warp_n[32], s_digit, s_need, own_n[2];
  pdl_trigger();
  const uint32_t cs = MANY ? a.cluster : 1, part = blockIdx.x % cs, kh = blockIdx.x / cs, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  if (tid < 2) own_n[tid] = 0;
  if (tid == 0) s_digit = s_need = 0;
  __syncthreads();  // set before any warp adds to them: where `take` is 0 no other barrier comes between
  pdl_wait();
  const int32_t len = paged_len(a.c, b), budget = (int32_t)a.p.budget;
  int32_t* kept = a.kept + ((uint64_t)b * a.c.n_kv + kh) * a.p.budget;
  if (len <= budget) {
    for (int32_t i = part * kSelectThreads + tid; i < budget; i += cs * kSelectThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int32_t t0 = (int32_t)a.p.sink, t1 = len - (int32_t)a.p.recent;  // the candidates
  const int32_t own = (int32_t)(((uint32_t)len + 4 * cs - 1) / (4 * cs)) * 4, from = (int32_t)part * own, end = min(len, from + own);  // this CTA's slots
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
  auto keys_at = [&](int32_t t) -> uint4 { return HELD ? *reinterpret_cast<const uint4*>(held + (t - from)) : fetch(t); };
  const uint32_t take = a.p.budget - a.p.sink - a.p.recent;
  uint32_t cut = 0, need = take;  // the keys' common prefix so far, and how many of it are taken
  for (int shift = 24; take && shift >= 0; shift -= 8) {
    for (uint32_t i = tid; i < 8 * 260; i += kSelectThreads) hist[0][i] = 0;
    __syncthreads();
    for (int32_t base = from; base < end; base += kSelectKeys) {
      const int32_t t = base + 4 * (int32_t)tid;
      uint4 k = make_uint4(0, 0, 0, 0);
      if (t < end) {
        if (HELD && shift == 24) *reinterpret_cast<uint4*>(held + (t - from)) = k = fetch(t);
        else k = keys_at(t);
      }
      const uint32_t ks[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (ks[e] && (shift == 24 || ks[e] >> (shift + 8) == cut >> (shift + 8))) atomicAdd(&hist[lane & 7][(ks[e] >> shift) & 255], 1u);
      }
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t s = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) s += hist[i][tid];
      (MANY ? sums[(shift >> 3) & 1] : hist[0])[tid] = s;
    }
    if constexpr (MANY) {  // over the cluster; the next pass writes the other sums, so one meeting a pass
      cluster_sync();
      if (tid < 256) {
        uint32_t s = 0;
        for (uint32_t r = 0; r < cs; r++) s += ld_cluster_u32(in_cta(&sums[(shift >> 3) & 1][tid], r));
        hist[0][tid] = s;
      }
    }
    __syncthreads();
    if (tid < 32) {  // the digit at which the sum from the top reaches `need`: 8 digits a lane
      uint32_t n[8], s = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) s += n[e] = hist[0][255 - 8 * lane - e];
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
  if constexpr (MANY) {
    for (int32_t t = from + 4 * (int32_t)tid; t < end; t += kSelectKeys) {
      const uint4 k = take ? keys_at(t) : make_uint4(0, 0, 0, 0);
      const uint32_t ks[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const bool must = t + e < len && (t + e < t0 || t + e >= t1), is_sure = must || (take && ks[e] > cut);
        sure += is_sure;
        ties += !is_sure && take && ks[e] == cut;
      }
    }
    sure = __reduce_add_sync(0xffffffffu, sure);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
      atomicAdd(&own_n[0], sure);
      atomicAdd(&own_n[1], ties);
    }
    cluster_sync();
    sure = ties = 0;
    for (uint32_t r = 0; r < part; r++) {
      sure += ld_cluster_u32(in_cta(&own_n[0], r));
      ties += ld_cluster_u32(in_cta(&own_n[1], r));
    }
  }
  for (int32_t base = from; base < end; base += kSelectKeys) {
    const int32_t t = base + 4 * (int32_t)tid;
    const uint4 k = take && t < end ? keys_at(t) : make_uint4(0, 0, 0, 0);
    const uint32_t ks[4] = {k.x, k.y, k.z, k.w};
    uint32_t mine = 0;  // sure ones, ties << 16
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool must = t < end && t + e < len && (t + e < t0 || t + e >= t1);
      mine += must || (take && ks[e] > cut) ? 1u : take && ks[e] == cut ? 1u << 16 : 0u;
    }
    uint32_t all;
    const uint32_t before = select_scan(mine, warp_n, all);
    uint32_t s = sure + (before & 0xFFFF), q = ties + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool must = t < end && t + e < len && (t + e < t0 || t + e >= t1);
      const bool is_sure = must || (take && ks[e] > cut), tie = !is_sure && take && ks[e] == cut;
      const uint32_t at = s + min(q, need);
      if ((is_sure || (tie && q < need)) && at < a.p.budget) kept[at] = t + e;
      s += is_sure;
      q += tie;
    }
    sure += all & 0xFFFF;
    ties += all >> 16;
  }
  if constexpr (MANY) cluster_sync();  // no CTA ends while another reads its counts
}

constexpr uint32_t kMoveThreads = 256, kMoveRows = 8 * 32;  // rows of one step: 8 per group of 8 threads

// Moves kept slots to their new places within the batch's own pages. A CTA takes 128 bytes of
// every row (8 threads to a row) of k or v, or the weights, and walks the rows in order, so
// that a place is overwritten only after its slot was read: kept slots never move up. Its steps
// of 256 rows follow one another, each a trip to memory: 1100 slots to 1024 take 25 us with their
// selection (to new pages 11), 8 x 16384 to 4096 120 us (272 MB).
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
  // Without sequences the batch's arrays have no elements, and maybe no address.
  if (!c->k || !c->v || (b->n_seqs && (!b->table || !b->start || !b->len))) return fail(SNL_E_INVALID, w + ": null array");
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
  if (reinterpret_cast<uintptr_t>(table) & 7) return fail(SNL_E_INVALID, "snl_rope_table: table must be aligned to 8 bytes");
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
  if (!(p->eps >= 0.f) || p->eps > 3e38f) return fail(SNL_E_INVALID, w + ": eps must be finite and not negative");
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
  if (paged_overlap(b->n_rows, p->out_row, p->n_heads ? c->head_dim : 0) || paged_overlap(p->n_heads, p->out_head, c->head_dim))
    return fail(SNL_E_INVALID, w + ": the rows of q_out overlap");
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
  // Heads of one warp: with many rows as many as it holds, with few rows they spread over the SMs.
  const uint32_t heads = p->n_heads + 2 * c->n_kv;
  const uint64_t all = (uint64_t)b->n_rows * heads, warps = (uint64_t)std::max(1, sm_count()) * kAppendWarps * 4;
  const uint32_t span = (uint32_t)std::min<uint64_t>(append_heads(c->head_dim), std::max<uint64_t>(1, all / warps));
  const uint64_t pieces = (p->n_heads + span - 1) / span + 2ull * ((c->n_kv + span - 1) / span);
  if (pieces > 65535) return fail(SNL_E_UNSUPPORTED, w + ": too many heads");
  const uint32_t e = c->head_dim / 32;  // elements of a lane: a lane turns whole where they divide rot_dim
  const int turn = !p->rot_dim ? kTurnNone : p->pairs == SNL_ROPE_ADJACENT && p->rot_dim % e == 0 ? kTurnLane
                   : p->pairs == SNL_ROPE_HALVES && p->rot_dim / 2 % e == 0 ? kTurnShuffle : kTurnShared;
  auto go = [&](auto kern) -> int {
    SNL_PDL_LAUNCH("append_kernel", kern, dim3((b->n_rows + kAppendWarps - 1) / kAppendWarps, (unsigned)pieces), dim3(kAppendWarps * 32),
                   (size_t)0, (cudaStream_t)stream, a, span);
    return SNL_OK;
  };
  auto by_turn = [&](auto d, auto in32) -> int {
    constexpr int D = decltype(d)::value;
    constexpr bool I = decltype(in32)::value;
    return turn == kTurnNone      ? go(append_kernel<D, kTurnNone, I>)
           : turn == kTurnLane    ? go(append_kernel<D, kTurnLane, I>)
           : turn == kTurnShuffle ? go(append_kernel<D, kTurnShuffle, I>)
                                  : go(append_kernel<D, kTurnShared, I>);
  };
  auto by_type = [&](auto d) -> int {
    return p->in_type == SNL_T_F32 ? by_turn(d, std::true_type()) : by_turn(d, std::false_type());
  };
  return c->head_dim == 256 ? by_type(std::integral_constant<int, 256>()) : by_type(std::integral_constant<int, 128>());
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
  if (b->n_seqs && (!kept || !new_len)) return fail(SNL_E_INVALID, w + ": null argument");
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
  // CTAs of a list: 4096 slots for each, and no more CTAs than the SMs hold, two each (32 lists of
  // 16384 slots, with the copy of 1024: 28 us with one, 24 with 2, 21 with 4, 23 with 8; of 65536
  // 90, 40, 37, 32; 128 lists of 16384 48, 43, 53, 86).
  const uint64_t lists = (uint64_t)c->n_kv * b->n_seqs;
  a.cluster = 8;
  while (a.cluster > 1 && ((uint32_t)a.c.max_len < 4096 * a.cluster || lists * a.cluster > 2ull * sm_count())) a.cluster /= 2;
  const dim3 sel(c->n_kv * a.cluster, b->n_seqs);
  const uint32_t own = (uint32_t)(((uint64_t)a.c.max_len + 4 * a.cluster - 1) / (4 * a.cluster)) * 4;
  auto select = [&](auto kern, bool held, bool* done) -> int {
    int dev = 0;
    cudaGetDevice(&dev);
    if (held && (dev < 0 || dev >= 64 || !done[dev])) {
      SNL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSelectHeld * sizeof(uint32_t))));
      if (dev >= 0 && dev < 64) done[dev] = true;
    }
    const cudaError_t e = launch_pdl_clusters(kern, a.cluster, sel, dim3(kSelectThreads), held ? own * sizeof(uint32_t) : 0, s, a);
    if (e != cudaSuccess) return cuda_fail(e, "evict_select_kernel");
    count_launch();
    return SNL_OK;
  };
  static bool attr[2][64] = {};
  const bool many = a.cluster > 1;
  if (own <= kSelectHeld) SNL_TRY(many ? select(evict_select_kernel<true, true>, true, attr[1]) : select(evict_select_kernel<true, false>, true, attr[0]));
  else SNL_TRY(many ? select(evict_select_kernel<false, true>, false, nullptr) : select(evict_select_kernel<false, false>, false, nullptr));
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
