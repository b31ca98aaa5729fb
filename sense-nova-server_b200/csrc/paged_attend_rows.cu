// Attention over the paged cache for single tokens (and two rows a sequence): the work is
// reading the keys and values once.
#include <algorithm>
#include <string>

#include "paged_attend.cuh"
#include "paged_rows.cuh"

namespace snl {
namespace {

// Shared memory: each warp's ring of stages (8 keys of K, then of V, each [64-element chunk]
// [8 keys][128 bytes], 128-byte swizzled), then each warp's output for up to 8 heads.
template <int D>
struct RowGeo {
  static constexpr uint32_t kGroup = D * 16, kStage = 2 * kGroup;
  static constexpr uint32_t kStages = 2, kPerSm = D == 256 ? 1 : 2;
  static constexpr uint32_t kRing = kRowWarps * kStages * kStage;
  static constexpr uint32_t kSmem = kRing + kRowWarps * 8 * D * 4;
};

struct RowArgs {
  AttendArgs a;
  float* part;      // [CTA][2][group][D], then the same of (max, sum): a CTA's first and last unfinished piece
  float2* part_ml;
  int2* span;       // [row][KV head]: first and last CTA
  uint32_t cluster;  // CTAs of a row and KV head (attend_short_kernel)
};

// The keys of a row.
struct RowKeys {
  uint32_t b;
  int32_t lo, hi, t, len;
};
__device__ __forceinline__ RowKeys row_keys(const PagedView& c, const PagedMask& m, uint32_t r) {
  uint32_t b = min(r, c.n_seqs - 1);  // mostly start[b] = b
  const int32_t s0 = __ldg(c.start + b), s1 = __ldg(c.start + b + 1), n = __ldg(c.len + b);
  const int32_t first = m.first ? __ldg(m.first + r) : 0;
  if (s0 == (int32_t)r && s1 == (int32_t)r + 1 && s1 <= (int32_t)c.n_rows && n > 0 && n <= c.max_len) {
    // the sequence's only row, at its last slot, which no `last` can pass: nothing more to look up
    RowKeys k{b, m.window ? max(first, n - m.window) : first, n, n - 1, n};
    k.lo = max(k.lo, 0);
    if (k.lo >= k.hi) k.lo = k.hi = 0;
    return k;
  }
  if (s0 > (int32_t)r || s1 <= (int32_t)r) {
    uint32_t lo = 0, hi = c.n_seqs;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if ((uint32_t)__ldg(c.start + mid) <= r) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  const int2 rr = paged_rows(c, b);
  RowKeys k{b, 0, 0, 0, paged_len(c, b)};
  k.t = k.len - (rr.y - (int32_t)r);
  if ((int32_t)r < rr.x || (int32_t)r >= rr.y) return k;
  const int2 keys = paged_keys(m, r, k.t, k.len);
  k.lo = keys.x, k.hi = keys.y;
  return k;
}
__device__ __forceinline__ uint32_t row_blocks(const RowKeys& k) {
  return k.lo < k.hi ? ((uint32_t)k.hi + kBlock - 1) / kBlock - (uint32_t)k.lo / kBlock : 0;
}

// Where a walk over the blocks stands: blocks of (KV head, row) in that order of importance.
struct Walk {
  uint64_t left;  // blocks, this one included
  uint32_t kh, row, blk, end, first;  // block numbers of the row: this one, one past its last, its first
  RowKeys k;
};
__device__ __forceinline__ void enter_row(const RowArgs& A, Walk& w) {
  w.k = row_keys(A.a.c, A.a.m, w.row);
  w.first = (uint32_t)w.k.lo / kBlock;
  w.end = w.first + row_blocks(w.k);
}
__device__ __forceinline__ void next_block(const RowArgs& A, Walk& w) {
  w.left--;
  w.blk++;
  while (w.left && w.blk >= w.end) {
    if (++w.row == A.a.c.n_rows) w.row = 0, w.kh++;
    enter_row(A, w);
    w.blk = w.first;
  }
}

// One element of the output: x gated, and with the first of a head its log-sum-exp.
__device__ __forceinline__ void put_element(const AttendArgs& a, uint32_t row, uint32_t head, uint32_t d, float x, float l, float zero) {
  auto value = [](const void* p, uint64_t i, uint32_t type) {
    return type == SNL_T_F32 ? static_cast<const float*>(p)[i]
           : type == SNL_T_F16 ? __half2float(static_cast<const __half*>(p)[i])
                               : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  };
  if (a.gate && l != 0.f) x *= sigmoidf_(value(a.gate, (uint64_t)row * a.p.gate_row + (uint64_t)head * a.p.gate_head + d, a.p.gate_type));
  const uint64_t to = (uint64_t)row * a.p.out_row + (uint64_t)head * a.p.out_head + d;
  if (a.p.out_type == SNL_T_F32) static_cast<float*>(a.out)[to] = x;
  else if (a.p.out_type == SNL_T_F16) static_cast<__half*>(a.out)[to] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(a.out)[to] = __float2bfloat16_rn(x);
  if (a.lse && d == 0) a.lse[(uint64_t)row * a.p.n_heads + head] = l == 0.f ? -INFINITY : (zero + log2f(l)) * (1.f / kLog2e);
}
constexpr uint32_t kRowCluster = 8;  // at most
__device__ __forceinline__ float ld_cluster(uint32_t addr) { return __uint_as_float(ld_cluster_u32(addr)); }

// The blocks of 64 keys of all (KV head, row) pairs form one line that is cut into equal
// shares, one for each CTA: every SM reads the same number of bytes whatever the lengths are.
// A row that ends inside its CTA is written at once; pieces of rows cut by a share's end are
// left to rows_join_kernel. A warp takes 8 keys of each block through its own ring of TMA
// boxes: S = Q K^T on m16n8k16 (query heads as rows), O^T += V^T P^T on m16n8k8, whose B
// operand is the score fragment as it stands: its weights are rounded to the cache's type (2^-11 or
// 2^-8 of each, as V itself is), sums and output stay in 32 bits.
//
// Bound by memory: 16 tokens of 16 heads of 256 over up to 32768 keys 189 us (1.19 GB, 6.3
// TB/s, 0.97 of a copy's rate; 243 with the tiles of attend_kernel), 64 of 32 heads of 128 over
// up to 4096 keys with capped scores 82 us (5.5 TB/s; 113 with one CTA an SM).
//
// CLUSTER: a cluster of 1 to 8 CTAs takes each (KV head, row) instead, an equal share of its
// blocks each, and joins them through shared memory: one launch in place of two, for short rows.
template <typename T, int D, bool CLUSTER>
__device__ __forceinline__ void attend_rows(const RowArgs& A, const CUtensorMap& kmap, const CUtensorMap& vmap) {
  using G = RowGeo<D>;
  constexpr uint32_t NS = G::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[kRowWarps][NS];
  __shared__ uint32_t scan_sh[kRowWarps], found_sh[2];
  __shared__ float2 ml_sh[kRowWarps][8], own_ml[8];
  float* mo = reinterpret_cast<float*>(smem + G::kRing);  // [warp][8 heads][D]
  const AttendArgs& a = A.a;
  pdl_trigger();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023) {
    report_timeout(a.c.err);
    return;
  }
  if (lane == 0)
    for (uint32_t s = 0; s < NS; s++) mbar_init(&bars[warp][s], 1);
  fence_mbar_init();
  pdl_wait();

  Walk now;
  uint32_t total = 0;
  uint64_t share = 0, g1 = 0;
  if constexpr (CLUSTER) {
    now.row = blockIdx.x / A.cluster / a.c.n_kv;
    now.kh = blockIdx.x / A.cluster % a.c.n_kv;
    enter_row(A, now);
    const uint32_t n = now.end - now.first, part = blockIdx.x % A.cluster, from = (uint32_t)((uint64_t)n * part / A.cluster);
    now.left = (uint32_t)((uint64_t)n * (part + 1) / A.cluster) - from;
    now.blk = now.first + from;
    for (uint32_t i = tid; i < a.group * D; i += kRowWarps * 32) mo[i] = 0.f;
    if (tid < 8) own_ml[tid] = make_float2(-INFINITY, 0.f);
    __syncthreads();
  } else {
    // Blocks before each thread's rows, this CTA's share, and the row that it starts in.
    const uint32_t per = (a.c.n_rows + kRowWarps * 32 - 1) / (kRowWarps * 32), r0 = min(tid * per, a.c.n_rows),
                   r1 = min(r0 + per, a.c.n_rows);
    uint32_t mine = 0;
    for (uint32_t r = r0; r < r1; r++) mine += row_blocks(row_keys(a.c, a.m, r));
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= (uint32_t)o) upto += v;
    }
    if (lane == 31) scan_sh[warp] = upto;
    __syncthreads();
    for (uint32_t i = 0; i < kRowWarps; i++) {
      if (i < warp) upto += scan_sh[i];
      total += scan_sh[i];
    }
    const uint64_t all = (uint64_t)total * a.c.n_kv;
    share = (all + gridDim.x - 1) / gridDim.x;
    const uint64_t g0 = blockIdx.x * share;
    if (g0 >= all) return;
    g1 = min(g0 + share, all);
    {
      uint32_t off = (uint32_t)(g0 % total);
      if (off >= upto - mine && off < upto) {
        off -= upto - mine;
        uint32_t r = r0;
        for (;; r++) {
          const uint32_t n = row_blocks(row_keys(a.c, a.m, r));
          if (off < n) break;
          off -= n;
        }
        found_sh[0] = r;
        found_sh[1] = off;
      }
    }
    __syncthreads();
    now.left = g1 - g0;
    now.kh = (uint32_t)(g0 / total);
    now.row = found_sh[0];
    enter_row(A, now);
    now.blk = now.first + found_sh[1];
  }
  Walk ahead = now;  // of the loads

  const uint32_t ring = smem_u32(smem) + warp * NS * G::kStage;
  // Pages of this warp's keys in 32 blocks from `base` on, one a lane.
  int32_t pages = -1;
  uint32_t base = 0xFFFFFFFFu, prow = 0xFFFFFFFFu;
  uint32_t issued = 0, taken = 0;
  auto active = [&](const Walk& w) {
    const int32_t key = (int32_t)(w.blk * kBlock + warp * 8);
    return key + 8 > w.k.lo && key < w.k.hi;
  };
  auto issue = [&] {  // the next group that this warp has, if any
    while (ahead.left) {
      const bool use = active(ahead);
      if (use) {
        if (prow != ahead.row || ahead.blk - base >= 32) {
          prow = ahead.row;
          base = ahead.blk;
          const uint32_t key = (base + lane) * kBlock + warp * 8;
          pages = (int32_t)key < ahead.k.hi ? paged_page(a.c, ahead.k.b, key) : -1;
        }
        const int32_t page = __shfl_sync(0xffffffffu, pages, ahead.blk - base);
        if (lane == 0) {
          const uint32_t st = issued % NS, dst = ring + st * G::kStage;
          const int slot = (int)((ahead.blk * kBlock + warp * 8) & ((1u << a.c.shift) - 1)),
                    pg = page < 0 ? (int)a.c.n_pages : page;  // past the end: zeros
          mbar_arrive_expect_tx(&bars[warp][st], G::kStage);
          tma_group(dst, &kmap, slot, (int)ahead.kh, pg, &bars[warp][st]);
          tma_group(dst + G::kGroup, &vmap, slot, (int)ahead.kh, pg, &bars[warp][st]);
        }
        issued++;
      }
      next_block(A, ahead);
      if (use) return;
    }
  };
  for (uint32_t s = 0; s < NS; s++) issue();

  const uint32_t g = lane >> 2, t = lane & 3;
  const float flip = a.m.scale < 0.f ? -1.f : 1.f, sl = fmaxf(fabsf(a.m.scale) * kLog2e, 1e-30f) * flip;
  const float cap = a.m.cap, pre = cap > 0.f ? a.m.scale / cap : 0.f;
  bool ok = true;
  uint32_t q[D / 16][2];
  float o[D / 16][4];
  float m_run = -INFINITY, l_run = 0.f;
  bool fresh = true;
  float slope = 0.f;
  const uint32_t head = g;  // of the group
  while (now.left) {
    if (fresh) {  // a new row: its queries (heads past the group are 0)
      fresh = false;
#pragma unroll
      for (int c = 0; c < D / 16; c++) {
        q[c][0] = q[c][1] = 0;
        if (head < a.group) {
          const uint16_t* s = a.q + (uint64_t)now.row * a.p.q_row + (uint64_t)(now.kh * a.group + head) * a.p.q_head + 16 * c + 2 * t;
          q[c][0] = *reinterpret_cast<const uint32_t*>(s);
          q[c][1] = *reinterpret_cast<const uint32_t*>(s + 8);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) o[c][e] = 0.f;
      }
      slope = a.m.slopes && head < a.group ? __ldg(a.m.slopes + now.kh * a.group + head) * kLog2e : 0.f;
      m_run = -INFINITY;
      l_run = 0.f;
    }
    if (active(now)) {
      const uint32_t st = taken % NS, kat = ring + st * G::kStage, vat = kat + G::kGroup;
      ok = __all_sync(0xffffffffu, ok && wait_mbar(&bars[warp][st], (taken / NS) & 1));
      taken++;
      const int32_t key = (int32_t)(now.blk * kBlock + warp * 8 + 2 * t);
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t c = 0; c < D / 32; c++) {
        uint32_t kb[4];
        ldsm4(kb, box_at(kat, c, lane));
        mma_k16<T>(s0, q[2 * c][0], 0, q[2 * c][1], 0, kb[0], kb[1]);  // rows 8-15 are not used
        mma_k16<T>(s1, q[2 * c + 1][0], 0, q[2 * c + 1][1], 0, kb[2], kb[3]);
      }
      // head g, keys `key` and key + 1
      float x0 = s0[0] + s1[0], x1 = s0[1] + s1[1];
      if (cap > 0.f) {
        x0 = cap * kLog2e * tanh_(x0 * pre);
        x1 = cap * kLog2e * tanh_(x1 * pre);
      } else {
        x0 *= sl;
        x1 *= sl;
      }
      if (slope != 0.f) {
        x0 -= slope * fabsf((float)(now.k.t - key));
        x1 -= slope * fabsf((float)(now.k.t - key - 1));
      }
      const bool in0 = key >= now.k.lo && key < now.k.hi, in1 = key + 1 >= now.k.lo && key + 1 < now.k.hi;
      if (!in0) x0 = -INFINITY;
      if (!in1) x1 = -INFINITY;
      float mx = fmaxf(x0, x1);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (__any_sync(0xffffffffu, mx > m_run + 8.f)) {  // the reference moves only for scores 2^8 above it
        const float to = mx > m_run + 8.f ? mx : m_run, f = to == m_run ? 1.f : ex2(m_run - to);
        m_run = to;
        l_run *= f;
        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < D / 16; c++) o[c][0] *= f0, o[c][1] *= f1, o[c][2] *= f0, o[c][3] *= f1;
      }
      const float zero = m_run == -INFINITY ? 0.f : m_run;
      x0 = ex2(x0 - zero);
      x1 = ex2(x1 - zero);
      l_run += x0 + x1;
      const uint32_t p = pack2(x0, x1, T());
      // values of keys that the row does not see may be anything: not 0 * that, but 0
      const uint32_t keep = (in0 ? 0xFFFFu : 0u) | (in1 ? 0xFFFF0000u : 0u);
#pragma unroll
      for (uint32_t c = 0; c < D / 32; c++) {
        uint32_t v[4];
        ldsm4_t(v, box_at(vat, c, lane));
        mma_k8<T>(o[2 * c], v[0] & keep, v[1] & keep, p);
        mma_k8<T>(o[2 * c + 1], v[2] & keep, v[3] & keep, p);
      }
      fence_proxy_async_smem();  // the stage was read; the next box is written to it after that
      __syncwarp();
      issue();
    }
    const Walk was = now;
    next_block(A, now);
    if (now.left && now.row == was.row && now.kh == was.kh) continue;
    // The row's piece in this CTA is done: join the warps.
    fresh = true;
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
#pragma unroll
    for (int c = 0; c < D / 16; c++) {  // column 2t, 2t + 1: heads; row g, g + 8: elements
      float* at = mo + (warp * 8 + 2 * t) * D + 16 * c + g;
      if (2 * t < a.group) at[0] = o[c][0], at[8] = o[c][2];
      if (2 * t + 1 < a.group) at[D] = o[c][1], at[D + 8] = o[c][3];
    }
    if (t == 0) ml_sh[warp][g] = make_float2(m_run, l_run);
    __syncthreads();
    uint64_t c_first = 0;
    bool whole = false;
    if constexpr (!CLUSTER) {
      const uint64_t g_row = g1 - was.left + 1 - (was.blk - was.first + 1);  // the line's block where the row starts
      const uint64_t n_row = was.end - was.first, c_last = (g_row + n_row - 1) / share;
      c_first = g_row / share;
      whole = c_first == c_last;
      if (c_first == blockIdx.x && tid == 0)
        A.span[(uint64_t)was.row * a.c.n_kv + was.kh] = make_int2((int)c_first, (int)c_last);
    }
    for (uint32_t h = tid / D; h < a.group; h += kRowWarps * 32 / D) {
      const uint32_t d = tid % D;
      float top = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < kRowWarps; i++) top = fmaxf(top, ml_sh[i][h].x);
      const float zero = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (uint32_t i = 0; i < kRowWarps; i++) {
        const float2 ml = ml_sh[i][h];
        if (ml.y == 0.f) continue;
        const float f = ml.x == -INFINITY ? 1.f : ex2(ml.x - zero);
        l = fmaf(ml.y, f, l);
        x = fmaf(mo[(i * 8 + h) * D + d], f, x);
      }
      if constexpr (CLUSTER) {
        mo[h * D + d] = x;  // this thread alone read it
        if (d == 0) own_ml[h] = make_float2(top, l);
        continue;
      }
      if (!whole) {
        const uint64_t at = ((uint64_t)blockIdx.x * 2 + (c_first == blockIdx.x ? 1 : 0)) * a.group + h;
        A.part[at * D + d] = x;
        if (d == 0) A.part_ml[at] = make_float2(top, l);
        continue;
      }
      put_element(a, was.row, was.kh * a.group + h, d, l == 0.f ? 0.f : x / l, l, zero);
    }
    __syncthreads();
  }
  if (!ok) {
    // A wait gave up: this warp's boxes still in flight land before the CTA ends.
    if (lane == 0) report_timeout(a.c.err);
    for (uint32_t i = issued > NS ? issued - NS : 0; i < issued; i++) (void)wait_mbar(&bars[warp][i % NS], (i / NS) & 1);
  }
  if constexpr (CLUSTER) {  // each CTA joins its part of the row's elements
    cluster_sync();
    const uint32_t n = a.group * D / A.cluster, part = blockIdx.x % A.cluster;
    for (uint32_t i = part * n + tid; i < (part + 1) * n; i += kRowWarps * 32) {
      float2 ml[kRowCluster];
      float x[kRowCluster], top = -INFINITY;
#pragma unroll
      for (uint32_t r = 0; r < kRowCluster; r++) {
        ml[r] = make_float2(-INFINITY, 0.f);
        x[r] = 0.f;
        if (r >= A.cluster) continue;
        ml[r].x = ld_cluster(in_cta(&own_ml[i / D].x, r));
        ml[r].y = ld_cluster(in_cta(&own_ml[i / D].y, r));
        x[r] = ld_cluster(in_cta(&mo[i], r));
        top = fmaxf(top, ml[r].x);
      }
      const float zero = top == -INFINITY ? 0.f : top;
      float l = 0.f, sum = 0.f;
#pragma unroll
      for (uint32_t r = 0; r < kRowCluster; r++) {
        if (ml[r].y == 0.f) continue;
        const float f = ml[r].x == -INFINITY ? 1.f : ex2(ml[r].x - zero);
        l = fmaf(ml[r].y, f, l);
        sum = fmaf(x[r], f, sum);
      }
      put_element(a, now.row, now.kh * a.group + i / D, i % D, l == 0.f ? 0.f : sum / l, l, zero);
    }
    cluster_sync();  // no CTA ends while another reads its memory
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32, RowGeo<D>::kPerSm)
    attend_rows_kernel(const __grid_constant__ RowArgs A, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
  attend_rows<T, D, false>(A, kmap, vmap);
}
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32, RowGeo<D>::kPerSm)
    attend_short_kernel(const __grid_constant__ RowArgs A, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap) {
  attend_rows<T, D, true>(A, kmap, vmap);
}

// Joins the pieces of rows that lie in several shares, and writes rows without keys. One warp
// per (row, head).
constexpr uint32_t kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) rows_join_kernel(const __grid_constant__ RowArgs A) {
  constexpr int E = D / 32;
  const AttendArgs& a = A.a;
  pdl_trigger();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t item = (uint64_t)blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  const uint32_t r = (uint32_t)(item / a.p.n_heads), hq = (uint32_t)(item % a.p.n_heads), kh = hq / a.group, h = hq % a.group;
  pdl_wait();
  if (r >= a.c.n_rows) return;
  const int2 span = A.span[(uint64_t)r * a.c.n_kv + kh];  // not set for a row without keys
  const RowKeys k = row_keys(a.c, a.m, r);
  float l = 0.f, zero = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; i++) o[i] = 0.f;
  if (k.lo < k.hi) {
    if (span.x == span.y) return;  // written already
    auto place = [&](int c) { return ((uint64_t)c * 2 + (c == span.x ? 1 : 0)) * a.group + h; };
    float top = -INFINITY;
    for (int c0 = span.x; c0 <= span.y; c0 += 32) {
      const int c = c0 + (int)lane;
      if (c <= span.y) top = fmaxf(top, A.part_ml[place(c)].x);
    }
    top = warp_max(top);
    zero = top == -INFINITY ? 0.f : top;
#pragma unroll 4
    for (int c = span.x; c <= span.y; c++) {
      const float2 x = A.part_ml[place(c)];
      float v[E];
      load_as_float<E>(A.part, place(c) * D + lane * E, SNL_T_F32, v);
      const float f = x.y == 0.f ? 0.f : x.x == -INFINITY ? 1.f : ex2(x.x - zero);
      l = fmaf(x.y, f, l);
#pragma unroll
      for (int i = 0; i < E; i++) o[i] = x.y == 0.f ? o[i] : fmaf(v[i], f, o[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float gate[E];
  if (a.gate) load_as_float<E>(a.gate, (uint64_t)r * a.p.gate_row + (uint64_t)hq * a.p.gate_head + lane * E, a.p.gate_type, gate);
#pragma unroll
  for (int i = 0; i < E; i++) o[i] = l == 0.f ? 0.f : o[i] * (a.gate ? inv * sigmoidf_(gate[i]) : inv);
  store_from_float<E>(a.out, (uint64_t)r * a.p.out_row + (uint64_t)hq * a.p.out_head + lane * E, a.p.out_type, o);
  if (a.lse && lane == 0) a.lse[item] = l == 0.f ? -INFINITY : (zero + log2f(l)) * (1.f / kLog2e);
}

uint32_t rows_grid(const snl_paged_cache& c, const snl_paged_batch& b) {
  const uint64_t len = std::min<uint64_t>(b.max_len, (uint64_t)b.table_stride * c.page_size);
  const uint64_t most = (uint64_t)b.n_rows * c.n_kv * ((len + kBlock - 1) / kBlock + 1);
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, (uint64_t)std::max(1, sm_count()) * (c.head_dim == 256 ? RowGeo<256>::kPerSm : RowGeo<128>::kPerSm)));
}

template <typename T, int D>
int go_rows(const snl_paged_cache& c, const RowArgs& r, uint32_t grid, cudaStream_t s) {
  CUtensorMap km, vm;
  SNL_TRY(page_map(&km, c, c.k, 8, D / 64));
  SNL_TRY(page_map(&vm, c, c.v, 8, D / 64));
  static bool attr[64] = {};
  static int room[64][4] = {};  // clusters of 1, 2, 4 and 8 CTAs that the GPU runs at once
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(SNL_E_UNSUPPORTED, "snl_paged_attend: device number");
  if (!attr[dev]) {
    SNL_CUDA_TRY(cudaFuncSetAttribute(attend_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RowGeo<D>::kSmem));
    SNL_CUDA_TRY(cudaFuncSetAttribute(attend_short_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RowGeo<D>::kSmem));
    for (uint32_t i = 0; i < 4; i++) {
      cudaLaunchAttribute at{};
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim.x = 1u << i;
      at.val.clusterDim.y = at.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(1u << i);
      cfg.blockDim = dim3(kRowWarps * 32);
      cfg.dynamicSmemBytes = RowGeo<D>::kSmem;
      cfg.attrs = &at;
      cfg.numAttrs = 1;
      int n = 0;
      SNL_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, attend_short_kernel<T, D>, &cfg));
      room[dev][i] = n;
    }
    attr[dev] = true;
  }
  // The largest clusters of which one wave holds all rows, up to 512 keys for each CTA. Against
  // equal shares, one to 16 rows of one length, and of lengths from an eighth of the longest up: up
  // to 512 keys a CTA all gain (head_dim 256: 1 row of 517 keys 12.0 -> 8.5 us, of 4096 18.5 -> 15.0; 8 of
  // 1024 14.9 -> 11.4; 16 of up to 1024 19.0 -> 15.4), with 1024 uneven rows lose (8 of up to 8192 29 -> 40).
  constexpr uint32_t kShortKeys = 512;
  const uint64_t pairs = (uint64_t)r.a.c.n_rows * c.n_kv;
  int i = 3;
  while (i >= 0 && pairs > (uint64_t)room[dev][i]) i--;
  if (i >= 0 && (uint32_t)r.a.c.max_len <= kShortKeys << i) {
    RowArgs brief = r;
    brief.cluster = 1u << i;
    const cudaError_t e = launch_pdl_clusters(attend_short_kernel<T, D>, brief.cluster, dim3((unsigned)pairs * brief.cluster),
                                              dim3(kRowWarps * 32), (size_t)RowGeo<D>::kSmem, s, brief, km, vm);
    if (e != cudaSuccess) return cuda_fail(e, "attend_short_kernel");
    count_launch();
    return SNL_OK;
  }
  SNL_PDL_LAUNCH("attend_rows_kernel", (attend_rows_kernel<T, D>), dim3(grid), dim3(kRowWarps * 32), (size_t)RowGeo<D>::kSmem, s,
                 r, km, vm);
  const uint64_t items = (uint64_t)r.a.c.n_rows * r.a.p.n_heads;
  SNL_PDL_LAUNCH("rows_join_kernel", rows_join_kernel<D>, dim3((unsigned)((items + kJoinWarps - 1) / kJoinWarps)),
                 dim3(kJoinWarps * 32), (size_t)0, s, r);
  return SNL_OK;
}

}  // namespace

// The query heads of a KV head are rows of one 16-row product whose last 8 are not used. A
// second row of a sequence reads its keys again here, where a tile of the other kernel holds
// all rows: at head_dim 256 and 27 rows of 16 sequences of up to 32768 keys 212 us against 182
// (single rows 193 against 243), at 13 rows of 8 of up to 2048 keys 24 against 26, and 2 rows of
// one 17 against 21; at head_dim 128 and 104 rows of 64 sequences of up to 4096 keys 129
// against 161.
//
// Those rows were spread evenly. The host knows how many there are, not where: one sequence with
// many of them beside single tokens passes too, and its keys are read once for each of its rows. 32
// tokens over 512 keys of heads of 128 and 34 rows over 4096 take 113 us, in two calls 15 + 23; over
// 32768 633, in two calls 15 + 60; at head_dim 256 32 tokens over 2048 keys and 9 rows over 8192 85,
// in two calls 52 + 23. A caller that has both kinds gives them a batch each.
bool attend_rows_fits(const snl_paged_cache& c, const snl_paged_batch& b, uint32_t group) {
  const uint64_t blocks = (uint64_t)b.n_rows * (b.max_len / kBlock + 2);
  const bool small = blocks * c.n_kv <= 8192, wide = c.head_dim == 256;
  return group <= 8 && blocks < (1ull << 31) &&
         (wide && !small ? 4ull * b.n_rows <= 5ull * b.n_seqs : b.n_rows <= 2ull * b.n_seqs);
}

size_t attend_rows_workspace(const snl_paged_cache& c, const snl_paged_batch& b, uint32_t group) {
  return (size_t)rows_grid(c, b) * 2 * group * (c.head_dim + 2) * sizeof(float) + (size_t)b.n_rows * c.n_kv * sizeof(int2);
}

int launch_attend_rows(const snl_paged_cache& c, const snl_paged_batch& b, const AttendArgs& a, void* work, cudaStream_t s) {
  const uint32_t grid = rows_grid(c, b);
  RowArgs r{};
  r.a = a;
  r.part = static_cast<float*>(work);
  r.part_ml = reinterpret_cast<float2*>(r.part + (size_t)grid * 2 * a.group * c.head_dim);
  r.span = reinterpret_cast<int2*>(r.part_ml + (size_t)grid * 2 * a.group);
  if (c.type == SNL_T_F16) return c.head_dim == 256 ? go_rows<__half, 256>(c, r, grid, s) : go_rows<__half, 128>(c, r, grid, s);
  return c.head_dim == 256 ? go_rows<__nv_bfloat16, 256>(c, r, grid, s) : go_rows<__nv_bfloat16, 128>(c, r, grid, s);
}

}  // namespace snl
