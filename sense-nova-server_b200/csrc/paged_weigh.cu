// Accumulated attention weights of the paged cache's slots (snl_paged_weigh).
#include <algorithm>
#include <string>

#include "paged_tc.cuh"

namespace snl {
namespace {

struct WeighArgs {
  PagedView c;
  PagedMask m;
  snl_paged_attn_p p;
  const uint16_t* q;
  const float* lse;
  float decay;
  uint32_t group, toks;  // query heads per KV head; tokens of half a query tile (64 / group)
};

// The new weight of a slot: sums start at 0 for the step's own slots.
__device__ __forceinline__ void put_weight(const WeighArgs& a, uint32_t b, uint32_t kh, int32_t key, int32_t old_len,
                                           float sum) {
  const int32_t page = paged_page(a.c, b, key);
  if (page < 0) return;
  float* w = a.c.weight + paged_weight_at(a.c, page, kh, key);
  *w = a.decay != 0.f && key < old_len ? fmaf(*w, a.decay, sum) : sum;
}
// log2 of what a row's exponentials are divided by; rows without keys divide by infinity.
__device__ __forceinline__ float log2_sum(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// ---- few rows: one pass over the keys ------------------------------------------------------

constexpr uint32_t kWeighWarps = 8, kWeighGroups = 4;  // 8-key groups of one warp

// One warp takes 8 keys (of one page) at a time, a lane D / 32 elements of each; the products
// with 4 heads at once are 32 sums over the lanes, folded so that each lane ends with one.
template <typename T, int D>
__global__ void __launch_bounds__(kWeighWarps * 32, 2) weigh_rows_kernel(const __grid_constant__ WeighArgs a) {
  constexpr int E = D / 32, W = E / 2;
  pdl_trigger();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, kh = blockIdx.y, b = blockIdx.z;
  const int32_t len = paged_len(a.c, b);
  const int32_t key0 = (int32_t)((blockIdx.x * kWeighWarps + (threadIdx.x >> 5)) * kWeighGroups * 8);
  if (key0 >= len) return;
  const int2 rr = paged_rows(a.c, b);
  auto load = [&](int32_t key, uint32_t (&x)[8][W]) -> int32_t {
    const int32_t page = key < len ? paged_page(a.c, b, key) : -1;
#pragma unroll
    for (int k = 0; k < 8; k++) {
#pragma unroll
      for (int e = 0; e < W; e++) x[k][e] = 0;
      if (page < 0 || key + k >= len) continue;
      const uint16_t* s = a.c.k + paged_at(a.c, page, kh, key + k) + lane * E;
      if constexpr (E == 8) {
        const uint4 v = ld_stream16(s);
        x[k][0] = v.x, x[k][1] = v.y, x[k][2] = v.z, x[k][3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(s);
        x[k][0] = v.x, x[k][1] = v.y;
      }
    }
    return page;
  };
  uint32_t x[8][W], next[8][W];
  load(key0, x);
  for (uint32_t n = 0; n < kWeighGroups; n++) {
    const int32_t key = key0 + (int32_t)n * 8, mine = key + (int32_t)(lane & 7);
    if (key >= len) return;
    if (n + 1 < kWeighGroups) load(key + 8, next);
    float sum = 0.f;
    for (int32_t r = rr.x; r < rr.y; r++) {
      const int32_t t = len - (rr.y - r);
      const int2 keys = paged_keys(a.m, r, t, len);
      if (key + 8 <= keys.x || key >= keys.y) continue;
      for (uint32_t g = 0; g < a.group; g += 4) {
        float v[32];
#pragma unroll
        for (int h = 0; h < 4; h++) {
          float q[E];
          if (g + h < a.group) {
            load_as_float<E>(a.q, (uint64_t)r * a.p.q_row + (uint64_t)(kh * a.group + g + h) * a.p.q_head + lane * E,
                             std::is_same<T, __half>::value ? SNL_T_F16 : SNL_T_BF16, q);
          } else {
#pragma unroll
            for (int e = 0; e < E; e++) q[e] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < 8; k++) {
            float2 s = make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < W; e++) s = fma2(unpack2(x[k][e], T()), make_float2(q[2 * e], q[2 * e + 1]), s);
            v[h * 8 + k] = s.x + s.y;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const bool up = lane & o;
#pragma unroll
          for (int i = 0; i < o; i++) {
            const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
        }
        // lane 8 h + k: head g + h, key + k
        const uint32_t h = g + lane / 8, head = kh * a.group + h;
        if (h < a.group && mine >= keys.x && mine < keys.y) {
          float s = v[0] * a.m.scale;
          if (a.m.cap > 0.f) s = a.m.cap * tanh_(s / a.m.cap);
          if (a.m.slopes) s -= __ldg(a.m.slopes + head) * fabsf((float)(t - mine));
          sum += ex2(fmaf(s, kLog2e, -log2_sum(__ldg(a.lse + (uint64_t)r * a.p.n_heads + head))));
        }
      }
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    if (lane < 8 && mine < len) put_weight(a, b, kh, mine, len - (rr.y - rr.x), sum);
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
      for (int e = 0; e < W; e++) x[k][e] = next[k][e];
  }
}

// ---- many rows: S^T = K Q^T on the tensor cores ---------------------------------------------

// Shared memory of one CTA: its 128 keys [8-key group][64-element chunk][8 keys][128 bytes],
// and stages of half a query tile [chunk][64 rows][128 bytes]. Tensor memory: three tiles of
// 128 keys x 128 (token, head) rows, and from column 384 the keys, the products' A operand
// (from shared memory it and the queries would take the whole of its bandwidth).
template <int D>
struct WeighGeo {
  static constexpr uint32_t kK = 128 * D * 2, kGroup = D * 16;
  static constexpr uint32_t kQ = 64 * D * 2;
  static constexpr uint32_t kStages = 4, kMeta = 4, kBufs = 3, kTK = 384;
  static constexpr uint32_t kSmem = D == 256 ? kK + kStages * kQ : 160 * 1024;  // one CTA an SM, and none that holds tensor memory
};
constexpr uint32_t kSumWarps = 16, kWeighThreads = (kSumWarps + 3) * 32;  // 16: the exponentials bound the sums

// What the sums need of a query tile's 128 rows (read 16 bytes at a time).
struct alignas(16) WeighMeta {
  float lse2[128], t[128], slope[128];
  int32_t lo[128], hi[128];
  int32_t tile;  // -1: no more tiles
  int32_t full;  // every row sees every key of the cluster
};

// A cluster = (256 keys of a sequence and KV head), a CTA 128 of them, thread = key: the
// scores of a query tile come with a key's row in one lane of tensor memory, so its sum over
// the rows needs no exchange. The last warp lists the query tiles that see the keys, with what
// each row needs; one loads their queries by TMA, one of the first CTA issues the products.
template <typename T, int D, bool GENERAL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWeighThreads, 1)
    weigh_tile_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap qmap) {
  using G = WeighGeo<D>;
  constexpr uint32_t NS = G::kStages, NM = G::kMeta, NB = G::kBufs;
  extern __shared__ __align__(1024) uint8_t smem_k[];
  uint8_t* smem_q = smem_k + G::kK;
  __shared__ WeighMeta meta[NM];
  __shared__ uint64_t k_full, q_full[NS], q_empty[NS], m_full[NM], m_empty[NM], s_full[G::kBufs], s_empty[G::kBufs], k_there, drained;
  __shared__ uint32_t tmem_sh;
  __shared__ float part_sh[3][128];
  __shared__ volatile int fail_sh;
  pdl_trigger();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = cluster_rank();
  const uint32_t cl = blockIdx.x / 2, kh = cl % a.c.n_kv, b = cl / a.c.n_kv % a.c.n_seqs, kt = cl / a.c.n_kv / a.c.n_seqs;
  if (smem_u32(smem_k) & 1023) {  // the swizzle needs it; the same for every CTA
    report_timeout(a.c.err);
    return;
  }
  if (tid == 0) {
    mbar_init(&k_full, 1);
    for (uint32_t s = 0; s < NS; s++) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (uint32_t s = 0; s < NM; s++) {
      mbar_init(&m_full[s], 1);
      mbar_init(&m_empty[s], kSumWarps + 2);
    }
    for (uint32_t s = 0; s < NB; s++) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 2 * kSumWarps);  // of both CTAs
    }
    mbar_init(&k_there, 2 * kSumWarps);
    mbar_init(&drained, 1);
    fail_sh = 0;
    fence_mbar_init();
  }
  if (warp == kSumWarps + 1) tmem_alloc2<512>(&tmem_sh);
  pdl_wait();
  const int32_t len = paged_len(a.c, b), k0 = (int32_t)(kt * 256);
  const int2 rr = paged_rows(a.c, b);
  const int32_t rows = rr.y - rr.x, t0 = len - rows;
  const uint32_t per = 2 * a.toks, tiles = k0 < len ? ((uint32_t)rows + per - 1) / per : 0;
  const int32_t k1 = min(k0 + 256, len);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh;
  cluster_sync();
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity)) ok = ok && !fail_sh && wait_mbar(bar, parity);
  };
  float sum = 0.f;
  if (warp == kSumWarps + 2) {
    // A lane has columns lane + 32 e. The next tile's sums are on their way while this one's
    // wait for their place.
    struct Cols {
      uint32_t i;
      int32_t lo[4], hi[4], row[4], full;
      float lse[4];
    };
    // Token of the tile (past any sequence for a column without a row) and head of each column.
    uint32_t tok0[4], head[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
      const uint32_t col = lane + 32 * e, in = col % 64;
      tok0[e] = in < a.toks * a.group ? (col / 64) * a.toks + in / a.group : 1u << 30;
      head[e] = kh * a.group + in % a.group;
    }
    // The first tile from i on that sees a key, or `tiles`.
    auto find = [&](uint32_t i, Cols& x) {
      for (; i < tiles; i++) {
        int32_t ulo = INT32_MAX, uhi = 0, ilo = 0, ihi = INT32_MAX;  // of the union, of the intersection
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const uint32_t tok = i * per + tok0[e];
          int2 keys = make_int2(0, 0);
          x.row[e] = -1;
          if (tok < (uint32_t)rows) {
            x.row[e] = rr.x + (int32_t)tok;
            keys = paged_keys(a.m, x.row[e], t0 + (int32_t)tok, len);
          }
          x.lo[e] = keys.x, x.hi[e] = keys.y;
          if (keys.x < keys.y) {
            ulo = min(ulo, keys.x);
            uhi = max(uhi, keys.y);
          }
          ilo = max(ilo, keys.x < keys.y ? keys.x : INT32_MAX);
          ihi = min(ihi, keys.y);
        }
        ulo = __reduce_min_sync(0xffffffffu, ulo);
        uhi = __reduce_max_sync(0xffffffffu, uhi);
        if (ulo >= k1 || uhi <= k0) continue;
        x.full = __reduce_max_sync(0xffffffffu, ilo) <= k0 && __reduce_min_sync(0xffffffffu, ihi) >= k0 + 256;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++)
          x.lse[e] = x.row[e] < 0 ? -INFINITY
                                  : __ldg(a.lse + (uint64_t)x.row[e] * a.p.n_heads + head[e]);
        break;
      }
      x.i = i;
    };
    Cols now, next;
    // Under a causal mask alone the first rows see only earlier keys.
    find(!a.m.last && k0 > t0 ? (uint32_t)(k0 - t0) / per : 0, now);
    for (uint32_t n = 0;; n++) {
      const uint32_t ms = n % NM;
      if (now.i < tiles) find(now.i + 1, next);
      if (n >= NM) wait(&m_empty[ms], (n / NM - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      WeighMeta& m = meta[ms];
      if (now.i < tiles) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const uint32_t col = lane + 32 * e;
          m.lse2[col] = log2_sum(now.lse[e]);
          m.lo[col] = now.lo[e];
          m.hi[col] = now.hi[e];
          if (GENERAL) {
            m.t[col] = (float)(t0 + now.row[e] - rr.x);
            m.slope[col] = a.m.slopes ? __ldg(a.m.slopes + head[e]) * kLog2e : 0.f;
          }
        }
      }
      if (lane == 0) {
        m.tile = now.i < tiles ? (int32_t)now.i : -1;
        m.full = now.full;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&m_full[ms]);
      if (now.i >= tiles) break;
      now = next;
    }
  } else if (warp == kSumWarps) {
    // The keys of this CTA, 8 of a page at a time (pages past the length read zeros), then queries.
    if (tiles) {
      if (lane == 0) mbar_arrive_expect_tx(&k_full, G::kK);
      __syncwarp();
      if (lane < 16) {
        const int32_t key = k0 + (int32_t)(rank * 128 + 8 * lane);
        const int32_t page = key < len ? paged_page(a.c, b, key) : -1;
        tma_load_5d(smem_u32(smem_k) + lane * G::kGroup, &kmap, key & (int32_t)((1u << a.c.shift) - 1), 0, (int)kh,
                    page < 0 ? (int32_t)a.c.n_pages : page, smem_u32(&k_full));
      }
      __syncwarp();
    }
    uint32_t n = 0;
    for (;; n++) {
      const uint32_t ms = n % NM, st = n % NS;
      wait(&m_full[ms], (n / NM) & 1);
      ok = __all_sync(0xffffffffu, ok);
      const int32_t tile = ok ? meta[ms].tile : -1;
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&m_empty[ms]);
      if (tile < 0) break;
      if (n >= NS) wait(&q_empty[st], (n / NS - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&q_full[st], 2 * (D / 64) * a.toks * a.group * 128);
      __syncwarp();
      if (lane < D / 64)  // (64 elements, head of the group, token, chunk, KV head)
        tma_load_5d(smem_u32(smem_q) + st * G::kQ + lane * 8192, &qmap, 0, rr.x + tile * (int32_t)per + (int32_t)(rank * a.toks),
                    (int)lane, (int)kh, in_cta(&q_full[st], 0));
    }
    if (!ok && lane == 0) fail_sh = 1;
    if (tiles) (void)wait_mbar(&k_full, 0);
    if (rank == 0) {  // every load of both CTAs lands before they part
      for (uint32_t i = n > NS ? n - NS : 0; i < n; i++) (void)wait_mbar(&q_full[i % NS], (i / NS) & 1);
    }
  } else if (warp == kSumWarps + 1) {
    const uint32_t lead = rank == 0 ? elect_one() : 0;
    if (tiles && rank == 0) wait(&k_there, 0);
    ok = __all_sync(0xffffffffu, ok);
    // Whether there is an n-th tile, and it can be issued.
    auto ready = [&](uint32_t n) -> bool {
      wait(&m_full[n % NM], (n / NM) & 1);
      ok = __all_sync(0xffffffffu, ok);
      const bool more = __all_sync(0xffffffffu, ok && meta[n % NM].tile >= 0);
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&m_empty[n % NM]);
      if (!more || rank != 0) return more;
      if (n >= NB) wait(&s_empty[n % NB], (n / NB - 1) & 1);
      wait(&q_full[n % NS], (n / NS) & 1);
      return ok = __all_sync(0xffffffffu, ok);
    };
    bool more = ready(0);
    for (uint32_t n = 0; more; n++) {
      if (rank != 0) {
        more = ready(n + 1);
        continue;
      }
      tc_fence_after();
      const uint32_t b_lo = desc_lo(smem_u32(smem_q) + n % NS * G::kQ, 16), d = tmem + n % NB * 128;
      // The waits for the next tile pass while the first half of this one's products is at work.
#pragma unroll
      for (uint32_t kk = 0; kk < D / 16; kk++) {
        if (kk == D / 32) more = ready(n + 1);
        mma2_ts(lead, d, tmem + G::kTK + kk * 8, b_lo + (kk / 4) * 512 + (kk % 4) * 2, desc_hi(1024), idesc16<T>(128, false),
                kk != 0);
      }
      commit2(lead, &q_empty[n % NS]);
      commit2(lead, &s_full[n % NB]);
    }
    if (!ok && lane == 0) {
      fail_sh = 1;
      report_timeout(a.c.err);
    }
    if (rank == 0) {
      commit_own(lead, &drained);
      (void)wait_mbar(&drained, 0);
    }
    __syncwarp();
  } else {
    // Warpgroup wg: columns 32 wg to 32 wg + 31 of every tile.
    const uint32_t wg = warp >> 2, lanes = ((warp & 3) * 32) << 16, kl = tid & 127;
    const int32_t key = k0 + (int32_t)(rank * 128 + kl);
    const float sl = a.m.scale * kLog2e, cap = a.m.cap, pre = GENERAL && cap > 0.f ? a.m.scale / cap : 0.f;
    if (tiles) {  // the keys into tensor memory, a quarter of head_dim each
      wait(&k_full, 0);
      ok = __all_sync(0xffffffffu, ok);
      uint32_t r[D / 8];
#pragma unroll
      for (uint32_t u = 0; u < D / 32; u++) {
        const uint32_t c = wg * (D / 32) + u;  // 16 bytes of the row
        const uint4 x = *reinterpret_cast<const uint4*>(smem_k + kl / 8 * G::kGroup + c / 8 * 1024 + kl % 8 * 128 + ((c % 8 ^ kl % 8) << 4));
        r[4 * u] = x.x, r[4 * u + 1] = x.y, r[4 * u + 2] = x.z, r[4 * u + 3] = x.w;
      }
      tm_st<D / 8>(tmem + lanes + G::kTK + wg * (D / 8), r);
      tm_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(in_cta(&k_there, 0), false);
    }
    for (uint32_t n = 0;; n++) {
      const uint32_t ms = n % NM, buf = n % NB;
      wait(&m_full[ms], (n / NM) & 1);
      ok = __all_sync(0xffffffffu, ok);
      const WeighMeta& m = meta[ms];
      if (!ok || m.tile < 0) break;
      wait(&s_full[buf], (n / NB) & 1);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      float s[32];
      uint32_t* r = reinterpret_cast<uint32_t*>(s);
      tm_ld32(tmem + lanes + buf * 128 + wg * 32, r);
      tm_wait_ld<32>(r);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(in_cta(&s_empty[buf], 0), false);
      float2 acc[2] = {{0.f, 0.f}, {0.f, 0.f}};
      const bool full = m.full;
#pragma unroll
      for (uint32_t c = 0; c < 32; c += 4) {
        const uint32_t col = wg * 32 + c;
        const float4 z = *reinterpret_cast<const float4*>(&m.lse2[col]);
        if constexpr (GENERAL) {
          const float4 t = *reinterpret_cast<const float4*>(&m.t[col]);
          const float4 w = *reinterpret_cast<const float4*>(&m.slope[col]);
          const float ts[4] = {t.x, t.y, t.z, t.w}, ws[4] = {w.x, w.y, w.z, w.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float v = cap > 0.f ? cap * kLog2e * tanh_(s[c + e] * pre) : s[c + e] * sl;
            s[c + e] = ex2(fmaf(-ws[e], fabsf(ts[e] - (float)key), v) - zs[e]);
          }
        } else {
          const float2 v0 = fma2(make_float2(s[c], s[c + 1]), make_float2(sl, sl), make_float2(-z.x, -z.y));
          const float2 v1 = fma2(make_float2(s[c + 2], s[c + 3]), make_float2(sl, sl), make_float2(-z.z, -z.w));
          s[c] = ex2(v0.x), s[c + 1] = ex2(v0.y), s[c + 2] = ex2(v1.x), s[c + 3] = ex2(v1.y);
        }
        if (!full) {
          const int4 lo = *reinterpret_cast<const int4*>(&m.lo[col]), hi = *reinterpret_cast<const int4*>(&m.hi[col]);
          if (key < lo.x || key >= hi.x) s[c] = 0.f;
          if (key < lo.y || key >= hi.y) s[c + 1] = 0.f;
          if (key < lo.z || key >= hi.z) s[c + 2] = 0.f;
          if (key < lo.w || key >= hi.w) s[c + 3] = 0.f;
        }
        acc[0] = add2(acc[0], make_float2(s[c], s[c + 1]));
        acc[1] = add2(acc[1], make_float2(s[c + 2], s[c + 3]));
      }
      acc[0] = add2(acc[0], acc[1]);
      sum += acc[0].x + acc[0].y;
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&m_empty[ms]);
    }
    if (!ok && lane == 0) fail_sh = 1;
    if (wg) part_sh[wg - 1][kl] = sum;
    bar_sync(1, kSumWarps * 32);
    if (wg == 0 && key < len)
      put_weight(a, b, kh, key, len - rows, (sum + part_sh[0][kl]) + (part_sh[1][kl] + part_sh[2][kl]));
  }
  __syncwarp();
  cluster_sync();  // nothing of one CTA is used by the other after this
  if (warp == kSumWarps + 1) tmem_dealloc2<512>(tmem);
}

// Queries as (64 elements, head of the group, token, chunk of 64, KV head): a box is one chunk
// of half a query tile.
int query_map(CUtensorMap* map, const snl_paged_cache& c, const snl_paged_batch& b, const snl_paged_attn_p& p, const void* q,
              uint32_t group, uint32_t toks) {
  PFN_cuTensorMapEncodeTiled enc = tensor_map_encoder();
  if (!enc) return fail(SNL_E_CUDA, "paged cache: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[5] = {64, group, b.n_rows, c.head_dim / 64, c.n_kv};
  const cuuint64_t str[4] = {group > 1 ? p.q_head * 2 : 128, b.n_rows > 1 ? p.q_row * 2 : 128, 128,
                             c.n_kv > 1 ? p.q_head * group * 2 : 128};
  const cuuint32_t box[5] = {64, group, toks, 1, 1}, one[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, c.type == SNL_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                         const_cast<void*>(q), dims, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SNL_OK : fail(SNL_E_INVALID, "paged cache: the strides of q do not fit a tensor map");
}

template <typename T, int D>
int go_weigh(const snl_paged_cache& c, const snl_paged_batch& b, const WeighArgs& a, cudaStream_t s) {
  // Few rows a sequence: the keys are read once and the products are few. From about 3 rows on
  // the tensor cores' passes are the shorter ones.
  if (b.n_rows <= 2 * (uint64_t)b.n_seqs) {
    const uint32_t per = kWeighWarps * kWeighGroups * 8;
    SNL_PDL_LAUNCH("weigh_rows_kernel", (weigh_rows_kernel<T, D>), dim3((a.c.max_len + per - 1) / per, c.n_kv, b.n_seqs),
                   dim3(kWeighWarps * 32), (size_t)0, s, a);
    return SNL_OK;
  }
  CUtensorMap km, qm;
  SNL_TRY(page_map(&km, c, c.k, 8, D / 64));
  SNL_TRY(query_map(&qm, c, b, a.p, a.q, a.group, a.toks));
  const uint64_t grid = 2ull * c.n_kv * b.n_seqs * ((a.c.max_len + 255) / 256);
  if (grid > 0x7fffffffull) return fail(SNL_E_UNSUPPORTED, "snl_paged_weigh: too many keys");
  auto go = [&](auto kern, bool& done) -> int {
    if (!done) SNL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)WeighGeo<D>::kSmem));
    done = true;
    SNL_PDL_LAUNCH("weigh_tile_kernel", kern, dim3((unsigned)grid), dim3(kWeighThreads), (size_t)WeighGeo<D>::kSmem, s, a, km, qm);
    return SNL_OK;
  };
  static bool attr[2][64] = {};
  bool none = false;
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64, general = a.m.cap > 0.f || a.m.slopes;
  return general ? go(weigh_tile_kernel<T, D, true>, known ? attr[1][dev] : none)
                 : go(weigh_tile_kernel<T, D, false>, known ? attr[0][dev] : none);
}

}  // namespace
}  // namespace snl

using namespace snl;

extern "C" int snl_paged_weigh(const snl_paged_cache* c, const snl_paged_batch* b, const snl_paged_attn_p* p,
                               const void* q, const float* lse, float decay, void* stream) {
  const std::string w = "snl_paged_weigh";
  WeighArgs a{};
  SNL_TRY(paged_check("snl_paged_weigh", c, b, &a.c));
  if (!p || (b->n_rows && (!q || !lse))) return fail(SNL_E_INVALID, w + ": null argument");
  SNL_TRY(paged_check_attn("snl_paged_weigh", *c, *b, p, &a.m));
  if (!c->weight) return fail(SNL_E_INVALID, w + ": the cache has no weights");
  if (!(decay >= 0.f) || decay > 3e38f) return fail(SNL_E_INVALID, w + ": decay must be finite and not negative");
  if (!paged_aligned(q)) return fail(SNL_E_INVALID, w + ": q rows must be aligned to 16 bytes");
  if (b->n_seqs == 0 || a.c.max_len == 0) return SNL_OK;
  SNL_TRY(paged_error_word(&a.c.err));
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.lse = lse;
  a.decay = decay;
  a.group = p->n_heads / c->n_kv;
  a.toks = 64 / a.group;
  const cudaStream_t s = (cudaStream_t)stream;
  if (c->type == SNL_T_F16) return c->head_dim == 256 ? go_weigh<__half, 256>(*c, *b, a, s) : go_weigh<__half, 128>(*c, *b, a, s);
  return c->head_dim == 256 ? go_weigh<__nv_bfloat16, 256>(*c, *b, a, s) : go_weigh<__nv_bfloat16, 128>(*c, *b, a, s);
}
