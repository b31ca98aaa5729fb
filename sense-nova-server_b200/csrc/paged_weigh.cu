// Accumulated attention weights of the paged cache's slots (snl_paged_weigh).
#include <algorithm>
#include <string>

#include "paged_rows.cuh"

namespace snl {
namespace {

struct WeighArgs {
  PagedView c;
  PagedMask m;
  snl_paged_attn_p p;
  const uint16_t* q;
  const float* lse;
  float decay;
  uint32_t group, toks;  // query heads per KV head; tokens of half a query tile (32 / group, at least 1)
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

template <int D>
struct WeighRowGeo {
  static constexpr uint32_t kStage = D * 16;  // 8 keys
  static constexpr uint32_t kStages = D == 256 ? 3 : 6, kPerSm = 2;  // a group's chain of steps is long: two CTAs an SM
  static constexpr uint32_t kSmem = kRowWarps * kStages * kStage;
};

// Where a walk over the blocks of (KV head, sequence) stands.
struct WeighWalk {
  uint64_t left;
  uint32_t kh, b, blk, end;
  int32_t len, lo, hi;  // keys that some row sees
  int2 rows;
};
__device__ __forceinline__ void enter_seq(const WeighArgs& a, WeighWalk& w) {
  w.len = paged_len(a.c, w.b);
  w.rows = paged_rows(a.c, w.b);
  w.end = ((uint32_t)w.len + kBlock - 1) / kBlock;
  w.lo = INT32_MAX, w.hi = 0;
  for (int32_t r = w.rows.x; r < w.rows.y; r++) {
    const int2 keys = paged_keys(a.m, r, w.len - (w.rows.y - r), w.len);
    if (keys.x < keys.y) w.lo = min(w.lo, keys.x), w.hi = max(w.hi, keys.y);
  }
}
__device__ __forceinline__ void next_block(const WeighArgs& a, WeighWalk& w) {
  w.left--;
  w.blk++;
  while (w.left && w.blk >= w.end) {
    if (++w.b == a.c.n_seqs) w.b = 0, w.kh++;
    enter_seq(a, w);
    w.blk = 0;
  }
}

// The blocks of 64 keys of all (KV head, sequence) pairs form one line that is cut into equal
// shares, one for each CTA. A warp takes 8 keys of each block through its own ring of TMA
// boxes: S = Q K^T on m16n8k16 with the heads of two rows as the 16 rows, so a key's sum over
// heads and rows is one over the lanes of its column; its old weights come with its keys. 8 tokens
// over up to 16384 keys: 31 us (142 MB, 4.6 TB/s, 0.71 of a copy's rate: the chain of a group's
// steps, about 2500 cycles, not the bytes; 35 with intervals and scale anew for each group, half as
// much again with one CTA an SM, twice with products on the FMA units).
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32, WeighRowGeo<D>::kPerSm)
    weigh_rows_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ CUtensorMap kmap) {
  using G = WeighRowGeo<D>;
  constexpr uint32_t NS = G::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[kRowWarps][NS];
  __shared__ __align__(16) float old_sh[kRowWarps][NS][8];  // the weights of a stage's keys, and their page
  __shared__ int32_t page_sh[kRowWarps][NS];
  __shared__ uint32_t scan_sh[kRowWarps], found_sh[2];
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

  // Blocks before each thread's sequences, this CTA's share, and the sequence that it starts in.
  const uint32_t per = (a.c.n_seqs + kRowWarps * 32 - 1) / (kRowWarps * 32), b0 = min(tid * per, a.c.n_seqs),
                 b1 = min(b0 + per, a.c.n_seqs);
  auto blocks = [&](uint32_t b) { return ((uint32_t)paged_len(a.c, b) + kBlock - 1) / kBlock; };
  uint32_t mine = 0;
  for (uint32_t b = b0; b < b1; b++) mine += blocks(b);
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= (uint32_t)o) upto += v;
  }
  if (lane == 31) scan_sh[warp] = upto;
  __syncthreads();
  uint32_t total = 0;
  for (uint32_t i = 0; i < kRowWarps; i++) {
    if (i < warp) upto += scan_sh[i];
    total += scan_sh[i];
  }
  const uint64_t all = (uint64_t)total * a.c.n_kv, share = (all + gridDim.x - 1) / gridDim.x, g0 = blockIdx.x * share;
  if (g0 >= all) return;
  const uint64_t g1 = min(g0 + share, all);
  {
    uint32_t off = (uint32_t)(g0 % total);
    if (off >= upto - mine && off < upto) {
      off -= upto - mine;
      uint32_t b = b0;
      for (;; b++) {
        const uint32_t n = blocks(b);
        if (off < n) break;
        off -= n;
      }
      found_sh[0] = b;
      found_sh[1] = off;
    }
  }
  __syncthreads();
  WeighWalk now;
  now.left = g1 - g0;
  now.kh = (uint32_t)(g0 / total);
  now.b = found_sh[0];
  enter_seq(a, now);
  now.blk = found_sh[1];
  WeighWalk ahead = now;  // of the loads

  const uint32_t ring = smem_u32(smem) + warp * NS * G::kStage;
  int32_t pages = -1;  // of this warp's keys in 32 blocks from `base` on, one a lane
  uint32_t base = 0xFFFFFFFFu, pseq = 0xFFFFFFFFu, issued = 0, taken = 0;
  auto active = [&](const WeighWalk& w) {
    const int32_t key = (int32_t)(w.blk * kBlock + warp * 8);
    return key + 8 > w.lo && key < w.hi;
  };
  auto issue = [&] {  // the next group that this warp has to read, if any
    while (ahead.left) {
      const bool use = active(ahead);
      if (use) {
        if (pseq != ahead.b || ahead.blk - base >= 32) {
          pseq = ahead.b;
          base = ahead.blk;
          const uint32_t key = (base + lane) * kBlock + warp * 8;
          pages = (int32_t)key < ahead.len ? paged_page(a.c, ahead.b, key) : -1;
        }
        const int32_t page = __shfl_sync(0xffffffffu, pages, ahead.blk - base);
        if (lane == 0) {
          const uint32_t st = issued % NS;
          const bool old = page >= 0 && a.decay != 0.f;
          page_sh[warp][st] = page;
          mbar_arrive_expect_tx(&bars[warp][st], G::kStage + (old ? 32 : 0));
          if (old)
            bulk_g2s_plain(old_sh[warp][st], a.c.weight + paged_weight_at(a.c, page, ahead.kh, ahead.blk * kBlock + warp * 8), 32,
                           &bars[warp][st]);
          tma_group(ring + st * G::kStage, &kmap, (int)((ahead.blk * kBlock + warp * 8) & ((1u << a.c.shift) - 1)),
                    (int)ahead.kh, page < 0 ? (int)a.c.n_pages : page, &bars[warp][st]);
        }
        issued++;
      }
      next_block(a, ahead);
      if (use) return;
    }
  };
  for (uint32_t s = 0; s < NS; s++) issue();

  const uint32_t g = lane >> 2, t = lane & 3;
  const float cap = a.m.cap, sl = a.m.scale * kLog2e, pre = cap > 0.f ? a.m.scale / cap : 0.f;
  bool ok = true, fresh = true;
  uint32_t q[D / 16][4];
  float z[2], slope = 0.f;
  int2 keys[2];    // what a row sees, of its keys from the lane's first key of block 0 on
  float gap[2];    // from that key to the row's own slot
  auto load_rows = [&](int32_t r0) {  // rows r0 and r0 + 1: this lane's head g of each
    const uint32_t head = now.kh * a.group + g;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const bool there = g < a.group && r0 + e < now.rows.y;
      const uint16_t* s = a.q + (uint64_t)(r0 + e) * a.p.q_row + (uint64_t)head * a.p.q_head + 2 * t;
#pragma unroll
      for (int c = 0; c < D / 16; c++) {
        q[c][e] = there ? *reinterpret_cast<const uint32_t*>(s + 16 * c) : 0;
        q[c][2 + e] = there ? *reinterpret_cast<const uint32_t*>(s + 16 * c + 8) : 0;
      }
      z[e] = there ? log2_sum(__ldg(a.lse + (uint64_t)(r0 + e) * a.p.n_heads + head)) : INFINITY;
      const int32_t pos = now.len - (now.rows.y - (r0 + e)), k0 = (int32_t)(warp * 8 + 2 * t);
      keys[e] = there ? paged_keys(a.m, r0 + e, pos, now.len) : make_int2(0, 0);
      keys[e].x -= k0, keys[e].y -= k0;
      gap[e] = (float)(pos - k0);
    }
    slope = a.m.slopes && g < a.group ? __ldg(a.m.slopes + head) * kLog2e : 0.f;
  };
  while (now.left) {
    if (fresh) load_rows(now.rows.x);
    fresh = false;
    const int32_t key0 = (int32_t)(now.blk * kBlock + warp * 8), key = key0 + 2 * (int32_t)t;
    if (key0 < now.len) {
      // The old weights of the lane's two keys come with the keys, or alone where no row sees them.
      const int32_t old_len = now.len - (now.rows.y - now.rows.x);
      const bool seen = active(now);
      int32_t page = seen ? 0 : paged_page(a.c, now.b, key0);
      float2 w = make_float2(0.f, 0.f);
      auto slot = [&] { return reinterpret_cast<float2*>(a.c.weight + paged_weight_at(a.c, page, now.kh, key)); };
      if (!seen && g == 0 && page >= 0) w = *slot();
      float sum0 = 0.f, sum1 = 0.f;
      if (seen) {
        const uint32_t st = taken % NS, box = ring + st * G::kStage;
        ok = __all_sync(0xffffffffu, ok && wait_mbar(&bars[warp][st], (taken / NS) & 1));
        taken++;
        w = *reinterpret_cast<const float2*>(&old_sh[warp][st][2 * t]);
        page = page_sh[warp][st];
        for (int32_t r0 = now.rows.x; r0 < now.rows.y; r0 += 2) {
          if (now.rows.y - now.rows.x > 2) load_rows(r0);  // a sequence of more rows than most
          float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (uint32_t c = 0; c < D / 32; c++) {
            uint32_t kb[4];
            ldsm4(kb, box_at(box, c, lane));
            mma_k16<T>(s0, q[2 * c][0], q[2 * c][1], q[2 * c][2], q[2 * c][3], kb[0], kb[1]);
            mma_k16<T>(s1, q[2 * c + 1][0], q[2 * c + 1][1], q[2 * c + 1][2], q[2 * c + 1][3], kb[2], kb[3]);
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {  // row r0 + e / 2, key + e % 2
            const int32_t k = (int32_t)(now.blk * kBlock) + e % 2;
            const float s = s0[e] + s1[e];
            float x = cap > 0.f ? fmaf(cap * kLog2e, tanh_(s * pre), -z[e / 2]) : fmaf(s, sl, -z[e / 2]);
            if (a.m.slopes) x = fmaf(-slope, fabsf(gap[e / 2] - (float)k), x);
            const float p = k >= keys[e / 2].x && k < keys[e / 2].y ? ex2(x) : 0.f;
            if (e % 2) sum1 += p;
            else sum0 += p;
          }
        }
        fence_proxy_async_smem();  // the stage was read; the next box is written to it after that
        __syncwarp();
        issue();
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, o);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
      }
      if (g == 0 && page >= 0) {
        w.x = a.decay != 0.f && key < old_len ? fmaf(w.x, a.decay, sum0) : sum0;
        w.y = a.decay != 0.f && key + 1 < old_len ? fmaf(w.y, a.decay, sum1) : sum1;
        if (key + 1 < now.len) *slot() = w;
        else if (key < now.len) slot()->x = w.x;
      }
    }
    const uint32_t b = now.b, kh = now.kh;
    next_block(a, now);
    fresh = now.b != b || now.kh != kh;
  }
  if (!ok) {
    // A wait gave up: this warp's boxes still in flight land before the CTA ends.
    if (lane == 0) report_timeout(a.c.err);
    for (uint32_t i = issued > NS ? issued - NS : 0; i < issued; i++) (void)wait_mbar(&bars[warp][i % NS], (i / NS) & 1);
  }
}

// ---- many rows: S^T = K Q^T on the tensor cores ---------------------------------------------

// Shared memory of one CTA: stages of half a query tile [chunk][32 rows][128 bytes], the last
// four of them in the place of its 128 keys [8-key group][64-element chunk][8 keys][128 bytes],
// which are there first and move to tensor memory. Tensor memory, half of an SM's: two tiles of
// 128 keys x 64 (token, head) rows, and from column 128 the keys, the products' A operand.
// Two CTAs share an SM: the sums' latencies of one pass beside the other's products.
template <int D>
struct WeighGeo {
  static constexpr uint32_t kK = 128 * D * 2, kGroup = D * 16;
  static constexpr uint32_t kQ = 32 * D * 2;
  static constexpr uint32_t kStages = 6, kMeta = 8, kBufs = 2, kTK = 128;
  static constexpr uint32_t kSmem = D == 256 ? 2 * kQ + kK : 80 * 1024;  // at most two CTAs an SM
};
constexpr uint32_t kSumWarps = 8, kWeighThreads = (kSumWarps + 3) * 32, kCols = 64;

// What the sums need of a query tile's 64 rows (read 16 bytes at a time).
struct alignas(16) WeighMeta {
  float lse2[kCols], t[kCols], slope[kCols];
  int32_t lo[kCols], hi[kCols];
  int32_t tile;  // -1: no more tiles
  int32_t full;  // every row sees every key of the cluster
};

// A cluster = (256 keys of a sequence and KV head), a CTA 128 of them, thread = key: the
// scores of a query tile come with a key's row in one lane of tensor memory, so its sum over
// the rows needs no exchange, and its order is fixed. The last warp lists the query tiles that
// see the keys, with what each row needs; one loads their queries by TMA, one of the first CTA
// issues the products. 2048 rows of 16 heads over 8192 keys: 152 us (790 TFLOP/s), the tensor
// pipe active 41% and the special-function unit 42% of the time: both wait on the hand-over
// between them, and 128 clusters are 1.7 for each pair of SMs.
template <typename T, int D, bool GENERAL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWeighThreads, 2)
    weigh_tile_kernel(const __grid_constant__ WeighArgs a, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap qmap) {
  using G = WeighGeo<D>;
  constexpr uint32_t NS = G::kStages, NM = G::kMeta, NB = G::kBufs;
  extern __shared__ __align__(1024) uint8_t smem_q[];
  uint8_t* smem_k = smem_q + 2 * G::kQ;
  __shared__ WeighMeta meta[NM];
  __shared__ uint64_t k_full, q_full[NS], q_empty[NS], m_full[NM], m_empty[NM], s_full[G::kBufs], s_empty[G::kBufs], k_there, k_moved, drained;
  __shared__ uint32_t tmem_sh;
  __shared__ float part_sh[128];
  __shared__ volatile int fail_sh;
  pdl_trigger();
  const uint32_t tid = threadIdx.x, warp = same_in_warp(tid >> 5), lane = tid & 31, rank = same_in_warp(cluster_rank());
  const uint32_t cl = blockIdx.x / 2, kh = cl % a.c.n_kv, b = cl / a.c.n_kv % a.c.n_seqs, kt = cl / a.c.n_kv / a.c.n_seqs;
  if (smem_u32(smem_q) & 1023) {  // the swizzle needs it; the same for every CTA
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
    mbar_init(&k_moved, kSumWarps);
    mbar_init(&drained, 1);
    fail_sh = 0;
    fence_mbar_init();
  }
  if (warp == kSumWarps + 1) tmem_alloc2<256>(&tmem_sh);
  pdl_wait();
  const int32_t len = paged_len(a.c, b), k0 = (int32_t)(kt * 256);
  const int2 rr = paged_rows(a.c, b);
  const int32_t rows = rr.y - rr.x, t0 = len - rows;
  // A half tile is toks whole tokens; of more than 32 heads, half of one token's.
  const bool wide = a.group > 32;
  const uint32_t per = wide ? 1 : 2 * a.toks, tiles = k0 < len ? ((uint32_t)rows + per - 1) / per : 0;
  const int32_t k1 = min(k0 + 256, len);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = same_in_warp(tmem_sh);
  cluster_sync();
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity)) ok = ok && !fail_sh && wait_mbar(bar, parity);
  };
  float sum = 0.f;
  if (warp == kSumWarps + 2) {
    // A lane has column `lane` of both halves. The next tile's sums are on their way while this one's
    // wait for their place.
    struct Cols {
      uint32_t i;
      int32_t lo[2], hi[2], row[2], full;
      float lse[2];
    };
    // Token of the tile (past any sequence for a column without a row) and head of each column.
    uint32_t tok0[2], head[2];
#pragma unroll
    for (uint32_t e = 0; e < 2; e++) {
      if (wide) {
        tok0[e] = e * 32 + lane < a.group ? 0 : 1u << 30;
        head[e] = kh * a.group + e * 32 + lane;
      } else {
        tok0[e] = lane < a.toks * a.group ? e * a.toks + lane / a.group : 1u << 30;
        head[e] = kh * a.group + lane % a.group;
      }
    }
    // The first tile from i on that sees a key, or `tiles`.
    auto find = [&](uint32_t i, Cols& x) {
      for (; i < tiles; i++) {
        int32_t ulo = INT32_MAX, uhi = 0, ilo = 0, ihi = INT32_MAX;  // of the union, of the intersection
#pragma unroll
        for (uint32_t e = 0; e < 2; e++) {
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
        for (uint32_t e = 0; e < 2; e++)
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
        for (uint32_t e = 0; e < 2; e++) {
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
      if (n == 2) wait(&k_moved, 0);  // the stages from here on are the keys' place
      if (n >= NS) wait(&q_empty[st], (n / NS - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&q_full[st], 2 * (D / 64) * (wide ? 32 : a.toks * a.group) * 128);
      __syncwarp();
      if (lane < D / 64)  // (64 elements, head of the group, token, chunk, KV head)
        tma_query(smem_u32(smem_q) + st * G::kQ + lane * 4096, &qmap, wide ? (int)(rank * 32) : 0,
                  rr.x + tile * (int32_t)per + (wide ? 0 : (int32_t)(rank * a.toks)), (int)lane, (int)kh, in_cta(&q_full[st], 0));
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
      const uint32_t b_lo = __reduce_max_sync(0xffffffffu, desc_lo(smem_u32(smem_q) + n % NS * G::kQ, 16)),
                     d = __reduce_max_sync(0xffffffffu, tmem + n % NB * kCols);  // into uniform registers
      // The waits for the next tile pass while the first half of this one's products is at work.
#pragma unroll
      for (uint32_t kk = 0; kk < D / 16; kk++) {
        if (kk == D / 32) more = ready(n + 1);
        mma2_ts(lead, d, tmem + G::kTK + kk * 8, b_lo + (kk / 4) * 256 + (kk % 4) * 2, desc_hi(1024), idesc16<T>(kCols, false),
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
    if (tiles) {  // the keys into tensor memory, half of head_dim each
      wait(&k_full, 0);
      ok = __all_sync(0xffffffffu, ok);
#pragma unroll
      for (uint32_t c0 = 0; c0 < D / 16; c0 += 8) {  // 16-byte pieces of the row
        uint32_t r[32];
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) {
          const uint32_t c = wg * (D / 16) + c0 + u;
          const uint4 x = *reinterpret_cast<const uint4*>(smem_k + kl / 8 * G::kGroup + c / 8 * 1024 + kl % 8 * 128 + ((c % 8 ^ kl % 8) << 4));
          r[4 * u] = x.x, r[4 * u + 1] = x.y, r[4 * u + 2] = x.z, r[4 * u + 3] = x.w;
        }
        tm_st32(tmem + lanes + G::kTK + wg * (D / 4) + c0 * 4, r);
      }
      fence_proxy_async_smem();  // the keys' place is read; boxes of queries are written to it next
      tm_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&k_moved);
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
      tm_ld32(tmem + lanes + buf * kCols + wg * 32, r);
      tm_wait_ld<32>(r);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(in_cta(&s_empty[buf], 0), false);
      if (GENERAL && cap > 0.f) {  // mostly all scores are far below the cap, and need no exponentials
        float most = 0.f;
#pragma unroll
        for (uint32_t c = 0; c < 32; c++) most = fmaxf(most, fabsf(s[c]));
        if (__any_sync(0xffffffffu, most * fabsf(pre) >= kTanhNear)) {
#pragma unroll
          for (uint32_t c = 0; c < 32; c++) s[c] = cap * kLog2e * tanh_(s[c] * pre);
        } else {
#pragma unroll
          for (uint32_t c = 0; c < 32; c++) s[c] = cap * kLog2e * tanh_near(s[c] * pre);
        }
      }
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
            const float v = cap > 0.f ? s[c + e] : s[c + e] * sl;
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
    if (wg) part_sh[kl] = sum;
    bar_sync(1, kSumWarps * 32);
    if (wg == 0 && key < len) put_weight(a, b, kh, key, len - rows, sum + part_sh[kl]);
  }
  __syncwarp();
  cluster_sync();  // nothing of one CTA is used by the other after this
  if (warp == kSumWarps + 1) tmem_dealloc2<256>(tmem);
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
  const cuuint32_t box[5] = {64, std::min(group, 32u), toks, 1, 1}, one[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, c.type == SNL_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                         const_cast<void*>(q), dims, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SNL_OK : fail(SNL_E_INVALID, "paged cache: the strides of q do not fit a tensor map");
}

template <typename T, int D>
int go_weigh(const snl_paged_cache& c, const snl_paged_batch& b, const WeighArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64, general = a.m.cap > 0.f || a.m.slopes;
  auto allow = [&](auto kern, bool* done, uint32_t smem) -> int {
    if (known && done[dev]) return SNL_OK;
    SNL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (known) done[dev] = true;
    return SNL_OK;
  };
  // Few rows a sequence on the average: the keys are read once and the products are few (two rows
  // of up to 8 heads are one tile of them). A sequence with many rows beside single tokens passes
  // too, and its queries are loaded again for every 8 keys: 32 tokens over 2048 keys and 34 rows over
  // 8192 of heads of 256 take 724 us, in two calls 30 + 10; at head_dim 128 with 512 and 4096 keys
  // 227, in two calls 14 + 10. A caller that has both kinds gives them a batch each.
  if (a.group <= 8 && b.n_rows <= 2 * (uint64_t)b.n_seqs && (uint64_t)b.n_seqs * (a.c.max_len / kBlock + 1) < (1ull << 31)) {
    static bool attr[64] = {};
    SNL_TRY(allow(weigh_rows_kernel<T, D>, attr, WeighRowGeo<D>::kSmem));
    CUtensorMap km;
    SNL_TRY(page_map(&km, c, c.k, 8, D / 64));
    const uint64_t most = (uint64_t)b.n_seqs * c.n_kv * ((a.c.max_len + kBlock - 1) / kBlock);
    const uint32_t grid = (uint32_t)std::min<uint64_t>(most, (uint64_t)std::max(1, sm_count()) * WeighRowGeo<D>::kPerSm);
    SNL_PDL_LAUNCH("weigh_rows_kernel", (weigh_rows_kernel<T, D>), dim3(grid), dim3(kRowWarps * 32),
                   (size_t)WeighRowGeo<D>::kSmem, s, a, km);
    return SNL_OK;
  }
  CUtensorMap km, qm{};  // no query is loaded for a batch without rows, and no map describes an empty tensor
  SNL_TRY(page_map(&km, c, c.k, 8, D / 64));
  if (b.n_rows) SNL_TRY(query_map(&qm, c, b, a.p, a.q, a.group, a.toks));
  // Clusters past a sequence's length only meet and leave: 8 x 64 rows over 2000 keys take 23 us with
  // that bound, 52 with one of 16384 keys, 310 with 131072.
  const uint64_t grid = 2ull * c.n_kv * b.n_seqs * ((a.c.max_len + 255) / 256);
  if (grid > 0x7fffffffull) return fail(SNL_E_UNSUPPORTED, "snl_paged_weigh: too many keys");
  static bool attr[2][64] = {};
  auto go = [&](auto kern, bool* done) -> int {
    SNL_TRY(allow(kern, done, WeighGeo<D>::kSmem));
    SNL_PDL_LAUNCH("weigh_tile_kernel", kern, dim3((unsigned)grid), dim3(kWeighThreads), (size_t)WeighGeo<D>::kSmem, s, a, km, qm);
    return SNL_OK;
  };
  return general ? go(weigh_tile_kernel<T, D, true>, attr[1]) : go(weigh_tile_kernel<T, D, false>, attr[0]);
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
  if (!paged_aligned(c->weight)) return fail(SNL_E_INVALID, w + ": the weights must be aligned to 16 bytes");
  if (b->n_seqs == 0 || a.c.max_len == 0) return SNL_OK;
  SNL_TRY(paged_error_word(&a.c.err));
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.lse = lse;
  a.decay = decay;
  a.group = p->n_heads / c->n_kv;
  a.toks = std::max(1u, 32 / a.group);
  const cudaStream_t s = (cudaStream_t)stream;
  if (c->type == SNL_T_F16) return c->head_dim == 256 ? go_weigh<__half, 256>(*c, *b, a, s) : go_weigh<__half, 128>(*c, *b, a, s);
  return c->head_dim == 256 ? go_weigh<__nv_bfloat16, 256>(*c, *b, a, s) : go_weigh<__nv_bfloat16, 128>(*c, *b, a, s);
}
