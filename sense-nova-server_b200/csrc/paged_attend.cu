// Attention over the paged cache (snl_paged_attend).
#include <algorithm>
#include <string>

#include "paged_attend.cuh"

namespace snl {
namespace {

// Two CTAs of a cluster work as one (cta_group::2): each holds 128 rows of queries, half of
// every K tile (half of its keys) and half of every V tile (half of head_dim), so each byte
// of the cache is fetched and held once for 256 rows. One CTA's leader thread issues the
// MMAs of both.

// Shared and tensor memory of one CTA. A K or V tile's half is [8-key group][64-element
// chunk][8 keys][128 bytes], 128-byte swizzled (V: 16 keys where the pages hold them); queries
// are [chunk][128 rows][128 bytes]. Tensor memory: the output from column 0, then two score
// tiles, which the probabilities overwrite. At head_dim 256 that is all of an SM's; at 128
// with tiles of 64 keys it is half, and two CTAs share an SM: one's softmax, start and end
// run beside the other's products (6 x 1000 rows: 211 us with tiles of 128 keys and one CTA).
template <int D>
struct Geo {
  static constexpr uint32_t KT = D == 256 ? 128 : 64;  // keys of a tile
  static constexpr uint32_t kPerSm = D == 256 ? 1 : 2;
  static constexpr uint32_t kQ = 128 * D * 2;      // bytes of the queries
  static constexpr uint32_t kTile = KT / 2 * D * 2;  // bytes of half a K tile, of half a V tile
  static constexpr uint32_t kGroupK = D * 16, kGroupV = D * 8;  // bytes of 8 keys
  static constexpr uint32_t kStagesK = D == 256 ? 2 : 4, kStagesV = D == 256 ? 3 : 4;
  static constexpr uint32_t kSmem = kQ + (kStagesK + kStagesV) * kTile;
  static constexpr uint32_t kS = D, kCols = D == 256 ? 512 : 256;
};

// Where a tile of rows lies: sequence, first row, tokens, slot of the first token.
struct TileInfo {
  uint32_t b, row0, toks;
  int32_t t0, len;
};

// Slot s belongs to the last sequence b with start[b] / (2 toks) + b <= s: a sequence has at
// least as many slots as tiles, found without a sum over the batch. One warp.
__device__ __forceinline__ TileInfo find_tile(const AttendArgs& a, uint32_t s, uint32_t lane) {
  const uint32_t per = 2 * a.toks;
  uint32_t lo = 0, hi = a.c.n_seqs;
  while (hi - lo > 32) {
    const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
    const bool le = at < hi && (at == lo || (uint32_t)__ldg(a.c.start + at) / per + at <= s);
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, le));
    const uint32_t below = lo + (max(n, 1u) - 1) * step;
    hi = min(hi, below + step);
    lo = below;
  }
  // Of up to 32 sequences all that is needed is fetched at once.
  const uint32_t at = min(lo + lane, hi - 1);
  const int32_t from = __ldg(a.c.start + at), to = __ldg(a.c.start + at + 1), n_at = __ldg(a.c.len + at);
  const bool le = lo + lane < hi && (lane == 0 || (uint32_t)from / per + at <= s);
  const uint32_t pick = max(__popc(__ballot_sync(0xffffffffu, le)), 1) - 1;
  lo += pick;
  TileInfo w{lo, 0, 0, 0, 0};
  const int2 rr = paged_rows(a.c, __shfl_sync(0xffffffffu, from, pick), __shfl_sync(0xffffffffu, to, pick));
  const int32_t len = paged_length(a.c, __shfl_sync(0xffffffffu, n_at, pick));
  const uint32_t base = (uint32_t)rr.x / per + lo;
  if (s < base) return w;
  const uint32_t off = (s - base) * per;
  if (off >= (uint32_t)(rr.y - rr.x)) return w;
  w.row0 = rr.x + off;
  w.toks = min(per, (uint32_t)(rr.y - rr.x) - off);
  w.len = len;
  w.t0 = w.len - (rr.y - rr.x) + (int32_t)off;
  return w;
}

constexpr uint32_t kSoftWarps = 8;
constexpr uint32_t kAttendThreads = (kSoftWarps + 3) * 32;
constexpr float kRefSlack = 8.f;  // log2 that scores may exceed the reference before O is rescaled

// Softmax in one pass over the keys: with m the reference and l the sum so far, a tile's
// scores s (in units of log2) give P = 2^(s - m), l += sum P, O += P V, and out = O / l. P is
// rounded to the cache's type for the product (2^-11 or 2^-8 of each weight, as V itself is),
// l and O stay in 32 bits.
//
// A cluster = (two tiles of 128 (token, head) rows of one KV head's group, part of the
// keys). Warps 8 and 10 of each CTA load its halves of the K and V tiles by TMA, 8 or 16 keys
// of one page at a time (one box takes about 70 cycles to issue: a single warp for both
// held the MMAs up); warp 9 of the first issues S = Q K^T and O += P V; two warpgroups of each CTA
// turn half of a score tile's columns into probabilities each, thread = row. The maximum
// that the exponentials refer to moves only when a score exceeds it by kRefSlack.
//
// Bound by the products and the hand-over between them and the softmax: 2048 rows of 16 heads of
// 256 over 8192 keys take 232 us called back to back (1040 TFLOP/s; 199 in a short burst), the
// tensor pipe active 66% of the time and the card at its power limit (981 W, 1.79 of 1.965
// GHz). 6 x up to 1000 rows of 32 heads of 128 under a window, documents and a distance bias: 134
// us; a tile of 64 keys takes 1970 cycles of a CTA, 1000 when the softmax warps do nothing, and 15
// tiles a pair of CTAs leave a third of its time to the start and the end (queries and tiles are
// on their way together, gates are loaded ahead of the stores: 146 us without either).
template <typename T, int D, bool GENERAL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kAttendThreads, Geo<D>::kPerSm)
    attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using G = Geo<D>;
  constexpr uint32_t KT = G::KT, NK = G::kStagesK, NV = G::kStagesV;
  extern __shared__ __align__(1024) uint8_t smem_q[];
  __shared__ uint64_t k_full[NK], k_empty[NK], v_full[NV], v_empty[NV], s_full[2], p_ready[2], pv_done[2], v_landed, q_ready, drained;
  __shared__ uint32_t tmem_sh;
  __shared__ TileInfo info_sh;
  __shared__ int32_t lohi[4][kSoftWarps / 2];  // per warp: least and largest lo, least and largest hi
  __shared__ float max_sh[2][2][128];
  __shared__ volatile int fail_sh;
  __shared__ int odd_v;
  pdl_trigger();
  const uint32_t tid = threadIdx.x, warp = same_in_warp(tid >> 5), lane = tid & 31, rank = same_in_warp(cluster_rank());
  const uint32_t kh = (blockIdx.x / 2) % a.c.n_kv, unit = (blockIdx.x / 2) / a.c.n_kv;
  const uint32_t split = unit % a.n_split, slot = a.slots - 1 - unit / a.n_split;
  uint8_t *smem_k = smem_q + G::kQ, *smem_v = smem_k + NK * G::kTile;
  if (smem_u32(smem_q) & 1023) {  // the swizzle needs it; the same for every CTA
    report_timeout(a.c.err);
    return;
  }

  if (tid == 0) {
    for (uint32_t s = 0; s < NK; s++) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (uint32_t s = 0; s < NV; s++) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; s++) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 2 * kSoftWarps);  // the warps of both CTAs
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(&v_landed, 1);
    mbar_init(&q_ready, 2 * kSoftWarps);
    mbar_init(&drained, 1);
    fail_sh = 0;
    odd_v = 0;
    fence_mbar_init();
  }
  __syncwarp();
  cluster_arrive();  // the barriers of this CTA are there
  if (warp == 9) tmem_alloc2<G::kCols>(&tmem_sh);
  pdl_wait();
  if (warp == 8) {
    const TileInfo w = find_tile(a, slot, lane);
    if (lane == 0) info_sh = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = same_in_warp(tmem_sh);
  const TileInfo w = info_sh;  // of the cluster: up to 2 a.toks tokens

  // Row of this thread (both warpgroups hold all 128): token and head, its keys.
  const uint32_t row = tid & 127, tok0 = row / a.group, head = kh * a.group + row % a.group;
  const uint32_t tok = tok0 + rank * a.toks;
  const bool mine = warp < kSoftWarps && tok0 < a.toks, valid = mine && tok < w.toks;
  // The row's interval, and that of the same row of the other CTA: both walk the same tiles.
  const uint32_t tok1 = tok0 + (rank ^ 1) * a.toks, most = w.toks ? w.toks - 1 : 0;
  const uint32_t ra = w.row0 + min(tok, most), rb = w.row0 + min(tok1, most);
  int32_t first0 = 0, first1 = 0, last0 = 0, last1 = 0;
  if (a.m.first && warp < kSoftWarps) first0 = __ldg(a.m.first + ra), first1 = __ldg(a.m.first + rb);
  if (a.m.last && warp < kSoftWarps) last0 = __ldg(a.m.last + ra), last1 = __ldg(a.m.last + rb);
  // Queries into shared memory, the sign of the scale folded in; the first of them are on their
  // way while the rows' keys are looked up, all of them while the first tiles come.
  // 16-byte pieces of a row; loads on their way at once
  constexpr uint32_t per = D / 8, batch = 8, batches = G::kQ / 16 / (batch * kSoftWarps * 32);
  const uint32_t by_group = 65535 / a.group + 1;  // r * by_group >> 16 is r / group: r < 128, group <= 64
  uint4 x[batch];
  auto fetch_q = [&](uint32_t n) {
#pragma unroll
    for (uint32_t i = 0; i < batch; i++) {
      const uint32_t e = tid + (n * batch + i) * kSoftWarps * 32, r = e / per, u = e % per, t0 = r * by_group >> 16, t = t0 + rank * a.toks;
      x[i] = make_uint4(0, 0, 0, 0);
      if (t0 < a.toks && t < w.toks)
        x[i] = __ldg(reinterpret_cast<const uint4*>(a.q + (uint64_t)(w.row0 + t) * a.p.q_row +
                                                    (uint64_t)(kh * a.group + r - t0 * a.group) * a.p.q_head + 8 * u));
    }
  };
  if (warp < kSoftWarps) fetch_q(0);
  int2 keys = make_int2(0, 0);
  if (valid) keys = paged_interval(a.m, first0, last0, w.t0 + (int32_t)tok, w.len);
  if (warp < kSoftWarps / 2) {
    int2 k1 = make_int2(0, 0);
    if (mine && tok1 < w.toks) k1 = paged_interval(a.m, first1, last1, w.t0 + (int32_t)tok1, w.len);
    const bool s0 = keys.x < keys.y, s1 = k1.x < k1.y;
    const int32_t lo0 = min(s0 ? keys.x : INT32_MAX, s1 ? k1.x : INT32_MAX), lo1 = max(s0 ? keys.x : 0, s1 ? k1.x : 0);
    const int32_t hi0 = min(s0 ? keys.y : INT32_MAX, s1 ? k1.y : INT32_MAX), hi1 = max(s0 ? keys.y : 0, s1 ? k1.y : 0);
    const int32_t r0 = __reduce_min_sync(0xffffffffu, lo0), r1 = __reduce_max_sync(0xffffffffu, lo1);
    const int32_t r2 = __reduce_min_sync(0xffffffffu, hi0), r3 = __reduce_max_sync(0xffffffffu, hi1);
    if (lane == 0) {
      lohi[0][warp] = r0;
      lohi[1][warp] = r1;
      lohi[2][warp] = r2;
      lohi[3][warp] = r3;
    }
  }
  const float sl = fmaxf(fabsf(a.m.scale) * kLog2e, 1e-30f);  // not 0: -inf of a masked score has to stay
  cluster_wait();  // the other CTA's barriers are there
  __syncthreads();
  if (warp < kSoftWarps) {
    const uint32_t flip = a.m.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (uint32_t n = 0; n < batches; n++) {
      if (n) fetch_q(n);
#pragma unroll
      for (uint32_t i = 0; i < batch; i++) {
        const uint32_t e = tid + (n * batch + i) * kSoftWarps * 32, r = e / per, u = e % per;
        x[i].x ^= flip, x[i].y ^= flip, x[i].z ^= flip, x[i].w ^= flip;
        *reinterpret_cast<uint4*>(smem_q + (u / 8) * 16384 + r * 128 + ((u % 8 ^ r % 8) << 4)) = x[i];
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) arrive_cluster(in_cta(&q_ready, 0), true);
  }
  int32_t lo0 = lohi[0][0], lo1 = lohi[1][0], hi0 = lohi[2][0], hi1 = lohi[3][0];
#pragma unroll
  for (uint32_t i = 1; i < kSoftWarps / 2; i++) {
    lo0 = min(lo0, lohi[0][i]);
    lo1 = max(lo1, lohi[1][i]);
    hi0 = min(hi0, lohi[2][i]);
    hi1 = max(hi1, lohi[3][i]);
  }
  // Tiles [j0, j0 + nt): what the rows see, cut to this part, from the last one down. The
  // largest scores are mostly near the row itself, above all under a distance bias, whose
  // scores would outgrow the reference at every tile of the other order.
  const int32_t c0 = (int32_t)(split * a.split_len);
  const int32_t beg = max(lo0 == INT32_MAX ? 0 : lo0, c0), end = min(hi1, c0 + (int32_t)a.split_len);
  const uint32_t j0 = same_in_warp(beg < end ? (uint32_t)beg / KT : 0);
  const uint32_t nt = same_in_warp(beg < end ? ((uint32_t)end + KT - 1) / KT - j0 : 0), jl = j0 + nt - 1;
  // Tiles with a key that some row of the cluster does not see.
  auto masked_tile = [&](uint32_t j) { return (int32_t)(j * KT) < lo1 || (int32_t)(j * KT + KT) > hi0; };

  // Results of the softmax warps, used after the loop.
  float l = 0.f, ref = -INFINITY;
  const uint32_t vrun = a.vrun;  // keys of a V box: 8 or 16
  if (warp == 8 || warp == 10) {
    // Lane g loads the g-th run of keys of the tile (K: of this CTA's half). Runs of which no row
    // sees a key, whose pages may be gone, and pages outside the cache come from a page coordinate
    // past the end, which reads zeros.
    const bool is_k = warp == 8;
    const uint32_t run = is_k ? 8 : vrun, lanes = is_k ? KT / 16 : KT / vrun, key0 = (is_k ? rank * (KT / 2) : 0) + lane * run;
    const uint32_t NS = is_k ? NK : NV;
    uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
    auto page_of = [&](uint32_t i) -> int32_t {
      const uint32_t key = (jl - i) * KT + key0;
      int32_t p = -1;
      if (i < nt && lane < lanes && (int32_t)key < end && (int32_t)(key + run) > beg) p = paged_page(a.c, w.b, key);
      return p < 0 ? (int32_t)a.c.n_pages : p;
    };
    int32_t now = page_of(0), next = page_of(1);
    uint32_t st = 0, par = 0, n = 0;
    bool ok = true;
    for (; n < nt; n++) {
      const int32_t later = page_of(n + 2);
      if (n >= NS) ok = __all_sync(0xffffffffu, mbar_try_wait(&empty[st], par ^ 1) || (!fail_sh && wait_mbar(&empty[st], par ^ 1)));
      if (!ok) break;
      if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&full[st], 2 * G::kTile);
      __syncwarp();
      if (lane < lanes)
        tma_load_5d(smem_u32((is_k ? smem_k : smem_v) + st * G::kTile) + lane * run * (is_k ? D * 2 : D), is_k ? &kmap : &vmap,
                    (int)(((jl - n) * KT + key0) & ((1u << a.c.shift) - 1)), is_k ? 0 : (int)(rank * (D / 128)), (int)kh, now,
                    in_cta(&full[st], 0));
      now = next;
      next = later;
      if (++st == NS) st = 0, par ^= 1;
    }
    if (!ok && lane == 0) fail_sh = 1;
    // every load of both CTAs lands before they part, whatever became of its readers
    if (rank == 0)
      for (uint32_t i = n > NS ? n - NS : 0; i < n; i++) (void)wait_mbar(&full[i % NS], (i / NS) & 1);
  } else if (warp == 9) {
    if (rank == 0) {
      const uint32_t lead = elect_one();
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = __all_sync(0xffffffffu, ok && (mbar_try_wait(bar, parity) || (!fail_sh && wait_mbar(bar, parity))));
      };
      const uint32_t q_lo = desc_lo(smem_u32(smem_q), 16), v_hi = desc_hi(vrun == 8 ? G::kGroupV : 1024);
      auto scores = [&](uint32_t i) {
        const uint32_t st = i % NK;
        wait(&k_full[st], (i / NK) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint32_t k_lo = desc_lo(smem_u32(smem_k) + st * G::kTile, 16), d = tmem + G::kS + (i & 1) * KT;
#pragma unroll
        for (uint32_t kk = 0; kk < D / 16; kk++)
          mma2_ss(lead, d, q_lo + (kk / 4) * 1024 + (kk % 4) * 2, desc_hi(1024), k_lo + (kk / 4) * 64 + (kk % 4) * 2,
                  desc_hi(G::kGroupK), idesc16<T>(KT, false), kk != 0);
        commit2(lead, &k_empty[st]);
        commit2(lead, &s_full[i & 1]);
      };
      if (nt) {
        ok = __all_sync(0xffffffffu, wait_cluster(&q_ready, 0));
        if (ok) scores(0);
      }
      for (uint32_t i = 0; ok && i < nt; i++) {
        if (i + 1 < nt) scores(i + 1);
        const uint32_t st = i % NV;
        wait(&v_full[st], (i / NV) & 1);
        if (ok && masked_tile(jl - i)) {  // the warpgroups look through it first
          if (lane < 2) arrive_cluster(in_cta(&v_landed, lane), true);
          ok = __all_sync(0xffffffffu, wait_cluster(&p_ready[i & 1], (i >> 1) & 1));
        } else {
          wait(&p_ready[i & 1], (i >> 1) & 1);
        }
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_lo = desc_lo(smem_u32(smem_v) + st * G::kTile, vrun * 128), p = tmem + G::kS + (i & 1) * KT;
#pragma unroll
        for (uint32_t kk = 0; kk < KT / 16; kk++)
          mma2_ts(lead, tmem, p + kk * 8, v_lo + kk * 2 * (G::kGroupV / 16), v_hi, idesc16<T>(D, true), (i | kk) != 0);
        commit2(lead, &v_empty[st]);
        commit2(lead, &pv_done[i & 1]);
      }
      if (!ok && lane == 0) {
        fail_sh = 1;
        report_timeout(a.c.err);
      }
      commit_own(lead, &drained);  // and every MMA before the tensor memory is given back
      (void)wait_mbar(&drained, 0);
    }
  } else {
    // Half of a tile's columns each: warps w and w + 4 hold the same 32 rows.
    const uint32_t wg = warp >> 2, lanes = ((warp & 3) * 32) << 16;
    const bool live = __any_sync(0xffffffffu, valid);
    const float slope = GENERAL && a.m.slopes && valid ? __ldg(a.m.slopes + head) * kLog2e : 0.f;
    const float cap = a.m.cap, pre = GENERAL && cap > 0.f ? fabsf(a.m.scale / cap) : 0.f;
    const uint32_t ready[2] = {in_cta(&p_ready[0], 0), in_cta(&p_ready[1], 0)};
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!mbar_try_wait(bar, parity)) {
        ok = ok && !fail_sh && wait_mbar(bar, parity);
        if (!ok) fail_sh = 1;
      }
      __syncwarp();
    };
    // Tiles with a key that some row of this warp (one without keys counts) does not see.
    const bool some = keys.x < keys.y;
    const int32_t wlo = __reduce_max_sync(0xffffffffu, some ? keys.x : valid ? INT32_MAX : 0);
    const int32_t whi = __reduce_min_sync(0xffffffffu, some ? keys.y : valid ? 0 : INT32_MAX);
    constexpr uint32_t NC = KT / 2;  // columns of this warp
    uint32_t landed = 0;
    for (uint32_t i = 0; i < nt; i++) {
      const int32_t k0 = (int32_t)((jl - i) * KT + wg * NC);
      const uint32_t tm_s = tmem + lanes + G::kS + (i & 1) * KT;
      float s[NC];
      uint32_t* r = reinterpret_cast<uint32_t*>(s);
      wait(&s_full[i & 1], (i >> 1) & 1);
      tc_fence_after();
      if (live) {
#pragma unroll
        for (uint32_t c = 0; c < NC; c += 32) tm_ld32(tm_s + wg * NC + c, r + c);
        tm_wait_ld<NC>(r);
        if constexpr (GENERAL) {
          const float gap = (float)(w.t0 + (int32_t)tok - k0);
          if (cap > 0.f) {  // mostly all scores are far below the cap, and need no exponentials
            float most = 0.f;
#pragma unroll
            for (uint32_t c = 0; c < NC; c++) most = fmaxf(most, fabsf(s[c]));
            if (__any_sync(0xffffffffu, most * pre >= kTanhNear)) {
#pragma unroll
              for (uint32_t c = 0; c < NC; c++) s[c] = fmaf(-slope, fabsf(gap - (float)c), cap * kLog2e * tanh_(s[c] * pre));
            } else {
#pragma unroll
              for (uint32_t c = 0; c < NC; c++) s[c] = fmaf(-slope, fabsf(gap - (float)c), cap * kLog2e * tanh_near(s[c] * pre));
            }
          } else {
#pragma unroll
            for (uint32_t c = 0; c < NC; c++) s[c] = fmaf(-slope, fabsf(gap - (float)c), s[c] * sl);
          }
        }
        if (k0 < wlo || k0 + (int32_t)NC > whi) {
          const int32_t x0 = keys.x - k0, n = keys.y - keys.x;
#pragma unroll
          for (uint32_t c = 0; c < NC; c++)
            if ((uint32_t)((int32_t)c - x0) >= (uint32_t)n) s[c] = -INFINITY;
        }
        float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (uint32_t c = 4; c < NC; c += 2) m4[(c / 2) & 3] = fmaxf(fmaxf(m4[(c / 2) & 3], s[c]), s[c + 1]);
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if constexpr (!GENERAL) mx *= sl;
        // The tile's maximum from both halves; after this barrier both have read their scores, which
        // the probabilities overwrite.
        max_sh[i & 1][wg][row] = mx;
        bar_sync(1 + (warp & 3), 64);
        mx = fmaxf(mx, max_sh[i & 1][wg ^ 1][row]);
        const float now = mx > ref + kRefSlack ? mx : ref;
        if (i > 0 && __any_sync(0xffffffffu, now != ref)) {
          wait(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1);
          tc_fence_after();
          const float f = now != ref ? ex2(ref - now) : 1.f;
#pragma unroll 1
          for (uint32_t c = wg * (D / 2); c < (wg + 1) * (D / 2); c += 32) {
            uint32_t o[32];
            tm_ld32(tmem + lanes + c, o);
            tm_wait_ld<32>(o);
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tm_st32(tmem + lanes + c, o);
          }
          l *= f;
        }
        ref = now;
        const float zero = now == -INFINITY ? 0.f : now;
        float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (uint32_t c = 0; c < NC; c += 2) {
          float2 p = make_float2(s[c], s[c + 1]);
          p = GENERAL ? make_float2(p.x - zero, p.y - zero) : fma2(p, make_float2(sl, sl), make_float2(-zero, -zero));
          p = make_float2(ex2(p.x), ex2(p.y));
          sum[(c / 2) & 1] = add2(sum[(c / 2) & 1], p);
          r[c / 2] = pack2(p.x, p.y, T());
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tm_st<NC / 2>(tm_s + wg * (NC / 2), r);
        tm_wait_st();
      }
      bool mended = false;
      if (masked_tile(jl - i)) {
        // A row's probability for a key that it does not see is 0, but 0 * NaN is not: values that
        // are not finite leave the tile, and reach the rows that see them at the end.
        ok = __all_sync(0xffffffffu, ok && wait_cluster(&v_landed, landed & 1));
        landed++;
        if (ok) {
          constexpr uint32_t inf2 = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
          uint4* tile = reinterpret_cast<uint4*>(smem_v + (i % NV) * G::kTile);
          bool odd = false;
#pragma unroll 4
          for (uint32_t e = tid; e < G::kTile / 16; e += 256) {
            uint4 x = tile[e];
            const uint32_t b0 = __vcmpeq2(x.x & inf2, inf2), b1 = __vcmpeq2(x.y & inf2, inf2),
                           b2 = __vcmpeq2(x.z & inf2, inf2), b3 = __vcmpeq2(x.w & inf2, inf2);
            if (b0 | b1 | b2 | b3) {
              const int32_t key = (int32_t)((jl - i) * KT + e * 16 / (vrun * D) * vrun + e * 16 % (vrun * 128) / 128);
              odd = odd || (key >= lo0 && key < hi1);
              mended = true;
              tile[e] = make_uint4(x.x & ~b0, x.y & ~b1, x.z & ~b2, x.w & ~b3);
            }
          }
          if (odd) {
            odd_v = 1;
            asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(in_cta(&odd_v, rank ^ 1)) : "memory");
          }
          mended = __any_sync(0xffffffffu, mended);  // seldom: the MMAs read what was written then
          if (mended) fence_proxy_async_smem();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(ready[i & 1], mended);
    }
    if (nt) wait(&pv_done[(nt - 1) & 1], ((nt - 1) >> 1) & 1);
  }
  __syncwarp();
  cluster_sync();  // nothing of one CTA is used by the other after this
  if (warp < kSoftWarps) {
    const uint32_t wg = warp >> 2, lanes = ((warp & 3) * 32) << 16;
    // Sums of both halves; the maxima's memory is free after the barrier above.
    max_sh[0][wg][row] = l;
    bar_sync(1 + (warp & 3), 64);
    tc_fence_after();
    l += max_sh[0][wg ^ 1][row];
    const float fin = ref;
    const bool parts = a.n_split > 1;
    const uint64_t rh = (uint64_t)(w.row0 + tok) * a.p.n_heads + head;
    if (valid && wg == 0) {
      if (parts) a.part_ml[rh * a.n_split + split] = make_float2(fin, l);
      else if (a.lse) a.lse[rh] = l == 0.f ? -INFINITY : ((fin == -INFINITY ? 0.f : fin) + log2f(l)) * (1.f / kLog2e);
    }
    const float inv = parts ? 1.f : l == 0.f ? 0.f : 1.f / l;
    // 32 columns at a time go through the tiles' memory, free now, so that 8 lanes write 32
    // neighbouring elements of a row: from the accumulator's lanes each would write its own row.
    float* turn = reinterpret_cast<float*>(smem_k) + warp * 32 * 36;
    const uint64_t out_at = parts ? (rh * a.n_split + split) * D
                                  : (uint64_t)(w.row0 + tok) * a.p.out_row + (uint64_t)head * a.p.out_head;
    const uint64_t gate_at = (uint64_t)(w.row0 + tok) * a.p.gate_row + (uint64_t)head * a.p.gate_head;
    const uint32_t some_rows = __ballot_sync(0xffffffffu, valid && !(parts && nt == 0));
    // A row without weights is 0 whatever its gate holds, which is not looked at.
    const uint32_t gated_rows = __ballot_sync(0xffffffffu, valid && l != 0.f);
#pragma unroll 1
    for (uint32_t c = wg * (D / 2); some_rows && c < (wg + 1) * (D / 2); c += 32) {
      uint32_t r[32];
      float* o = reinterpret_cast<float*>(r);
      __syncwarp();
      if (nt) {
        tm_ld32(tmem + lanes + c, r);
        tm_wait_ld<32>(r);
      }
      if (odd_v && valid) {
        for (uint32_t j = j0; j < j0 + nt; j++) {
          if (!masked_tile(j)) continue;
          const int32_t k1 = min(min((int32_t)((j + 1) * KT), keys.y), end);
          for (int32_t key = max((int32_t)(j * KT), keys.x); key < k1; key++) {
            const int32_t page = paged_page(a.c, w.b, key);
            if (page < 0) continue;
            const T* v = reinterpret_cast<const T*>(a.c.v + paged_at(a.c, page, kh, key)) + c;
            for (int e = 0; e < 32; e++) {
              const float x = (float)v[e];
              if (!(fabsf(x) < INFINITY))
#pragma unroll
                for (int f = 0; f < 32; f++)
                  if (f == e) o[f] += x;
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        *reinterpret_cast<float4*>(turn + lane * 36 + e) =
            l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
      __syncwarp();
      // Gates are loaded ahead of the stores, which no later load may pass: as many as registers hold.
      auto put = [&](auto gated) {
        constexpr bool with_gate = decltype(gated)::value;
        constexpr uint32_t ahead = !with_gate ? 1 : D == 256 ? 8 : 2;
        uint4 g4[ahead];
#pragma unroll
        for (uint32_t it = 0; it < 8; it++) {
          if (with_gate && it % ahead == 0) {
#pragma unroll
            for (uint32_t i = 0; i < ahead; i++) {
              const uint32_t row = (it + i) * 4 + lane / 8;
              const uint64_t from = __shfl_sync(0xffffffffu, gate_at, row) + c + lane % 8 * 4;
              g4[i] = make_uint4(0, 0, 0, 0);
              if (!(gated_rows >> row & 1)) continue;
              if (a.p.gate_type == SNL_T_F32) {
                g4[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(a.gate) + from));
              } else {
                const uint2 h = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.gate) + from));
                g4[i].x = h.x, g4[i].y = h.y;
              }
            }
          }
          const uint32_t row = it * 4 + lane / 8, col = lane % 8 * 4;
          const uint64_t to = __shfl_sync(0xffffffffu, out_at, row);
          if (!(some_rows >> row & 1)) continue;
          const float4 y = *reinterpret_cast<const float4*>(turn + row * 36 + col);
          float v[4] = {y.x, y.y, y.z, y.w};
          if constexpr (with_gate) {
            float g[4];
            load_as_float<4>(&g4[it % ahead], 0, a.p.gate_type, g);
#pragma unroll
            for (int f = 0; f < 4; f++) v[f] *= sigmoidf_(g[f]);
          } else if (parts) {
            store_from_float<4>(a.part, to + c + col, SNL_T_F32, v);
            continue;
          }
          store_from_float<4>(a.out, to + c + col, a.p.out_type, v);
        }
      };
      if (a.gate && !parts) put(std::true_type());
      else put(std::false_type());
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) tmem_dealloc2<G::kCols>(tmem);
}

// Joins the parts of a row: one warp per (row, head), over the parts that its keys touch, with
// o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m) in the order of the parts.
constexpr uint32_t kWarps = 8;
template <int D>
__global__ void __launch_bounds__(kWarps * 32) join_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int E = D / 32;
  pdl_trigger();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t item = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const uint32_t r = (uint32_t)(item / a.p.n_heads), h = (uint32_t)(item % a.p.n_heads);
  pdl_wait();
  if (r >= a.c.n_rows) return;
  const uint32_t b = paged_seq(a.c, r, lane);
  const int2 rr = paged_rows(a.c, b);
  const int32_t len = paged_len(a.c, b), t = len - (rr.y - (int32_t)r);
  const int2 keys = (int32_t)r < rr.x || (int32_t)r >= rr.y ? make_int2(0, 0) : paged_keys(a.m, r, t, len);
  const uint32_t p0 = (uint32_t)keys.x / a.split_len, p1 = keys.x < keys.y ? (uint32_t)(keys.y - 1) / a.split_len + 1 : p0;
  const float2* ml = a.part_ml + item * a.n_split;
  float top = -INFINITY, l = 0.f, o[E];
  for (uint32_t s = p0; s < p1; s++) top = fmaxf(top, ml[s].x);
  const float zero = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < E; i++) o[i] = 0.f;
  for (uint32_t s = p0; s < p1; s++) {
    const float2 x = ml[s];
    if (x.y == 0.f) continue;
    const float f = x.x == -INFINITY ? 1.f : ex2(x.x - zero);
    float v[E];
    load_as_float<E>(a.part, (item * a.n_split + s) * D + lane * E, SNL_T_F32, v);
    l = fmaf(x.y, f, l);
#pragma unroll
    for (int i = 0; i < E; i++) o[i] = fmaf(v[i], f, o[i]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float g[E];
  if (a.gate) load_as_float<E>(a.gate, r * a.p.gate_row + h * a.p.gate_head + lane * E, a.p.gate_type, g);
#pragma unroll
  for (int i = 0; i < E; i++) o[i] = l == 0.f ? 0.f : o[i] * (a.gate ? inv * sigmoidf_(g[i]) : inv);
  store_from_float<E>(a.out, r * a.p.out_row + h * a.p.out_head + lane * E, a.p.out_type, o);
  if (a.lse && lane == 0) a.lse[item] = l == 0.f ? -INFINITY : (zero + log2f(l)) * (1.f / kLog2e);
}

}  // namespace
}  // namespace snl

using namespace snl;

namespace {

struct AttendPlan {
  uint32_t toks, slots, n_split, split_len;
};

// How many parts the keys are cut into: the fewest microseconds of a model of waves of clusters
// (one per two SMs, two at head_dim 128), each with a start and an end, and the traffic and
// launch of the join. Measured over 11 shapes against 1 to 32 parts, the choice is within 11%
// of the best (128 rows over 8192 keys: 6 parts 37 us, 1 part 96, 32 parts 105; 512 rows: 2 parts
// 68, 1 part 98, 4 parts 81; 4 x 300 rows over up to 4000 keys: 1 part 64, 2 parts 75).
AttendPlan plan_attend(const snl_paged_cache& c, const snl_paged_batch& b, uint32_t n_heads) {
  AttendPlan pl{};
  const uint32_t group = n_heads / c.n_kv;
  pl.toks = 128 / group;
  pl.slots = b.n_rows / (2 * pl.toks) + b.n_seqs;
  const uint64_t max_len = std::min<uint64_t>(b.max_len, (uint64_t)b.table_stride * c.page_size);
  const uint64_t units = (uint64_t)std::min<uint64_t>(pl.slots, b.n_rows) * c.n_kv;
  const bool wide = c.head_dim == 256;
  const double per_key = wide ? 0.011 : 0.014, sms = std::max(1, wide ? sm_count() / 2 : sm_count());
  double best = 1e30;
  pl.n_split = 1;
  for (uint32_t n = 1; n <= 64; n++) {
    const uint64_t len = ((max_len + n - 1) / n + 127) / 128 * 128;
    if (n > 1 && len < 128) break;
    const double waves = std::max(1.0, (double)((units * n + (uint64_t)sms - 1) / (uint64_t)sms));
    double t = waves * (len * per_key + 3.0);
    if (n > 1) t += 3.0 + (double)b.n_rows * n_heads * n * c.head_dim * 8 / 4e6;
    if (t < best) {
      best = t;
      pl.n_split = n;
    }
  }
  pl.split_len = (uint32_t)(((max_len + pl.n_split - 1) / pl.n_split + 127) / 128 * 128);
  if (pl.split_len == 0) pl.split_len = 128;
  pl.n_split = std::max<uint32_t>(1, (uint32_t)((max_len + pl.split_len - 1) / pl.split_len));
  return pl;
}

size_t part_bytes(const AttendPlan& pl, const snl_paged_cache& c, const snl_paged_batch& b, uint32_t n_heads) {
  return pl.n_split == 1 ? 16 : (size_t)b.n_rows * n_heads * pl.n_split * (c.head_dim + 2) * sizeof(float);
}

template <typename T, int D, bool GENERAL>
int go_attend(const AttendArgs& a, const CUtensorMap& km, const CUtensorMap& vm, uint32_t grid, cudaStream_t s) {
  static bool attr[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr[dev]) {
    SNL_CUDA_TRY(cudaFuncSetAttribute(attend_kernel<T, D, GENERAL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)Geo<D>::kSmem));
    if (dev >= 0 && dev < 64) attr[dev] = true;
  }
  SNL_PDL_LAUNCH("attend_kernel", (attend_kernel<T, D, GENERAL>), dim3(grid), dim3(kAttendThreads),
                 (size_t)Geo<D>::kSmem, s, a, km, vm);
  return SNL_OK;
}

}  // namespace

extern "C" size_t snl_paged_attend_workspace(const snl_paged_cache* c, const snl_paged_batch* b, uint32_t n_heads) {
  if (!c || !b || c->n_kv == 0 || n_heads == 0 || n_heads % c->n_kv || n_heads / c->n_kv > 64) return 0;
  if (attend_rows_fits(*c, *b, n_heads / c->n_kv)) return std::max<size_t>(16, attend_rows_workspace(*c, *b, n_heads / c->n_kv));
  return part_bytes(plan_attend(*c, *b, n_heads), *c, *b, n_heads);
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
  if (paged_overlap(b->n_rows, p->out_row, c->head_dim) || paged_overlap(p->n_heads, p->out_head, c->head_dim))
    return fail(SNL_E_INVALID, w + ": the rows of out overlap");
  if (work_bytes < snl_paged_attend_workspace(c, b, p->n_heads)) return fail(SNL_E_INVALID, w + ": work is too small");
  if (!work) return fail(SNL_E_INVALID, w + ": null argument");
  if (b->n_rows == 0 || b->n_seqs == 0) return SNL_OK;
  SNL_TRY(paged_error_word(&a.c.err));
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.gate = gate;
  a.out = out;
  a.lse = lse;
  a.group = p->n_heads / c->n_kv;
  const cudaStream_t s = (cudaStream_t)stream;
  if (attend_rows_fits(*c, *b, a.group)) return launch_attend_rows(*c, *b, a, work, s);
  const AttendPlan pl = plan_attend(*c, *b, p->n_heads);
  const uint64_t grid = (uint64_t)pl.slots * pl.n_split * c->n_kv * 2;
  if (grid > 0x7fffffffull) return fail(SNL_E_UNSUPPORTED, w + ": too many rows");
  a.vrun = c->page_size >= 16 ? 16 : 8;
  CUtensorMap km, vm;
  SNL_TRY(page_map(&km, *c, c->k, 8, c->head_dim / 64));
  SNL_TRY(page_map(&vm, *c, c->v, a.vrun, c->head_dim / 128));
  a.toks = pl.toks;
  a.slots = pl.slots;
  a.n_split = pl.n_split;
  a.split_len = pl.split_len;
  a.part = static_cast<float*>(work);
  a.part_ml = reinterpret_cast<float2*>(a.part + (size_t)b->n_rows * p->n_heads * pl.n_split * c->head_dim);
  const bool half = c->type == SNL_T_F16, wide = c->head_dim == 256, gen = p->cap > 0.f || p->slopes;
  const uint32_t g = (uint32_t)grid;
  if (half && wide) SNL_TRY(gen ? (go_attend<__half, 256, true>(a, km, vm, g, s)) : (go_attend<__half, 256, false>(a, km, vm, g, s)));
  else if (half) SNL_TRY(gen ? (go_attend<__half, 128, true>(a, km, vm, g, s)) : (go_attend<__half, 128, false>(a, km, vm, g, s)));
  else if (wide) SNL_TRY(gen ? (go_attend<__nv_bfloat16, 256, true>(a, km, vm, g, s)) : (go_attend<__nv_bfloat16, 256, false>(a, km, vm, g, s)));
  else SNL_TRY(gen ? (go_attend<__nv_bfloat16, 128, true>(a, km, vm, g, s)) : (go_attend<__nv_bfloat16, 128, false>(a, km, vm, g, s)));
  if (pl.n_split == 1) return SNL_OK;
  const uint64_t items = (uint64_t)b->n_rows * p->n_heads;
  const dim3 jg((unsigned)((items + kWarps - 1) / kWarps));
  if (wide) SNL_PDL_LAUNCH("join_kernel", join_kernel<256>, jg, dim3(kWarps * 32), (size_t)0, s, a);
  else SNL_PDL_LAUNCH("join_kernel", join_kernel<128>, jg, dim3(kWarps * 32), (size_t)0, s, a);
  return SNL_OK;
}
