// What the paged cache's tensor-core kernels share: arithmetic of the scores, the tcgen05 and
// cluster instructions of a pair of CTAs, TMA boxes of the pages.
#pragma once
#include <type_traits>

#include "paged.cuh"
#include "tc.cuh"
#include "tensor_map.cuh"

namespace snl {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh x for |x| < 0.4: the first terms of its Taylor series.
constexpr float kTanhNear = 0.4f;
__device__ __forceinline__ float tanh_near(float x) {
  const float y = x * x;
  float p = fmaf(y, -1382.f / 155925.f, 62.f / 2835.f);
  p = fmaf(y, p, -17.f / 315.f);
  p = fmaf(y, p, 2.f / 15.f);
  p = fmaf(y, p, -1.f / 3.f);
  return fmaf(x * y, p, x);
}
// tanh x = 1 - 2 / (1 + e^2x), off by less than 2^-22 (tanh.approx: 2^-11), which near 0 is more
// than 32 bits should lose of a score that a far larger cap leaves as it is; 6e-7 of the value
// at most on either side of kTanhNear.
__device__ __forceinline__ float tanh_(float x) {
  const float far = fmaf(-2.f, rcp(1.f + ex2(2.f * kLog2e * x)), 1.f);
  return fabsf(x) < kTanhNear ? tanh_near(x) : far;
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ void bar_sync(uint32_t id, uint32_t n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
// A value that is the same in all lanes of a warp, said so: branches on it and addresses from
// it need no look at the lanes, and MMA operands come from uniform registers (weigh of 2048
// rows over 8192 keys 168 -> 143 us with the warp's and the CTA's number and the operands).
__device__ __forceinline__ uint32_t same_in_warp(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// 1 in one lane of the warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p;
}

template <typename T>
constexpr uint32_t idesc16(uint32_t n, bool b_mn) {  // D f32, A and B f16 or bf16, M = 256
  const uint32_t t = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((256u >> 4) << 24);
}
// Descriptor of a 128-byte swizzled operand, as halves. K-major: sbo between 8-row groups.
// MN-major: lbo between chunks of 64 along MN, sbo between groups of 8 along K. The low half
// of an address further on is the low half plus the distance / 16 (shared memory ends below
// 2^18), one addition where the whole descriptor anew took 80 cycles an MMA.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return saddr >> 4 | (lbo >> 4) << 16; }
__device__ __forceinline__ uint32_t desc_hi(uint32_t sbo) { return sbo >> 4 | 1u << 14 | 2u << 29; }
// The whole warp runs the code around an MMA and `lead` (one lane) issues it.
__device__ __forceinline__ void mma2_ss(uint32_t lead, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 q, %7, 0;\n mov.b64 a, {%1, %2};\n"
      " mov.b64 b, {%3, %4};\n @q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %5, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
// A from tensor memory.
__device__ __forceinline__ void mma2_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                        uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 q, %6, 0;\n mov.b64 b, {%2, %3};\n"
      " @q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
// Arrives on both CTAs' barriers, or this one's, once the MMAs issued so far have completed.
__device__ __forceinline__ void commit2(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}\n" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_own(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// Pairs of CTAs that hold tensor memory on one SM and wait for more on the other must not meet:
// kernels that take all 512 columns also take so much shared memory that no other such CTA
// fits beside them.
template <uint32_t COLS>
__device__ __forceinline__ void tmem_alloc2(uint32_t* dst) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "n"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
template <uint32_t COLS>
__device__ __forceinline__ void tmem_dealloc2(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
// The two halves of a cluster's meeting before which threads wrote nothing but barriers, which
// fence_mbar_init() has released.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive_cta(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// With release, what this thread wrote to memory is seen by who waits (about 1000 cycles at
// cluster scope); tensor memory is ordered by its own fences and needs none.
__device__ __forceinline__ void arrive_cluster(uint32_t bar, bool release) {
  if (release) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
  else asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded waits of about 0.15 s: the longest that one of these is due is some microseconds.
// The second sees what the other CTA released.
__device__ __forceinline__ bool wait_mbar(uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, 1ll << 28); }
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity) {
  if (try_wait_cluster(bar, parity)) return true;
  const long long t0 = clock64();
  while (!try_wait_cluster(bar, parity))
    if (clock64() - t0 > (1ll << 28)) return false;
  return true;
}
// A variable of the CTA whose address in_cta() gave.
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t x;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}
// Boxes into this CTA, counted on a barrier that may be the other CTA's: slots of a page, or
// one chunk of the queries of some tokens.
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int slot, int chunk, int head, int page,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(0), "r"(slot), "r"(chunk), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_query(uint32_t dst, const CUtensorMap* map, int head, int token, int chunk, int kv_head,
                                          uint32_t bar) {
  tma_load_5d(dst, map, head, token, chunk, kv_head, bar);
}

// 32 columns of this thread's lane, not waited for.
__device__ __forceinline__ void tm_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tm_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tm_st(uint32_t taddr, const uint32_t* r) {
  static_assert(N == 16 || N == 32, "columns");
  if constexpr (N == 16) tm_st16(taddr, r);
  else tm_st32(taddr, r);
}
// Waits for this thread's loads; the empty statements keep uses of the registers behind it.
template <int N>
__device__ __forceinline__ void tm_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The pages as (64 elements, slot, chunk of 64, head, page): a box is some slots of a head, or of
// half of one.
inline int page_map(CUtensorMap* map, const snl_paged_cache& c, void* base, uint32_t slots, uint32_t chunks) {
  PFN_cuTensorMapEncodeTiled enc = tensor_map_encoder();
  if (!enc) return fail(SNL_E_CUDA, "paged cache: cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[5] = {64, c.page_size, c.head_dim / 64, c.n_kv, c.n_pages};
  const cuuint64_t str[4] = {c.slot_stride * 2, 128, c.n_kv > 1 ? c.head_stride * 2 : 128,
                             c.n_pages > 1 ? c.page_stride * 2 : 128};
  const cuuint32_t box[5] = {64, slots, chunks, 1, 1}, one[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, c.type == SNL_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                         base, dims, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SNL_OK : fail(SNL_E_INVALID, "paged cache: the pages' strides do not fit a tensor map");
}

}  // namespace snl
