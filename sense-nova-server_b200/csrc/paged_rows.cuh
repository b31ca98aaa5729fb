// Pieces of the kernels that read the paged cache for one or two rows a sequence: m16n8k16
// tiles fed by ldmatrix from TMA boxes of 8 keys.
#pragma once
#include "paged_tc.cuh"

namespace snl {

constexpr uint32_t kRowWarps = 8, kBlock = 64;  // keys of a block: 8 of each warp

// S += Q K^T: rows 0-7 of A (a0, a2) and 8-15 (a1, a3).
template <typename T>
__device__ __forceinline__ void mma_k16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_k8(float d[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(b0));
  else
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Into this CTA's memory; the box is 8 slots of a head.
__device__ __forceinline__ void tma_group(uint32_t dst, const CUtensorMap* map, int slot, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(map), "r"(0), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// Address for ldmatrix x4 of elements 32 c to 32 c + 31 of a box's 8 keys: lane L gives row
// L % 8 of matrix L / 8, 16 bytes each, four along a swizzled row.
__device__ __forceinline__ uint32_t box_at(uint32_t box, uint32_t c, uint32_t lane) {
  const uint32_t row = lane & 7, sel = lane >> 3;
  return box + (c / 2) * 1024 + row * 128 + ((((c & 1) * 4 + sel) ^ row) << 4);
}

}  // namespace snl
