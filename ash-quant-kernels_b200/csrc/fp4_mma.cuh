// tcgen05 with block scales: 4-bit operands and their scales straight from memory to the tensor core.
//
// One instruction multiplies 64 columns of K (32 bytes of a row). The operands are K-major rows of 128
// bytes in 128-byte-swizzled atoms, as for 8-bit types; the scales are read from TMEM: scale tile
// (128 rows x 4 blocks) in four columns, row 32 c + l in lane l of column c, the four lane quarters alike.
#pragma once

#include "fp4.cuh"
#include "sm100.cuh"

namespace ashqk {

constexpr int kFp4BlockK = 256;  // columns of K per pipeline stage: one 128-byte row

template <int FMT>
struct Fp4Mma {
  static constexpr int kTilesPerStage = kFp4BlockK / fp4_block(FMT) / 4;  // scale tiles: 2 (MXFP4), 4 (NVFP4)
  // Instruction j of a stage covers 64 columns: half a scale tile (MXFP4) or one (NVFP4).
  static __device__ __forceinline__ constexpr int tile_of(int j) { return FMT == ASHQK_MXFP4 ? j / 2 : j; }
  // Byte of the tile's four that its scales start at.
  static __device__ __forceinline__ constexpr uint32_t sf_id(int j) { return FMT == ASHQK_MXFP4 ? (j & 1) * 2u : 0u; }

  // Instruction descriptor: E2M1 times E2M1, both K-major, scales E8M0 or E4M3, fp32 sums.
  static __device__ __forceinline__ constexpr uint32_t idesc(int m, int n, int j) {
    return (sf_id(j) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           ((FMT == ASHQK_MXFP4 ? 1u : 0u) << 23) | (static_cast<uint32_t>(m >> 4) << 24) | (sf_id(j) << 29);
  }

  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                             uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == ASHQK_MXFP4)
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
          " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
          ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
          : "memory");
    else
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
          " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
          ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
          : "memory");
  }

  static __device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                                  uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == ASHQK_MXFP4)
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
          " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
          ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
          : "memory");
    else
      asm volatile(
          "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
          " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
          ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
          : "memory");
  }
};

// Descriptor of one 512-byte scale tile for tcgen05.cp: no swizzle, 8-row groups of 128 bytes.
__device__ __forceinline__ uint64_t scale_tile_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) | (1ull << 46);
}
// Scale tile -> four TMEM columns, the same 32 lanes in every quarter. Ordered before later tcgen05.mma of
// the issuing thread.
__device__ __forceinline__ void scale_tile_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void scale_tile_to_tmem_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// 16 bytes into the shared memory of a CTA of the cluster, counted on that CTA's barrier (cluster addresses).
__device__ __forceinline__ void st_async_v4(uint32_t remote_addr, uint4 v, uint32_t remote_bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                   remote_addr),
               "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(remote_bar)
               : "memory");
}
// The same for a piece of this CTA's shared memory (16-byte aligned, a multiple of 16 bytes): several times st.async's
// rate from a kilobyte on.
__device__ __forceinline__ void bulk_to_cluster(uint32_t remote_addr, uint32_t src, uint32_t bytes, uint32_t remote_bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   remote_addr),
               "r"(src), "r"(bytes), "r"(remote_bar)
               : "memory");
}
// The halves of cluster_sync().
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The address in CTA `rank` of the cluster of a shared-memory address of this one.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// 32 lanes x 8 consecutive fp32 columns.
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

}  // namespace ashqk
