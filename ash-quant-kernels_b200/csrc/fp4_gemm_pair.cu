// y = alpha * A B^T with 4-bit operands, many rows of A: 256 x 256 tiles on CTA pairs.
//
// tcgen05.mma.cta_group::2 with block scales, M = 256 rows of A, N = 256 rows of B. Each CTA of a pair
// stages its own 128 rows of A with their scales, its own 128 of the 256 rows of B, and the scales of
// all 256 (the instruction wants them in both CTAs' TMEM). Persistent, one pair per two SMs.
//
//   both CTAs   warp 0, one thread: TMA into its own shared memory, completing on the even CTA's barrier;
//               warps 2..9: epilogue of its 128 rows, TMEM -> registers -> y.
//   even CTA    warp 1, one thread: scales to TMEM (tcgen05.cp into both CTAs), MMAs, commits to both CTAs.
//
// TMEM (512 columns): two accumulators of 256 columns that share 128 (0..255 and 128..383), and two
// buffers of scales. An epilogue reads the shared half first and hands it back, so the next tile's MMAs
// wait for half a read-out and no store.
#include <algorithm>
#include <atomic>

#include "fp4_mma.cuh"

namespace ashqk {
namespace {

constexpr int kBM = 128;     // rows of A per CTA
constexpr int kBN = 256;     // rows of B per pair (MMA N)
constexpr int kHalfN = 128;  // rows of B staged per CTA
constexpr int kEpiWarps = 8;
constexpr int kFirstEpiWarp = 2;
constexpr int kThreads = 32 * (kFirstEpiWarp + kEpiWarps);
constexpr int kGroupM = 8;  // tile order: row tiles walked together

struct PairMaps {
  CUtensorMap a, b, as, bs, y;
};

struct PairArgs {
  void* y;
  int64_t y_ld;
  int M, N, k_steps, num_kb;
  int tiles_m, tiles_n;
  float alpha;
  int bf16;
  int tma_y;  // y takes TMA stores: 16-byte aligned base and rows
};

template <int FMT>
struct PairSmem {
  static constexpr int kT = Fp4Mma<FMT>::kTilesPerStage;
  static constexpr int kStages = 5;
  static constexpr uint32_t kA = kBM * 128;
  static constexpr uint32_t kB = kHalfN * 128;
  static constexpr uint32_t kAS = kT * kFp4TileBytes;
  static constexpr uint32_t kBS = 2 * kAS;
  static constexpr uint32_t kStage = kA + kB + kAS + kBS;
  static constexpr uint32_t kOut = 32 * 128;  // an epilogue warp's 32 rows x 64 columns of y
  static constexpr uint32_t off_out = kStages * kStage;
  static constexpr uint32_t off_bar = off_out + kEpiWarps * kOut;
  static constexpr int kBars = 2 * kStages + 3 + 2;
  static constexpr uint32_t bytes = off_bar + kBars * 8 + 16;
  static_assert(kStage % 1024 == 0, "swizzle atoms need 1 KB alignment");
  // TMEM columns.
  static constexpr uint32_t kAcc1 = 128;
  static constexpr uint32_t kSf = 384;
  static constexpr uint32_t kSfA = kT * 4, kSfB = kT * 8;
  static_assert(kSf + 2 * (kSfA + kSfB) <= 512, "TMEM");
};

// Tile t -> (row tile, column tile): groups of kGroupM row tiles, walked column by column, so that the tiles
// in flight share both operands' rows in L2.
__device__ __forceinline__ void tile_of(const PairArgs& a, int t, int& tm, int& tn) {
  const int per_group = kGroupM * a.tiles_n;
  const int g = t / per_group;
  const int rows = min(kGroupM, a.tiles_m - g * kGroupM);
  const int r = t - g * per_group;
  tm = g * kGroupM + r % rows;
  tn = r / rows;
}

// TMA load completing on the barrier (cluster address) of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ uint16_t lds_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}

// 64 fp32 columns of one row, times alpha, as 16-bit pairs.
template <typename T>
__device__ __forceinline__ void round_row64(const uint32_t (&r0)[32], const uint32_t (&r1)[32], float alpha, uint32_t (&h)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    h[i] = pack2<T>(alpha * __uint_as_float(r0[2 * i]), alpha * __uint_as_float(r0[2 * i + 1]));
    h[16 + i] = pack2<T>(alpha * __uint_as_float(r1[2 * i]), alpha * __uint_as_float(r1[2 * i + 1]));
  }
}

template <int FMT>
__global__ void __launch_bounds__(kThreads, 1) fp4_pair_kernel(const __grid_constant__ PairMaps maps, const PairArgs a) {
  using L = PairSmem<FMT>;
  using Mma = Fp4Mma<FMT>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::off_bar);  // used in the even CTA
  uint64_t* empty = full + L::kStages;
  uint64_t* acc_full = empty + L::kStages;
  uint64_t* acc_free = acc_full + 2;  // used in the even CTA: both CTAs' epilogues arrive
  uint64_t* mma_done = acc_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 2);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // known to be uniform
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(acc_free, 2 * kEpiWarps);
    mbar_init(mma_done, 1);
    *abort = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&maps.a);
    prefetch_tensormap(&maps.b);
    prefetch_tensormap(&maps.as);
    prefetch_tensormap(&maps.bs);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_alloc_permit_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before anyone signals them
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  pdl_wait();
  pdl_launch_dependents();

  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int pairs = static_cast<int>(gridDim.x >> 1);
  const int tiles = a.tiles_m * a.tiles_n;

  if (warp == 0) {
    const uint32_t full_lead = map_shared_rank(full, 0);
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    for (int t = pair; t < tiles && !*abort; t += pairs) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      const int ra = 2 * tm + static_cast<int>(rank);  // 128-row tile of A
      const int rb = 2 * tn + static_cast<int>(rank);
      for (int kb = 0; kb < a.num_kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort, true)) break;
        unsigned char* base = smem + stage * L::kStage;
        const uint32_t bar = full_lead + 8u * stage;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * L::kStage);
          tma_load_2d_pair(base, &maps.a, kb * 128, ra * kBM, bar);
          tma_load_2d_pair(base + L::kA, &maps.b, kb * 128, rb * kHalfN, bar);
          tma_load_2d_pair(base + L::kA + L::kB, &maps.as, kb * (L::kAS / 8), ra, bar);
          tma_load_2d_pair(base + L::kA + L::kB + L::kAS, &maps.bs, kb * (L::kAS / 8), 2 * tn, bar);
        }
        __syncwarp();
        ++issued;
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // The even CTA's barriers count both CTAs' copies; the odd CTA leaves behind the cluster barrier below.
    if (rank == 0)
      for (int i = 1; i <= L::kStages && i <= issued; ++i) {
        const int f = issued - i;
        mbar_drain(&full[f % L::kStages], static_cast<uint32_t>(f / L::kStages) & 1u);
      }
  } else if (warp == 1) {
    if (rank == 0) {
      // The whole warp runs the loop and waits; one elected lane issues.
      int i = 0;  // stages consumed
      int stage = 0;
      uint32_t phase = 0, local = 0;
      for (int t = pair; t < tiles && !*abort; t += pairs, ++local) {
        // The accumulator before this one has handed back the half that the two share (and, before that, this one
        // was read out whole: the same warps read in order).
        if (local > 0 && !mbar_wait(acc_free, (local - 1) & 1u, abort, true)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + ((local & 1u) ? L::kAcc1 : 0u);
        bool ok = true;
        for (int kb = 0; kb < a.num_kb; ++kb, ++i) {
          if (!mbar_wait(&full[stage], phase, abort, true)) {
            ok = false;
            break;
          }
          // The scale buffer's last reader, stage i - 2, has finished.
          const int old = stage >= 2 ? stage - 2 : stage - 2 + L::kStages;
          if (i >= 2 && !mbar_wait(&empty[old], stage >= 2 ? phase : phase ^ 1u, abort, true)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t base = sbase + stage * L::kStage;
          const uint32_t sfa = tmem + L::kSf + (i & 1) * (L::kSfA + L::kSfB);
          const uint32_t sfb = sfa + L::kSfA;
          const uint64_t sa = scale_tile_desc(base + L::kA + L::kB);
          const uint64_t da = umma_desc_sw128(base, 16u, 1024u);
          const uint64_t db = umma_desc_sw128(base + L::kA, 16u, 1024u);
          const int steps = min(4, a.k_steps - kb * 4);
          if (elect_one()) {
#pragma unroll
            for (int s = 0; s < L::kT; ++s) {
              scale_tile_to_tmem_pair(sfa + s * 4, sa + s * (kFp4TileBytes >> 4));
              scale_tile_to_tmem_pair(sfb + s * 8, sa + ((L::kAS + s * kFp4TileBytes) >> 4));
              scale_tile_to_tmem_pair(sfb + s * 8 + 4, sa + ((2 * L::kAS + s * kFp4TileBytes) >> 4));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (j >= steps) break;
              Mma::mma_pair(d, da + 2 * j, db + 2 * j, Mma::idesc(2 * kBM, kBN, j), sfa + Mma::tile_of(j) * 4,
                            sfb + Mma::tile_of(j) * 8, (kb | j) != 0);
            }
            umma_commit_pair_mc(&empty[stage], 0x3);
            if (kb + 1 == a.num_kb) umma_commit_pair_mc(&acc_full[local & 1u], 0x3);
          }
          __syncwarp();
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
      }
      if (elect_one()) umma_commit_pair(mma_done);
      __syncwarp();
      mbar_drain(mma_done, 0);
    }
  } else {
    const int quad = warp & 3;
    const int part = (warp - kFirstEpiWarp) >> 2;  // which 64 columns of each half
    const uint32_t acc_free_lead = map_shared_rank(acc_free, 0);
    const uint32_t out = sbase + L::off_out + static_cast<uint32_t>(warp - kFirstEpiWarp) * L::kOut;
    uint32_t local = 0;
    for (int t = pair; t < tiles; t += pairs, ++local) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      if (!mbar_wait(&acc_full[local & 1u], (local >> 1) & 1u, abort)) break;
      tc_fence_after_sync();
      const int row0 = tm * (2 * kBM) + static_cast<int>(rank) * kBM + 32 * quad;
      const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quad) << 16);
      const uint32_t acc = lanes + ((local & 1u) ? L::kAcc1 : 0u);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // The shared half is this accumulator's second (even tiles) or first (odd tiles).
        const int col = ((h == 0) != ((local & 1u) != 0) ? 128 : 0) + 64 * part;
        uint32_t r0[32], r1[32];
        tmem_ld_32x32b_x32(acc + col, r0);
        tmem_ld_32x32b_x32(acc + col + 32, r1);
        tmem_wait_ld();
        if (h == 0) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acc_free_lead);
        }
        uint32_t v[32];
        if (a.bf16)
          round_row64<__nv_bfloat16>(r0, r1, a.alpha, v);
        else
          round_row64<__half>(r0, r1, a.alpha, v);
        const int n = tn * kBN + col;
        // Through shared memory in the swizzled layout (conflict-free: eight lanes write eight 16-byte columns).
        if (lane == 0) bulk_wait_read();
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; ++c)
          sts_v4(out + lane * 128 + ((c ^ (lane & 7)) << 4), make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]));
        if (a.tma_y) {  // out as one box of whole 128-byte rows
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < a.M && n < a.N) {
            tma_store_2d(&maps.y, n, row0, smem + L::off_out + (warp - kFirstEpiWarp) * L::kOut);
            bulk_commit();
          }
        } else {  // rows of any alignment: the warp writes one after the other
          __syncwarp();
          uint16_t* y = static_cast<uint16_t*>(a.y) + row0 * a.y_ld + n + lane;
          const int rows = min(32, a.M - row0);
          const bool in0 = n + lane < a.N, in1 = n + 32 + lane < a.N;
#pragma unroll 4
          for (int i = 0; i < rows; ++i, y += a.y_ld) {
            const uint32_t at = out + i * 128 + (lane & 7) * 2;
            if (in0) y[0] = lds_u16(at + (((lane >> 3) ^ (i & 7)) << 4));
            if (in1) y[32] = lds_u16(at + (((4 + (lane >> 3)) ^ (i & 7)) << 4));
          }
          __syncwarp();
        }
      }
      // The other half is only overwritten after the next tile's shared half was handed back, by these warps.
      tc_fence_before_sync();
    }
    if (lane == 0) bulk_wait();
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // the pair's MMAs have completed and read neither CTA's memory any more
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
}

template <int FMT>
int launch_pair(const PairMaps& maps, const PairArgs& a, cudaStream_t stream) {
  using L = PairSmem<FMT>;
  DeviceInfo dev;
  if (const int rc = device_info(&dev)) return rc;
  auto kernel = fp4_pair_kernel<FMT>;
  const size_t smem = L::bytes + 1024;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Persistent: every pair resident at once (pairs need two free SMs in one GPC, so fewer than half the SMs may fit).
  static std::atomic<int> resident[64];  // zero-initialised (static storage)
  int pairs = resident[dev.device].load(std::memory_order_acquire);
  if (pairs == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return ASHQK_ERR_CUDA;
    cfg.gridDim = dim3(2 * (dev.sm_count / 2));
    if (cudaOccupancyMaxActiveClusters(&pairs, kernel, &cfg) != cudaSuccess || pairs <= 0) return ASHQK_ERR_CUDA;
    pairs = std::min(pairs, dev.sm_count / 2);
    resident[dev.device].store(pairs, std::memory_order_release);
  }
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min(static_cast<int64_t>(pairs), static_cast<int64_t>(a.tiles_m) * a.tiles_n)));
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, maps, a) == cudaSuccess ? ASHQK_OK : ASHQK_ERR_CUDA;
}

}  // namespace

int fp4_matmul_pair(const void* a_codes, int64_t a_ld, const void* a_scales, const void* b_codes, int64_t b_ld,
                    const void* b_scales, void* y, int64_t y_ld, int dtype, int M, int N, int K, int format, float alpha,
                    cudaStream_t stream) {
  PairArgs a;
  a.y = y;
  a.y_ld = y_ld;
  a.M = M;
  a.N = N;
  a.k_steps = static_cast<int>(ceil_div64(fp4_padded_k(K), 64));
  a.num_kb = static_cast<int>(ceil_div64(fp4_padded_k(K), kFp4BlockK));
  a.tiles_m = ceil_div(M, 2 * kBM);
  a.tiles_n = ceil_div(N, kBN);
  if (static_cast<int64_t>(a.tiles_m) * a.tiles_n > (1 << 30)) return ASHQK_ERR_UNSUPPORTED;
  a.alpha = alpha;
  a.bf16 = dtype == ASHQK_BF16;
  a.tma_y = aligned(y, 16) && y_ld % 8 == 0;
  const uint64_t row_bytes = fp4_padded_k(K) / 2;
  const uint64_t scale_bytes = fp4_scale_tiles(K, format) * kFp4TileBytes;
  const uint32_t stage_scales = kFp4BlockK / fp4_block(format) / 4 * kFp4TileBytes;
  PairMaps maps;
  int rc = encode_tensor_map_2d(&maps.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<void*>(a_codes), row_bytes, M, a_ld, 128,
                                kBM, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc)
    rc = encode_tensor_map_2d(&maps.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<void*>(b_codes), row_bytes, N, b_ld, 128,
                              kHalfN, CU_TENSOR_MAP_SWIZZLE_128B);
  // Scale tiles as rows of 8-byte elements: one row per 128 rows of the matrix.
  if (!rc)
    rc = encode_tensor_map_2d(&maps.as, CU_TENSOR_MAP_DATA_TYPE_UINT64, const_cast<void*>(a_scales), scale_bytes / 8,
                              ceil_div(M, kFp4TileRows), scale_bytes, stage_scales / 8, 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!rc)
    rc = encode_tensor_map_2d(&maps.bs, CU_TENSOR_MAP_DATA_TYPE_UINT64, const_cast<void*>(b_scales), scale_bytes / 8,
                              ceil_div(N, kFp4TileRows), scale_bytes, stage_scales / 8, 2, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!rc)
    rc = a.tma_y ? encode_tensor_map_2d(&maps.y, CU_TENSOR_MAP_DATA_TYPE_UINT16, y, N, M, y_ld * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B)
                 : (maps.y = maps.a, ASHQK_OK);
  if (rc) return rc;
  return format == ASHQK_MXFP4 ? launch_pair<ASHQK_MXFP4>(maps, a, stream) : launch_pair<ASHQK_NVFP4>(maps, a, stream);
}

}  // namespace ashqk
