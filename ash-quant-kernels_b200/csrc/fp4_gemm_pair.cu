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
// With at most half as many tiles as pairs K is split: the two pairs of a four-CTA cluster take half of a tile's stages
// each, then half of the columns each, whose sums the other pair sends over (own shared memory, then bulk copies
// counted on a barrier) -- no workspace, added in a fixed order.
//
// Bound by the tensor pipe (71 % of cycles active, the scale copies queued between the MMAs) and, in long runs, by the
// part's power limit: 8192 x 24576 x 4096 on a B200, replayed in a graph, 300-340 us in MXFP4 (4.9-5.5 PFLOP/s), 310-330 in
// NVFP4; called in a row from Python 343-350 (4.7-4.8). 2048 x 4096 x 12288: 37 us in MXFP4, 38.5 in NVFP4. Tiles of 256 x
// 256 because each SM then takes 68 bytes a cycle from L2 at the MMAs' nominal rate.
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
// Stages from which splitting K pays: the exchange of the halves costs 2.9 us, a stage 0.3 to 0.35 us (512 rows
// 12288->4096, 48 stages: 19.3 -> 16.1 us; 512 rows 4096->4096, 16 stages: 9.8 against 10.8 split).
constexpr int kMinSplitKb = 24;

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
  static constexpr int kBars = 2 * kStages + 3 + 3;
  static constexpr uint32_t bytes = off_bar + kBars * 8 + 16;
  static_assert(kStage % 1024 == 0, "swizzle atoms need 1 KB alignment");
  // TMEM columns.
  static constexpr uint32_t kAcc1 = 128;
  static constexpr uint32_t kSf = 384;
  static constexpr uint32_t kSfA = kT * 4, kSfB = kT * 8;
  static_assert(kSf + 2 * (kSfA + kSfB) <= 512, "TMEM");
  // Split K: the sums that a CTA receives, then those that it sends, take the ring's place.
  static constexpr uint32_t kHalf = kBM * kBN / 2 * 4;
  static_assert(2 * kHalf <= kStages * kStage, "sums");
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
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
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
__device__ __forceinline__ void round_row64(const uint32_t (&r0)[32], const uint32_t (&r1)[32], float alpha,
                                            uint32_t (&h)[32]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    h[i] = pack2<T>(alpha * __uint_as_float(r0[2 * i]), alpha * __uint_as_float(r0[2 * i + 1]));
    h[16 + i] = pack2<T>(alpha * __uint_as_float(r1[2 * i]), alpha * __uint_as_float(r1[2 * i + 1]));
  }
}

// An epilogue warp's 32 rows x 64 columns of sums -> y. `out`: its staging buffer.
__device__ __forceinline__ void store_tile(const PairMaps& maps, const PairArgs& a, const uint32_t (&r0)[32],
                                           const uint32_t (&r1)[32], unsigned char* out, int row0, int n, int lane) {
  uint32_t v[32];
  if (a.bf16)
    round_row64<__nv_bfloat16>(r0, r1, a.alpha, v);
  else
    round_row64<__half>(r0, r1, a.alpha, v);
  // Through shared memory in the swizzled layout (conflict-free: eight lanes write eight 16-byte columns).
  const uint32_t at = smem_u32(out);
  if (lane == 0) bulk_wait_read();
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c)
    sts_v4(at + lane * 128 + ((c ^ (lane & 7)) << 4), make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]));
  if (a.tma_y) {  // out as one box of whole 128-byte rows
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && row0 < a.M && n < a.N) {
      tma_store_2d(&maps.y, n, row0, out);
      bulk_commit();
    }
  } else {  // rows of any alignment: the warp writes one after the other
    __syncwarp();
    uint16_t* y = static_cast<uint16_t*>(a.y) + row0 * a.y_ld + n + lane;
    const int rows = min(32, a.M - row0);
    const bool in0 = n + lane < a.N, in1 = n + 32 + lane < a.N;
#pragma unroll 4
    for (int i = 0; i < rows; ++i, y += a.y_ld) {
      const uint32_t from = at + i * 128 + (lane & 7) * 2;
      if (in0) y[0] = lds_u16(from + (((lane >> 3) ^ (i & 7)) << 4));
      if (in1) y[32] = lds_u16(from + (((4 + (lane >> 3)) ^ (i & 7)) << 4));
    }
    __syncwarp();
  }
}

template <int FMT, bool SPLIT>
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
  uint64_t* received = mma_done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // known to be uniform
  const int lane = threadIdx.x & 31;
  const uint32_t crank = cluster_rank();
  const uint32_t rank = crank & 1u;       // 0: issues the pair's MMAs
  const uint32_t lead = crank & ~1u;
  constexpr int split = SPLIT ? 2 : 1;
  const int part_k = static_cast<int>(crank >> 1);  // this pair's share of K
  const uint16_t both = static_cast<uint16_t>(3u << lead);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(acc_free, 2 * kEpiWarps);
    mbar_init(mma_done, 1);
    mbar_init(received, 1);
    *abort = 0;
    fence_mbarrier_init();
    if (SPLIT) mbar_arrive_expect_tx(received, L::kHalf);
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

  // Split K: a cluster has one tile.
  const int pair = static_cast<int>(blockIdx.x >> 1) / split;
  const int pairs = static_cast<int>(gridDim.x >> 1) / split;
  const int kb0 = a.num_kb * part_k / split, kb1 = a.num_kb * (part_k + 1) / split;
  const int tiles = a.tiles_m * a.tiles_n;

  if (warp == 0) {
    const uint32_t full_lead = map_shared_rank(full, lead);
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    for (int t = pair; t < tiles && !*abort; t += pairs) {
      int tm, tn;
      tile_of(a, t, tm, tn);
      const int ra = 2 * tm + static_cast<int>(rank);  // 128-row tile of A
      const int rb = 2 * tn + static_cast<int>(rank);
      for (int kb = kb0; kb < kb1; ++kb) {
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
        for (int kb = kb0; kb < kb1; ++kb, ++i) {
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
                            sfb + Mma::tile_of(j) * 8, kb > kb0 || j > 0);
            }
            umma_commit_pair_mc(&empty[stage], both);
            if (kb + 1 == kb1) umma_commit_pair_mc(&acc_full[local & 1u], both);
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
  } else if (!SPLIT) {
    const int quad = warp & 3;
    const int part = (warp - kFirstEpiWarp) >> 2;  // which 64 columns of each half
    const uint32_t acc_free_lead = map_shared_rank(acc_free, lead);
    unsigned char* out = smem + L::off_out + (warp - kFirstEpiWarp) * L::kOut;
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
        store_tile(maps, a, r0, r1, out, row0, tn * kBN + col, lane);
      }
      // The other half is only overwritten after the next tile's shared half was handed back, by these warps.
      tc_fence_before_sync();
    }
    if (lane == 0) bulk_wait();
  }

  if (SPLIT) {
    // Each warp: 64 of the columns that the other pair owns, then 64 of this pair's, for its 32 rows: 8 KB as
    // [four columns][row] x 16 bytes, sent in one copy.
    const bool epilogue = warp >= kFirstEpiWarp;
    const int quad = warp & 3;
    const int part = (warp - kFirstEpiWarp) >> 2;
    const uint32_t piece = sbase + static_cast<uint32_t>(warp - kFirstEpiWarp) * 8192 + lane * 16;
    bool ok = false;
    uint32_t r[2][32];
    auto load_half = [&](int owner) {
      const uint32_t at = tmem + (static_cast<uint32_t>(32 * quad) << 16) + 128 * owner + 64 * part;
      tmem_ld_32x32b_x32(at, r[0]);
      tmem_ld_32x32b_x32(at + 32, r[1]);
      tmem_wait_ld();
      if (!ok) {  // a wait ran out: the sums are not there; the peer still gets the bytes that it counts
#pragma unroll
        for (int i = 0; i < 32; ++i) r[0][i] = r[1][i] = 0x7fffffffu;
      }
    };
    if (epilogue) {
      ok = mbar_wait(&acc_full[0], 0, abort);
      tc_fence_after_sync();
      load_half(1 - part_k);
    }
    __syncthreads();
    cluster_sync();  // both pairs are through with their rings
    if (epilogue) {
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint32_t* p = &r[c / 8][4 * (c % 8)];
        sts_v4(piece + L::kHalf + c * 512, make_uint4(p[0], p[1], p[2], p[3]));
      }
      fence_proxy_async_smem();
      __syncwarp();
      const uint32_t peer = crank ^ 2u;
      if (lane == 0) bulk_to_cluster(map_rank(piece, peer), piece + L::kHalf, 8192, map_rank(smem_u32(received), peer));
      __syncwarp();
      load_half(part_k);
      if (mbar_wait_cluster(received, 0, abort)) {
        int tm, tn;
        tile_of(a, pair, tm, tn);
#pragma unroll
        for (int c = 0; c < 16; ++c) {  // a sum of two: the same in either order
          uint32_t* p = &r[c / 8][4 * (c % 8)];
          const uint4 v = lds_v4(piece + c * 512);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = __float_as_uint(__uint_as_float(p[i]) + __uint_as_float(w[i]));
        }
        const int row0 = tm * (2 * kBM) + static_cast<int>(rank) * kBM + 32 * quad;
        store_tile(maps, a, r[0], r[1], smem + L::off_out + (warp - kFirstEpiWarp) * L::kOut, row0,
                   tn * kBN + 128 * part_k + 64 * part, lane);
      }
      if (lane == 0) bulk_wait();
    }
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

// Clusters that are resident at once: fewer than the SMs would hold, since a cluster stays within a GPC.
template <int FMT, bool SPLIT>
int resident_clusters(const DeviceInfo& dev, int* clusters) {
  constexpr int kCtas = SPLIT ? 4 : 2;
  static std::atomic<int> resident[64];  // zero-initialised (static storage)
  *clusters = resident[dev.device].load(std::memory_order_acquire);
  if (*clusters) return ASHQK_OK;
  auto kernel = fp4_pair_kernel<FMT, SPLIT>;
  const size_t smem = PairSmem<FMT>::bytes + 1024;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return ASHQK_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(dev.sm_count / kCtas * kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCtas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg) != cudaSuccess || *clusters <= 0) return ASHQK_ERR_CUDA;
  *clusters = std::min(*clusters, dev.sm_count / kCtas);
  resident[dev.device].store(*clusters, std::memory_order_release);
  return ASHQK_OK;
}

template <int FMT, bool SPLIT>
int launch_pair(const PairMaps& maps, const PairArgs& a, int clusters, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((SPLIT ? 4 : 2) * clusters);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = PairSmem<FMT>::bytes + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLIT ? 4 : 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fp4_pair_kernel<FMT, SPLIT>, maps, a) == cudaSuccess ? ASHQK_OK : ASHQK_ERR_CUDA;
}

std::atomic<int> g_split{0};

template <int FMT>
int run_pair(const PairMaps& maps, const PairArgs& a, cudaStream_t stream) {
  DeviceInfo dev;
  if (const int rc = device_info(&dev)) return rc;
  const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  int clusters = 0;
  const int forced = g_split.load(std::memory_order_relaxed);
  if (a.num_kb >= 2 && tiles <= dev.sm_count / 4 && (forced ? forced == 2 : a.num_kb >= kMinSplitKb)) {
    if (const int rc = resident_clusters<FMT, true>(dev, &clusters)) return rc;
    if (tiles <= clusters) return launch_pair<FMT, true>(maps, a, static_cast<int>(tiles), stream);
  }
  if (const int rc = resident_clusters<FMT, false>(dev, &clusters)) return rc;
  return launch_pair<FMT, false>(maps, a, static_cast<int>(std::min<int64_t>(clusters, tiles)), stream);
}

}  // namespace

int fp4_matmul_pair(const Fp4Product& p, cudaStream_t stream) {
  const int M = p.a.rows, N = p.b.rows;
  PairArgs a;
  a.y = p.y;
  a.y_ld = p.y_ld;
  a.M = M;
  a.N = N;
  a.k_steps = static_cast<int>(ceil_div64(fp4_padded_k(p.K), 64));
  a.num_kb = static_cast<int>(ceil_div64(fp4_padded_k(p.K), kFp4BlockK));
  a.tiles_m = ceil_div(M, 2 * kBM);
  a.tiles_n = ceil_div(N, kBN);
  if (static_cast<int64_t>(a.tiles_m) * a.tiles_n > (1 << 30)) return ASHQK_ERR_UNSUPPORTED;
  a.alpha = p.alpha;
  a.bf16 = p.dtype == ASHQK_BF16;
  a.tma_y = aligned(p.y, 16) && p.y_ld % 8 == 0;
  const uint64_t row_bytes = fp4_padded_k(p.K) / 2;
  const uint64_t scale_bytes = fp4_scale_tiles(p.K, p.format) * kFp4TileBytes;
  const uint32_t stage_scales = kFp4BlockK / fp4_block(p.format) / 4 * kFp4TileBytes;
  auto codes_map = [&](CUtensorMap* map, const Fp4Matrix& m, int box_rows) {
    return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<uint8_t*>(m.codes), row_bytes, m.rows,
                                m.ld, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  // Scale tiles as rows of 8-byte elements: one row per 128 rows of the matrix.
  auto scales_map = [&](CUtensorMap* map, const Fp4Matrix& m, int box_rows) {
    return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, const_cast<uint8_t*>(m.scales), scale_bytes / 8,
                                ceil_div(m.rows, kFp4TileRows), scale_bytes, stage_scales / 8, box_rows,
                                CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  PairMaps maps;
  int rc = codes_map(&maps.a, p.a, kBM);
  if (!rc) rc = codes_map(&maps.b, p.b, kHalfN);
  if (!rc) rc = scales_map(&maps.as, p.a, 1);
  if (!rc) rc = scales_map(&maps.bs, p.b, 2);
  if (!rc && a.tma_y)
    rc = encode_tensor_map_2d(&maps.y, CU_TENSOR_MAP_DATA_TYPE_UINT16, p.y, N, M, p.y_ld * 2, 64, 32,
                              CU_TENSOR_MAP_SWIZZLE_128B);
  else
    maps.y = maps.a;  // not used
  if (rc) return rc;
  return p.format == ASHQK_MXFP4 ? run_pair<ASHQK_MXFP4>(maps, a, stream) : run_pair<ASHQK_NVFP4>(maps, a, stream);
}

void fp4_set_pair_split(int split) { g_split.store(split, std::memory_order_relaxed); }

}  // namespace ashqk
