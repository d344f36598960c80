// y = alpha * A B^T with 4-bit operands, for any number of rows of A; made for few.
//
// The weights' rows (B, N of them) take the tensor core's 128-row side and A's rows its column side, so that
// one token wastes 7 of 8 columns instead of 127 of 128 rows, and every weight byte goes from HBM
// through shared memory to the tensor core with no instruction touching it. With few rows the floor is the
// weights' bytes: a CTA owns 128 weight rows and a slice of K, the CTAs of a cluster split K and add
// their partial sums over distributed shared memory in rank order, so a result does not depend on timing.
//
//   warp 0      one elected lane: TMA of codes, bulk copies of scale tiles
//   warp 1      one elected lane: tcgen05.cp of a stage's scales, its four MMAs, commit
//   warps 2..5  after the last MMA: TMEM -> registers -> y, or -> shared memory and the cluster's sum
//
// The scales' TMEM columns are double-buffered: stage i's copies wait for the MMAs of stage i - 2. All
// waits are bounded.
#include <algorithm>
#include <atomic>

#include "fp4_mma.cuh"

namespace ashqk {
namespace {

constexpr int kTileN = 128;  // weight rows per CTA
constexpr int kThreads = 192;

struct RowsMaps {
  CUtensorMap w, x;
};

struct RowsArgs {
  const uint8_t* ws;  // scales
  const uint8_t* xs;
  void* y;
  int64_t y_ld;
  int M, N, k_steps, num_kb, scale_tiles;  // k_steps: MMAs of 64 columns over all of K
  int cluster, ring;
  float alpha;
  int bf16;
};

template <int FMT, int NT>
struct RowsSmem {
  static constexpr int kT = Fp4Mma<FMT>::kTilesPerStage;
  static constexpr int kXTiles = NT > 128 ? 2 : 1;  // 128-row scale tiles of A's rows
  static constexpr uint32_t kW = kTileN * 128;
  static constexpr uint32_t kX = NT * 128;
  static constexpr uint32_t kWS = kT * kFp4TileBytes;
  static constexpr uint32_t kXS = kXTiles * kT * kFp4TileBytes;
  static constexpr uint32_t kStage = kW + kX + kWS + kXS;
  static constexpr uint32_t kPartial = NT * kTileN * 4;
  static_assert(kStage % 1024 == 0, "swizzle atoms need 1 KB alignment");
  static constexpr int kMaxRing = 12;
  static constexpr uint32_t kMisc = (2 * kMaxRing + 2) * 8 + 16;
  // TMEM: the sums, then two buffers of scales.
  static constexpr int kSfW = kT * 4, kSfX = kXTiles * kT * 4;
  static constexpr int kSf0 = NT < 32 ? 32 : NT;
  static constexpr int kCols = kSf0 + 2 * (kSfW + kSfX);
  static constexpr uint32_t kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kCols <= 512, "TMEM");
};

template <typename T>
__device__ __forceinline__ void store4(T* y, const float (&v)[4], int count, bool vec) {
  if (vec && count >= 4) {
    *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) y[i] = from_f32<T>(v[i]);
  }
}

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads) fp4_rows_kernel(const __grid_constant__ RowsMaps maps, const RowsArgs a) {
  using L = RowsSmem<FMT, NT>;
  using Mma = Fp4Mma<FMT>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t data = max(static_cast<uint32_t>(a.ring) * L::kStage, a.cluster > 1 ? L::kPartial : 0u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + data);
  uint64_t* empty = full + L::kMaxRing;
  uint64_t* done = empty + L::kMaxRing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 2);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // known to be uniform
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % a.cluster;
  const int tile = static_cast<int>(blockIdx.x) / a.cluster;
  const int n0 = tile * kTileN;
  const int m0 = static_cast<int>(blockIdx.y) * NT;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.num_kb) * rank / a.cluster);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.num_kb) * (rank + 1) / a.cluster);

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.ring; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&maps.w);
    prefetch_tensormap(&maps.x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish_alloc_permit();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    const int x_tiles = min(L::kXTiles, (a.M - m0 + 127) / 128);
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(&empty[stage], phase ^ 1u, abort, true)) break;
      unsigned char* base = smem + stage * L::kStage;
      const int t0 = kb * L::kT;
      const uint32_t sf = static_cast<uint32_t>(min(L::kT, a.scale_tiles - t0)) * kFp4TileBytes;
      if (elect_one()) {
        mbar_arrive_expect_tx(&full[stage], L::kW + L::kX + sf * (1 + x_tiles));
        tma_load_2d(base, &maps.w, kb * 128, n0, &full[stage]);
        bulk_load(base + L::kW + L::kX, a.ws + (static_cast<int64_t>(tile) * a.scale_tiles + t0) * kFp4TileBytes, sf, &full[stage]);
        tma_load_2d(base + L::kW, &maps.x, kb * 128, m0, &full[stage]);
        for (int t = 0; t < x_tiles; ++t)
          bulk_load(base + L::kW + L::kX + L::kWS + t * L::kWS,
                    a.xs + (static_cast<int64_t>(m0 / 128 + t) * a.scale_tiles + t0) * kFp4TileBytes, sf, &full[stage]);
      }
      __syncwarp();
      ++issued;
      if (++stage == a.ring) {
        stage = 0;
        phase ^= 1u;
      }
    }
    for (int i = 1; i <= a.ring && i <= issued; ++i) {
      const int f = issued - i;
      mbar_drain(&full[f % a.ring], static_cast<uint32_t>(f / a.ring) & 1u);
    }
  } else if (warp == 1) {
    int stage = 0, old = 0;  // stage of kb, of kb - 2
    uint32_t phase = 0, old_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0;
      if (!mbar_wait(&full[stage], phase, abort, true)) break;
      if (i >= 2) {
        if (!mbar_wait(&empty[old], old_phase, abort, true)) break;
        if (++old == a.ring) {
          old = 0;
          old_phase ^= 1u;
        }
      }
      tc_fence_after_sync();
      const uint32_t base = sbase + stage * L::kStage;
      const uint32_t sfw = tmem + L::kSf0 + (i & 1) * (L::kSfW + L::kSfX);
      const uint32_t sfx = sfw + L::kSfW;
      const uint64_t sd = scale_tile_desc(base + L::kW + L::kX);
      const uint64_t dw = umma_desc_sw128(base, 16u, 1024u);
      const uint64_t dx = umma_desc_sw128(base + L::kW, 16u, 1024u);
      const int steps = min(4, a.k_steps - kb * 4);
      const int tiles = Mma::tile_of(steps - 1) + 1;
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < L::kT; ++t) {
          if (t >= tiles) break;
          scale_tile_to_tmem(sfw + t * 4, sd + t * (kFp4TileBytes >> 4));
#pragma unroll
          for (int r = 0; r < L::kXTiles; ++r)
            scale_tile_to_tmem(sfx + (t * L::kXTiles + r) * 4, sd + (((1 + r) * L::kWS + t * kFp4TileBytes) >> 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= steps) break;
          Mma::mma(tmem, dw + 2 * j, dx + 2 * j, Mma::idesc(kTileN, NT, j), sfw + Mma::tile_of(j) * 4,
                   sfx + Mma::tile_of(j) * L::kXTiles * 4, (i | j) != 0);
        }
        umma_commit(&empty[stage]);
        if (kb + 1 == kb1) umma_commit(done);
      }
      __syncwarp();
      if (++stage == a.ring) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (*abort) {  // the commit above may not have been reached
      if (elect_one()) umma_commit(done);
      __syncwarp();
    }
    mbar_drain(done, 0);
  } else {
    const int quad = warp & 3;
    const bool ok = mbar_wait(done, 0, abort);
    tc_fence_after_sync();
    const int row = 32 * quad + lane;  // weight row of the tile
    const int n = n0 + row;
    float* partial = reinterpret_cast<float*>(smem);
    const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * quad) << 16);
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < NT; c += 8) {
        if (m0 + c >= a.M) break;
        uint32_t r[8];
        tmem_ld_32x32b_x8(taddr + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int m = m0 + c + i;
          if (m >= a.M) break;
          if (a.cluster > 1) {
            partial[(c + i) * kTileN + row] = __uint_as_float(r[i]);
          } else if (n < a.N) {
            const float v = a.alpha * __uint_as_float(r[i]);
            if (a.bf16)
              static_cast<__nv_bfloat16*>(a.y)[m * a.y_ld + n] = __float2bfloat16_rn(v);
            else
              static_cast<__half*>(a.y)[m * a.y_ld + n] = __float2half_rn(v);
          }
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  // TMEM goes back before the CTA waits for its cluster: a CTA that holds it waits for nobody, so CTAs of
  // several clusters that share SMs cannot block one another in the allocation.
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, L::kTmemCols);
  }
  if (a.cluster > 1) {
    // Partial sums of every CTA are in its shared memory, whose ring is drained. Each rank adds and stores a
    // share of the tile.
    cluster_sync();
    const bool vec = (a.y_ld & 3) == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7) == 0;
    const int quads = min(NT, a.M - m0) * (kTileN / 4);
    for (int q = rank * kThreads + static_cast<int>(threadIdx.x); q < quads; q += a.cluster * kThreads) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < a.cluster; ++r) {
        const float4 p = ld_shared_cluster_v4(map_shared_rank(smem + q * 16, r));
        s[0] += p.x, s[1] += p.y, s[2] += p.z, s[3] += p.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] *= a.alpha;
      const int m = m0 + q / (kTileN / 4);
      const int n = n0 + q % (kTileN / 4) * 4;
      if (n < a.N) {
        if (a.bf16)
          store4(static_cast<__nv_bfloat16*>(a.y) + m * a.y_ld + n, s, a.N - n, vec);
        else
          store4(static_cast<__half*>(a.y) + m * a.y_ld + n, s, a.N - n, vec);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its partial sums
  }
}

template <int FMT, int NT>
int launch_rows(const RowsMaps& maps, RowsArgs a, cudaStream_t stream) {
  using L = RowsSmem<FMT, NT>;
  DeviceInfo dev;
  if (const int rc = device_info(&dev)) return rc;
  const int tiles = ceil_div(a.N, kTileN);
  const int cols = ceil_div(a.M, NT);
  if (cols > 65535) return ASHQK_ERR_UNSUPPORTED;
  // CTAs resident per SM by TMEM (512 columns), at most 2.
  const int per_sm = L::kTmemCols <= 256 ? 2 : 1;
  const int slots = dev.sm_count * per_sm;
  a.cluster = std::max(1, std::min({8, a.num_kb, slots / std::max(1, tiles * cols)}));
  const int local = ceil_div(a.num_kb, a.cluster);
  const uint32_t budget = per_sm == 2 ? 110 * 1024 : 220 * 1024;
  a.ring = std::max(2, std::min({L::kMaxRing, local, static_cast<int>(budget / L::kStage)}));
  const size_t smem = std::max<size_t>(a.ring * L::kStage, a.cluster > 1 ? L::kPartial : 0) + L::kMisc + 1024;
  auto kernel = fp4_rows_kernel<FMT, NT>;
  static std::atomic<bool> configured[64];  // zero-initialised (static storage)
  if (!configured[dev.device].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(dev.max_smem_optin)) != cudaSuccess)
      return ASHQK_ERR_CUDA;
    configured[dev.device].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * a.cluster, cols);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, maps, a) == cudaSuccess ? ASHQK_OK : ASHQK_ERR_CUDA;
}

template <int FMT>
int launch_rows_fmt(const RowsMaps& maps, const RowsArgs& a, int nt, cudaStream_t stream) {
  switch (nt) {
    case 8: return launch_rows<FMT, 8>(maps, a, stream);
    case 16: return launch_rows<FMT, 16>(maps, a, stream);
    case 32: return launch_rows<FMT, 32>(maps, a, stream);
    case 64: return launch_rows<FMT, 64>(maps, a, stream);
    case 128: return launch_rows<FMT, 128>(maps, a, stream);
    default: return launch_rows<FMT, 256>(maps, a, stream);
  }
}

}  // namespace

int fp4_matmul_rows(const void* a_codes, int64_t a_ld, const void* a_scales, const void* b_codes, int64_t b_ld,
                    const void* b_scales, void* y, int64_t y_ld, int dtype, int M, int N, int K, int format, float alpha,
                    cudaStream_t stream) {
  int nt = 8;
  while (nt < M && nt < 256) nt *= 2;
  RowsMaps maps;
  const uint64_t row_bytes = fp4_padded_k(K) / 2;
  int rc = encode_tensor_map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<void*>(b_codes), row_bytes, N, b_ld,
                                128, kTileN, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc)
    rc = encode_tensor_map_2d(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<void*>(a_codes), row_bytes, M, a_ld, 128,
                              nt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  RowsArgs a;
  a.ws = static_cast<const uint8_t*>(b_scales);
  a.xs = static_cast<const uint8_t*>(a_scales);
  a.y = y;
  a.y_ld = y_ld;
  a.M = M;
  a.N = N;
  a.k_steps = static_cast<int>(ceil_div64(fp4_padded_k(K), 64));
  a.num_kb = static_cast<int>(ceil_div64(fp4_padded_k(K), kFp4BlockK));
  a.scale_tiles = static_cast<int>(fp4_scale_tiles(K, format));
  a.alpha = alpha;
  a.bf16 = dtype == ASHQK_BF16;
  return format == ASHQK_MXFP4 ? launch_rows_fmt<ASHQK_MXFP4>(maps, a, nt, stream)
                               : launch_rows_fmt<ASHQK_NVFP4>(maps, a, nt, stream);
}

}  // namespace ashqk
