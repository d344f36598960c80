// y = alpha * A B^T with 4-bit operands, for any number of rows of A; made for few. A comes quantised, or
// (up to 32 rows) in 16 bits and is quantised here.
//
// The weights' rows (B, N of them) take the tensor core's 128-row side and A's rows its column side, so that
// one token wastes 7 of 8 columns instead of 127 of 128 rows, and every weight byte goes from HBM
// through shared memory to the tensor core with no instruction touching it. With few rows the floor is the
// weights' bytes: a CTA owns 128 weight rows and a slice of K, the CTAs of a cluster split K and add
// their partial sums in rank order, so a result does not depend on timing.
//
//   warp 0      one elected lane: prefetches its weights into L2 before the previous kernel has ended
//               (L2 is coherent, so what that kernel may still write is not missed), then TMA of codes and
//               bulk copies of scale tiles
//   warp 1      one elected lane: tcgen05.cp of a stage's scales, its four MMAs, commit
//   warps 2..9  fused form: quantise this CTA's slice of A into shared memory, in the layout in which TMA and
//               the scale tiles arrive otherwise; then all: TMEM -> registers -> y, or, with a split K,
//               -> the shared memory of the CTA that adds these rows of A, counted in bytes on its barrier
//               (st.async, or with 32 columns and more through own shared memory and bulk copies)
//
// Measured on a B200, launches back to back in a graph, weights from HBM, x in fp16, MXFP4: one token 4096->6144 5.0 us,
// 4096->4096 4.7, 4096->24576 12.1 (4.4 TB/s of weights), 12288->4096 8.9; sixteen 6.6, 6.0, 15.4, 10.8. A launch is
// latency from end to end (one token 4096->6144): 0.75 us until x is quantised, 0.35 per stage, 1 for the exchange, 1 to
// the next launch's start.
//
// The scales have two to eight buffers in TMEM: the copies of stage i wait for the MMAs of stage i - buffers. With
// two, that wait and not the tensor core set the pace of narrow tiles. All waits are bounded.
#include <algorithm>
#include <atomic>

#include "fp4_mma.cuh"

namespace ashqk {
namespace {

constexpr int kTileN = 128;  // weight rows per CTA
constexpr int kQuantWarps = 8;
constexpr int kThreads = 64 + 32 * kQuantWarps;
constexpr int kMaxRing = 12;
constexpr int kMaxCluster = 8;

struct RowsMaps {
  CUtensorMap w, x;
};

struct RowsArgs {
  const uint8_t* ws;  // scales
  const uint8_t* xs;  // scales of a quantised A
  const void* x;      // A in 16 bits (fused)
  int64_t x_ld;
  void* y;
  int64_t y_ld;
  int M, N, K, k_steps, num_kb, scale_tiles;  // k_steps: MMAs of 64 columns over all of K
  int cluster, ring;
  uint32_t off_x, off_slots, off_bar;  // shared memory after the ring
  float alpha;
  Fp4Quant xq;
  int bf16, gated;
  int align;  // of 16-column chunks of a 16-bit A
};

template <int FMT, int NT, bool FUSED>
struct RowsShape {
  static constexpr int kT = Fp4Mma<FMT>::kTilesPerStage;
  static constexpr uint32_t kW = kTileN * 128;
  static constexpr uint32_t kWS = kT * kFp4TileBytes;
  static constexpr uint32_t kX = NT * 128;
  static constexpr uint32_t kXS = kT * kFp4TileBytes;
  static constexpr uint32_t kStage = kW + kWS + (FUSED ? 0 : kX + kXS);
  static_assert(kStage % 1024 == 0, "swizzle atoms need 1 KB alignment");
  // Fused: the quantised slice, [stage][row][128] and after it the scale tiles, of which only the first NT rows
  // are there: the copy to TMEM reads on into the next tile, for rows that nobody uses.
  static constexpr uint32_t kXSTile = NT * 16;
  // TMEM: the sums, then as many buffers of scales as fit.
  static constexpr int kSfW = kT * 4, kSfX = kT * 4;
  static constexpr int kSf0 = NT < 32 ? 32 : NT;
  static constexpr uint32_t kTmemCols = NT <= 64 ? 128 : 256;
  static constexpr int kSfBufs = (static_cast<int>(kTmemCols) - kSf0) / (kSfW + kSfX);
  static_assert(kSfBufs >= 2, "TMEM");
  // Split K: whether the slots for partial sums have shared memory of their own or take the ring's, and whether
  // the sums go there by way of the own ring.
  static constexpr bool kOwnSlots = NT <= 32;
  static constexpr bool kStaged = NT >= 32;
  static_assert(kOwnSlots || kStaged, "this CTA's own sums need a place");
  static constexpr uint32_t kStaging = NT / 4 * kTileN * 16;
  static constexpr uint32_t slots(int cluster) {
    return static_cast<uint32_t>(((NT / 4 + cluster - 1) / cluster) * cluster) * kTileN * 16;
  }
};

__device__ __forceinline__ void l2_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void l2_prefetch(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(reinterpret_cast<uint64_t>(p)), "r"(bytes)
               : "memory");
}

// Quantises columns [256 kb0, 256 kb1) of A's rows into shared memory, sixteen columns per thread, as the quantiser
// proper does.
template <int FMT, int NT, typename T, bool GATED>
__device__ __forceinline__ void quantize_slice(const RowsArgs& a, int kb0, int kb1, uint32_t codes, uint32_t scales,
                                               int tid) {
  using L = RowsShape<FMT, NT, true>;
  constexpr int kLanes = fp4_block(FMT) / 16;
  constexpr int kBatch = GATED ? 1 : 2;  // chunks whose loads are in flight together
  constexpr int kStep = 32 * kQuantWarps;
  const int chunks = (kb1 - kb0) * 16;  // of a row
  const int total = a.M * chunks;
  const T* x = static_cast<const T*>(a.x);
  for (int i0 = tid; (i0 & ~31) < total; i0 += kBatch * kStep) {  // whole warps
    Raw16<T> g[kBatch], u[GATED ? kBatch : 1];
    int row[kBatch], chunk[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kStep;
      row[b] = i / chunks;
      chunk[b] = i - row[b] * chunks;
      const int k0 = kb0 * kFp4BlockK + chunk[b] * 16;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[b].w[j] = 0;
        if (GATED) u[b].w[j] = 0;
      }
      if (i < total && k0 < a.K) {
        const T* p = x + row[b] * a.x_ld + k0;
        const int align = k0 + 16 <= a.K ? a.align : 0;
        load16<T>(p, a.K - k0, align, g[b]);
        if (GATED) load16<T>(p + a.K, a.K - k0, align, u[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (((i0 + b * kStep) & ~31) >= total) break;  // whole warps
      float v[16];
      unpack16<T>(g[b], v);
      uint32_t amax;
      if constexpr (GATED) {
        float w[16];
        unpack16<T>(u[b], w);
        silu_mul16(v, w);
        amax = abs_max16(v);
      } else {
        amax = abs_max16(g[b]);
      }
      uint2 c;
      const uint32_t byte = fp4_quantize16<FMT>(v, amax, a.xq, &c);
      if (i0 + b * kStep < total) {
        const int m = row[b], kb = chunk[b] >> 4, cc = chunk[b] & 15;
        const uint32_t at =
            codes + kb * L::kX + (m >> 3) * 1024 + (m & 7) * 128 + (((cc >> 1) ^ (m & 7)) << 4) + (cc & 1) * 8;
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(c.x), "r"(c.y) : "memory");
        if (cc % kLanes == 0) {
          const int block = cc / kLanes;
          const uint32_t s = scales + (kb * L::kT + (block >> 2)) * L::kXSTile + m * 16 + (block & 3);
          asm volatile("st.shared.u8 [%0], %1;" ::"r"(s), "r"(byte) : "memory");
        }
      }
    }
  }
}

template <int FMT, int NT, bool FUSED>
__global__ void __launch_bounds__(kThreads, 3) fp4_rows_kernel(const __grid_constant__ RowsMaps maps, const RowsArgs a) {
  using L = RowsShape<FMT, NT, FUSED>;
  using Mma = Fp4Mma<FMT>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + a.off_bar);
  uint64_t* empty = full + kMaxRing;
  uint64_t* done = empty + kMaxRing;
  uint64_t* x_ready = done + 1;
  uint64_t* received = x_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // known to be uniform
  const int lane = threadIdx.x & 31;
  const int C = a.cluster;
  const int rank = static_cast<int>(blockIdx.x) % C;
  const int tile = static_cast<int>(blockIdx.x) / C;
  const int n0 = tile * kTileN;
  const int m0 = static_cast<int>(blockIdx.y) * NT;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.num_kb) * rank / C);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.num_kb) * (rank + 1) / C);
  const uint8_t* ws = a.ws + static_cast<int64_t>(tile) * a.scale_tiles * kFp4TileBytes;
  // Groups of four rows of A; group g's partial sums are added by the CTA of rank g % C.
  const int groups = (min(NT, a.M - m0) + 3) / 4;
  const int my_groups = (groups - rank + C - 1) / C;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.ring; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(x_ready, kQuantWarps);
    mbar_init(received, 1);
    *abort = 0;
    fence_mbarrier_init();
    if (C > 1) mbar_arrive_expect_tx(received, static_cast<uint32_t>(my_groups * (C - 1)) * kTileN * 16);
  }
  __syncthreads();
  // This CTA's barriers can be signalled (waited for before the first remote store). Before the allocation, which
  // can wait for CTAs of other clusters on this SM.
  if (C > 1) cluster_arrive();
  if (warp == 0 && elect_one()) {
    prefetch_tensormap(&maps.w);
    const int last = min(kb1, kb0 + 32);
    for (int kb = kb0; kb < last; ++kb) l2_prefetch_2d(&maps.w, kb * 128, n0);
    const int t0 = kb0 * L::kT, t1 = min(last * L::kT, a.scale_tiles);
    l2_prefetch(ws + static_cast<int64_t>(t0) * kFp4TileBytes, (t1 - t0) * kFp4TileBytes);
    if (!FUSED) prefetch_tensormap(&maps.x);
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
  // Behind the wait: what ran before this grid has then ended, also for a next launch that reads ahead of its own wait
  // (the decode GEMV loads its weights there). And behind the allocation: a CTA of the next launch that holds TMEM on
  // this SM waits for this grid, which must not still be waiting for TMEM.
  pdl_launch_dependents();

  const uint32_t x_codes = sbase + a.off_x;
  const uint32_t x_scales = x_codes + static_cast<uint32_t>(kb1 - kb0) * L::kX;

  if (warp == 0) {
    const uint8_t* xs = a.xs + static_cast<int64_t>(m0 / kFp4TileRows) * a.scale_tiles * kFp4TileBytes;
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(&empty[stage], phase ^ 1u, abort, true)) break;
      unsigned char* base = smem + stage * L::kStage;
      const int t0 = kb * L::kT;
      const uint32_t sf = static_cast<uint32_t>(min(L::kT, a.scale_tiles - t0)) * kFp4TileBytes;
      if (elect_one()) {
        mbar_arrive_expect_tx(&full[stage], L::kW + sf + (FUSED ? 0 : L::kX + sf));
        tma_load_2d(base, &maps.w, kb * 128, n0, &full[stage]);
        bulk_load(base + L::kW, ws + static_cast<int64_t>(t0) * kFp4TileBytes, sf, &full[stage]);
        if (!FUSED) {
          tma_load_2d(base + L::kW + L::kWS, &maps.x, kb * 128, m0, &full[stage]);
          bulk_load(base + L::kW + L::kWS + L::kX, xs + static_cast<int64_t>(t0) * kFp4TileBytes, sf, &full[stage]);
        }
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
    int stage = 0, old = 0, buf = 0;  // stage of kb, of kb - kSfBufs; scale buffer
    uint32_t phase = 0, old_phase = 0;
    bool ok = !FUSED || mbar_wait(x_ready, 0, abort, true);
    for (int kb = kb0; ok && kb < kb1; ++kb) {
      const int i = kb - kb0;
      if (!mbar_wait(&full[stage], phase, abort, true)) {
        ok = false;
        break;
      }
      // (In a ring of no more stages than buffers the wait above has seen to it: the producer waited for stage
      // i - ring.)
      if (L::kSfBufs < a.ring && i >= L::kSfBufs) {
        if (!mbar_wait(&empty[old], old_phase, abort, true)) {
          ok = false;
          break;
        }
        if (++old == a.ring) {
          old = 0;
          old_phase ^= 1u;
        }
      }
      tc_fence_after_sync();
      const uint32_t base = sbase + stage * L::kStage;
      const uint32_t sfw = tmem + L::kSf0 + buf * (L::kSfW + L::kSfX);
      if (++buf == L::kSfBufs) buf = 0;
      const uint32_t sfx = sfw + L::kSfW;
      const uint64_t sd = scale_tile_desc(base + L::kW);
      const uint64_t sx = scale_tile_desc(FUSED ? x_scales + i * L::kT * L::kXSTile : base + L::kW + L::kWS + L::kX);
      const uint64_t dw = umma_desc_sw128(base, 16u, 1024u);
      const uint64_t dx = umma_desc_sw128(FUSED ? x_codes + i * L::kX : base + L::kW + L::kWS, 16u, 1024u);
      const int steps = min(4, a.k_steps - kb * 4);
      const int tiles = Mma::tile_of(steps - 1) + 1;
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < L::kT; ++t) {
          if (t >= tiles) break;
          scale_tile_to_tmem(sfw + t * 4, sd + t * (kFp4TileBytes >> 4));
          scale_tile_to_tmem(sfx + t * 4, sx + t * ((FUSED ? L::kXSTile : kFp4TileBytes) >> 4));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= steps) break;
          Mma::mma(tmem, dw + 2 * j, dx + 2 * j, Mma::idesc(kTileN, NT, j), sfw + Mma::tile_of(j) * 4,
                   sfx + Mma::tile_of(j) * 4, (i | j) != 0);
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
    if (!ok) {  // the commit of the last stage was not reached
      if (elect_one()) umma_commit(done);
      __syncwarp();
    }
    mbar_drain(done, 0);
  } else if (FUSED) {
    const int tid = static_cast<int>(threadIdx.x) - 64;
    if (a.gated) {
      if (a.bf16)
        quantize_slice<FMT, NT, __nv_bfloat16, true>(a, kb0, kb1, x_codes, x_scales, tid);
      else
        quantize_slice<FMT, NT, __half, true>(a, kb0, kb1, x_codes, x_scales, tid);
    } else {
      if (a.bf16)
        quantize_slice<FMT, NT, __nv_bfloat16, false>(a, kb0, kb1, x_codes, x_scales, tid);
      else
        quantize_slice<FMT, NT, __half, false>(a, kb0, kb1, x_codes, x_scales, tid);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(x_ready);
  }

  // ---- sums: warps 2..9, one lane per weight row; the two warps of a lane quarter take turns ----
  const bool epilogue = warp >= 2;
  const int turn = (warp - 2) >> 2;
  const int row = 32 * (warp & 3) + lane;
  const int n = n0 + row;
  bool ok = false;
  if (epilogue) {
    ok = mbar_wait(done, 0, abort);
    tc_fence_after_sync();
  }
  // Slots: [group of this rank][sender][weight row] x 16 bytes. Staging: [group][weight row] x 16 bytes.
  const uint32_t slots = sbase + (L::kOwnSlots ? a.off_slots : L::kStaging);
  auto slot = [&](int l, int from) { return slots + static_cast<uint32_t>((l * C + from) * kTileN + row) * 16; };
  if (C > 1 && !L::kStaged) {
    __syncwarp();
    cluster_wait();
  }
  // Four sums of consecutive rows of A -> y. Lanes are consecutive columns of y: 64 bytes per row and warp.
  auto store4 = [&](int m, float v0, float v1, float v2, float v3) {
    if (n >= a.N) return;
    uint16_t* y = static_cast<uint16_t*>(a.y) + m * a.y_ld + n;
    v0 *= a.alpha, v1 *= a.alpha, v2 *= a.alpha, v3 *= a.alpha;
    const uint32_t lo = a.bf16 ? pack2<__nv_bfloat16>(v0, v1) : pack2<__half>(v0, v1);
    const uint32_t hi = a.bf16 ? pack2<__nv_bfloat16>(v2, v3) : pack2<__half>(v2, v3);
    if (m < a.M) y[0] = static_cast<uint16_t>(lo);
    if (m + 1 < a.M) y[a.y_ld] = static_cast<uint16_t>(lo >> 16);
    if (m + 2 < a.M) y[2 * a.y_ld] = static_cast<uint16_t>(hi);
    if (m + 3 < a.M) y[3 * a.y_ld] = static_cast<uint16_t>(hi >> 16);
  };
  if (epilogue) {
    constexpr int kCols = NT < 32 ? 8 : 32;  // columns of one TMEM load
    const uint32_t taddr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
#pragma unroll 1
    for (int g0 = turn * (kCols / 4); g0 < groups; g0 += 2 * (kCols / 4)) {
      uint32_t r[kCols];
      if constexpr (kCols == 8)
        tmem_ld_32x32b_x8(taddr + 4 * g0, r);
      else
        tmem_ld_32x32b_x32(taddr + 4 * g0, r);
      tmem_wait_ld();
      if (!ok) {  // a wait ran out: the sums are not there; peers still get the bytes that they count
#pragma unroll
        for (int i = 0; i < kCols; ++i) r[i] = 0x7fffffffu;
      }
#pragma unroll
      for (int h = 0; h < kCols / 4; ++h) {
        const int g = g0 + h;
        if (g >= groups) break;
        if (C == 1) {
          store4(m0 + 4 * g, __uint_as_float(r[4 * h]), __uint_as_float(r[4 * h + 1]), __uint_as_float(r[4 * h + 2]),
                 __uint_as_float(r[4 * h + 3]));
        } else {
          const int l = g / C, owner = g - l * C;
          const uint4 v = make_uint4(r[4 * h], r[4 * h + 1], r[4 * h + 2], r[4 * h + 3]);
          if (owner == rank && L::kOwnSlots)
            sts_v4(slot(l, rank), v);
          else if (L::kStaged)
            sts_v4(sbase + static_cast<uint32_t>(g * kTileN + row) * 16, v);
          else
            st_async_v4(map_rank(slot(l, rank), owner), v, map_rank(smem_u32(received), owner));
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
  if (C > 1) {
    __syncwarp();
    if (L::kStaged) {
      cluster_wait();
      if (!L::kOwnSlots) cluster_sync();  // every CTA of the cluster is through with its ring
      if (epilogue) {  // each warp sends the 512 bytes of every group that it has written
        constexpr int kPer = 8;  // groups of one TMEM load
        fence_proxy_async_smem();
        __syncwarp();
        const uint32_t first = static_cast<uint32_t>(row - lane) * 16;
        for (int g = lane; g < groups; g += 32) {
          const int l = g / C, owner = g - l * C;
          if (((g / kPer) & 1) != turn || owner == rank) continue;
          const uint32_t to = slots + static_cast<uint32_t>((l * C + rank) * kTileN) * 16 + first;
          bulk_to_cluster(map_rank(to, owner), sbase + static_cast<uint32_t>(g * kTileN) * 16 + first, 512,
                          map_rank(smem_u32(received), owner));
        }
        __syncwarp();
      }
    }
    // The last barrier: no CTA leaves while another may still store into it, nor while a copy still reads what it sent.
    // st.async takes its values from registers: issued, then arrived. A bulk copy reads the sender's shared memory until
    // its bytes are counted, and only the receiver sees that: there every CTA arrives behind its own receipt, so that
    // the barrier stands for all receipts and with them for every copy of every sender.
    if (!L::kStaged) cluster_arrive();
    const bool received_all = epilogue && my_groups > 0 && mbar_wait_cluster(received, 0, abort);
    if (L::kStaged) {
      __syncwarp();
      cluster_arrive();
    }
    if (received_all) {
#pragma unroll 2
      for (int l = turn; l < my_groups; l += 2) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int c = 0; c < C; ++c) {
          // without slots of its own, this CTA's sums are still where they were staged
          const bool staged = !L::kOwnSlots && c == rank;
          const uint4 p = lds_v4(staged ? sbase + static_cast<uint32_t>((l * C + rank) * kTileN + row) * 16 : slot(l, c));
          s[0] += __uint_as_float(p.x), s[1] += __uint_as_float(p.y);
          s[2] += __uint_as_float(p.z), s[3] += __uint_as_float(p.w);
        }
        store4(m0 + 4 * (l * C + rank), s[0], s[1], s[2], s[3]);
      }
    }
    __syncwarp();
    cluster_wait();
  }
}

std::atomic<int> g_cluster{0}, g_ring{0};

struct RowsPlan {
  int cluster, ring;
  uint32_t off_x, off_slots, off_bar, smem;
};

// CTAs per cluster and stages in flight for `tiles` tiles of 128 weight rows (times the row blocks of A). Measured on
// layers of 4096 columns and 32 to 192 tiles, every cluster size, launches back to back in a graph. What a split saves is
// a CTA's serial run over its stages; what it costs, beyond 1.35 CTAs per SM, is the room in which the next launch's CTAs
// start early: 32 tiles at one row 7.1 us with one CTA per cluster, 4.5 with 4, 4.8 with 6, 6.0 with 7; 48 tiles 7.1, 5.1
// with 4, 6.5 with 6. With more tiles than SMs a split in two evens out the last wave (192 tiles: 12.9 -> 12.2 us). With
// 12288 columns and more the run weighs more than the room, which this rule does not see: 32 tiles 8.8 us with its 6 CTAs,
// 7.5 with 7; 48 tiles 12.7 with its 4, 10.0 with 6.
template <int FMT, int NT, bool FUSED>
RowsPlan plan_rows(int tiles, int num_kb, int sm_count) {
  using L = RowsShape<FMT, NT, FUSED>;
  RowsPlan p;
  // 128 rows of A: the staged sums leave room for one CTA per SM, and clusters of those do not fill every SM (2048
  // columns of K and rows of B in clusters of eight: 15.8 us in two waves).
  const int ctas = NT > 64 ? sm_count * 9 / 10 : sm_count * 27 / 20;
  p.cluster = std::max(1, std::min({NT > 64 ? 4 : kMaxCluster, num_kb, ctas / std::max(1, tiles)}));
  if (p.cluster == 1 && L::kOwnSlots && num_kb >= 4 && tiles > sm_count && tiles <= ctas) p.cluster = 2;
  auto x_area = [&] {  // this CTA's slice of A, quantised
    return FUSED ? ceil_div(num_kb, p.cluster) * (L::kX + L::kT * L::kXSTile) + kFp4TileBytes : 0u;
  };
  while (p.cluster < std::min(kMaxCluster, num_kb) && x_area() > 64 * 1024) ++p.cluster;
  if (const int c = g_cluster.load(std::memory_order_relaxed)) p.cluster = std::min(c, num_kb);
  const int local = ceil_div(num_kb, p.cluster);
  const uint32_t x_bytes = x_area();
  const uint32_t slots = p.cluster > 1 ? L::slots(p.cluster) : 0;
  // Shared memory for the ring: a third of an SM for narrow tiles that split K (this launch's CTAs and the next's
  // are resident together), half of one otherwise.
  const uint32_t budget = (L::kOwnSlots && p.cluster > 1 ? 72 : 108) * 1024;
  const uint32_t fixed = x_bytes + (L::kOwnSlots ? slots : 0);
  p.ring = fixed + 2 * L::kStage > budget ? 2 : static_cast<int>((budget - fixed) / L::kStage);
  p.ring = std::max(2, std::min({kMaxRing, local, p.ring}));
  if (const int r = g_ring.load(std::memory_order_relaxed)) {
    constexpr uint32_t kMost = 222 * 1024;
    p.ring = std::max(2, std::min({r, local, static_cast<int>((kMost - std::min(fixed, kMost)) / L::kStage)}));
  }
  uint32_t ring = p.ring * L::kStage;
  if (p.cluster > 1 && L::kStaged)
    ring = std::max(ring, (L::kStaging + (L::kOwnSlots ? 0 : slots) + 1023) / 1024 * 1024);
  p.off_x = ring;
  p.off_slots = (p.off_x + x_bytes + 15) / 16 * 16;
  p.off_bar = (p.off_slots + (L::kOwnSlots ? slots : 0) + 7) / 8 * 8;
  p.smem = p.off_bar + (2 * kMaxRing + 3) * 8 + 16 + 1024;
  return p;
}

template <int FMT, int NT, bool FUSED>
int launch_rows(const RowsMaps& maps, RowsArgs a, cudaStream_t stream) {
  DeviceInfo dev;
  if (const int rc = device_info(&dev)) return rc;
  const int tiles = ceil_div(a.N, kTileN);
  const int cols = ceil_div(a.M, NT);
  if (cols > 65535) return ASHQK_ERR_UNSUPPORTED;
  const RowsPlan p = plan_rows<FMT, NT, FUSED>(tiles * cols, a.num_kb, dev.sm_count);
  if (p.smem > dev.max_smem_optin) return ASHQK_ERR_UNSUPPORTED;
  a.cluster = p.cluster;
  a.ring = p.ring;
  a.off_x = p.off_x;
  a.off_slots = p.off_slots;
  a.off_bar = p.off_bar;
  auto kernel = fp4_rows_kernel<FMT, NT, FUSED>;
  static std::atomic<bool> configured[64];  // zero-initialised (static storage)
  if (!configured[dev.device].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(dev.max_smem_optin)) != cudaSuccess)
      return ASHQK_ERR_CUDA;
    configured[dev.device].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * a.cluster, cols);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = p.smem;
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
int launch_rows_fmt(const RowsMaps& maps, const RowsArgs& a, int nt, bool fused, cudaStream_t stream) {
  if (fused)
    return nt == 8    ? launch_rows<FMT, 8, true>(maps, a, stream)
           : nt == 16 ? launch_rows<FMT, 16, true>(maps, a, stream)
                      : launch_rows<FMT, 32, true>(maps, a, stream);
  switch (nt) {
    case 8: return launch_rows<FMT, 8, false>(maps, a, stream);
    case 16: return launch_rows<FMT, 16, false>(maps, a, stream);
    case 32: return launch_rows<FMT, 32, false>(maps, a, stream);
    case 64: return launch_rows<FMT, 64, false>(maps, a, stream);
    default: return launch_rows<FMT, 128, false>(maps, a, stream);
  }
}

int encode_rows(CUtensorMap* map, const Fp4Matrix& m, int K, int box_rows) {
  return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, const_cast<uint8_t*>(m.codes), fp4_padded_k(K) / 2,
                              m.rows, m.ld, 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

int rows_args(RowsArgs& a, RowsMaps& maps, const Fp4Product& p) {
  a.ws = p.b.scales;
  a.y = p.y;
  a.y_ld = p.y_ld;
  a.M = p.a.rows;
  a.N = p.b.rows;
  a.K = p.K;
  a.k_steps = static_cast<int>(ceil_div64(fp4_padded_k(p.K), 64));
  a.num_kb = static_cast<int>(ceil_div64(fp4_padded_k(p.K), kFp4BlockK));
  a.scale_tiles = static_cast<int>(fp4_scale_tiles(p.K, p.format));
  a.alpha = p.alpha;
  a.bf16 = p.dtype == ASHQK_BF16;
  return encode_rows(&maps.w, p.b, p.K, kTileN);
}

}  // namespace

int fp4_matmul_rows(const Fp4Product& p, cudaStream_t stream) {
  int nt = 8;
  while (nt < p.a.rows && nt < 128) nt *= 2;
  RowsMaps maps;
  RowsArgs a = {};
  int rc = rows_args(a, maps, p);
  if (!rc) rc = encode_rows(&maps.x, p.a, p.K, nt);
  if (rc) return rc;
  a.xs = p.a.scales;
  return p.format == ASHQK_MXFP4 ? launch_rows_fmt<ASHQK_MXFP4>(maps, a, nt, false, stream)
                                 : launch_rows_fmt<ASHQK_NVFP4>(maps, a, nt, false, stream);
}

// Whether w4a4_linear quantises x inside the product: up to 32 rows, of a length whose slice fits beside the ring (an
// eighth of it at most 48 KB), and where every 128 weight rows quantising x anew costs less than a launch for it.
// Measured (MXFP4, us, fused against two launches, in a graph): up to 16 rows, at M K tiles = 6.3 million 13.1 / 15.8 (8
// rows 4096->24576) and 10.8 / 11.6 (16 rows 12288->4096), at 12.6 million 15.4 / 16.1 (16 rows 4096->24576; NVFP4 16.8 /
// 17.2); with the wider instruction of 32 rows 8.9 / 9.6 at 4.2 million (4096->4096) and 10.1 / 10.1 at 6.3 million
// (4096->6144). A gated value costs two loads, an exponential and a quotient more and counts three times (12288->4096: 4
// rows 9.8 / 11.2, 8 rows 11.7 / 11.5).
bool fp4_fused_ok(int M, int N, int K, bool gated) {
  const int64_t work = static_cast<int64_t>(M) * K * ceil_div(N, kTileN) * (gated ? 3 : 1);
  return M <= 16 ? K <= 32768 && work <= (1 << 24) : M <= 32 && K <= 16384 && work <= (6 << 20);
}

int fp4_linear_rows(const Fp4Source& x, const Fp4Product& p, cudaStream_t stream) {
  RowsMaps maps;
  RowsArgs a = {};
  if (const int rc = rows_args(a, maps, p)) return rc;
  maps.x = maps.w;  // not used
  a.x = x.x;
  a.x_ld = x.ld;
  a.xq = fp4_quant_params(x.gs);
  a.gated = x.gated;
  a.align = std::min(chunk_align(x.x, x.ld, 2), x.gated ? chunk_align(nullptr, p.K, 2) : 32);
  const int M = p.a.rows;
  const int nt = M <= 8 ? 8 : M <= 16 ? 16 : 32;
  return p.format == ASHQK_MXFP4 ? launch_rows_fmt<ASHQK_MXFP4>(maps, a, nt, true, stream)
                                 : launch_rows_fmt<ASHQK_NVFP4>(maps, a, nt, true, stream);
}

}  // namespace ashqk

extern "C" int ashqk_fp4_set_tuning(int cluster, int ring, int split) {
  if (split < 0 || split > 2) return ASHQK_ERR_INVALID_ARGUMENT;
  if (cluster < 0 || cluster > ashqk::kMaxCluster || ring < 0 || ring == 1 || ring > ashqk::kMaxRing)
    return ASHQK_ERR_INVALID_ARGUMENT;
  ashqk::g_cluster.store(cluster, std::memory_order_relaxed);
  ashqk::g_ring.store(ring, std::memory_order_relaxed);
  ashqk::fp4_set_pair_split(split);
  return ASHQK_OK;
}
