// Product of two matrices in four bits (layout: gn_four.cuh): out[token][feature] = alpha * sum over k of x[token][k] w[feature][k] + bias, sums in
// fp32 in tensor memory, alpha the product of the two tensors' own scales, one rounding at the end.
//
// Products of e2m1 codes with their block scales on tcgen05.mma, operands by TMA in K tiles of 256 codes (128 bytes a row, swizzled), block scales by
// copies of their 512-byte tiles to tensor memory, sums in tensor memory.  One thread loads, one multiplies, the others take the sums out.  Two kernels:
//
//   few tokens    the weight is the A operand: a tile has 128 features by all tokens up to 128, and what it costs is the weight's bytes.  Bound by HBM where the
//                 weight is large (8 x 5120 x 20480 14.1 us, 4.2 TB/s; floor 9.1), by the way there and back where it is not (1 x 4096 x 4096 5.5 us, floor 1.4): launch,
//                 one trip to memory, the cluster's meeting.  Where the tiles leave SMs idle, the K tiles are shared out over a cluster, whose sums are added over
//                 distributed shared memory in the order of their ranks; the weight's first K tiles are asked into L2 while the kernel before still runs.
//   many tokens   pairs of CTAs, 256 tokens by 256 or 128 features (below).  8192^3 224 us = 4.9 PFLOP/s in a short run, of 6.1 that the vendor's library reaches; at
//                 length the GPU's 1000 W bound it, 262 us at 1.49 GHz (the library 215).  The products alone would take 136.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "../../include/gnb200.h"
#include "gn_async.cuh"
#include "gn_four.cuh"
#include "gn_kernels.h"
#include "gn_turns.h"

namespace gnb200 {
namespace {

constexpr int kTileK = 256;       // codes of a K tile: the 128 bytes of a swizzled row
constexpr int kTileM = 128;       // features of a tile
constexpr int kThreads = 192;     // four warps for the sums, one to load, one to multiply
constexpr int kMostSplits = 8;    // CTAs of a cluster that share a tile's K
constexpr int kAhead = 8;         // K tiles of the weight that a CTA asks for ahead of its turn

struct LinearArgs {
  const uint8_t *w_scales, *x_scales;
  const float *w_scale, *x_scale;  // of the whole tensors, or NULL
  const void* bias;
  void* out;
  int tokens, features, K, tiles;  // tiles: of scales, along K
  int bias_dtype;
  int stores;  // features and output allow vectors (few tokens: of 4 features; many: of 16 bytes)
  WaitLimit wait;
};

// ---------------------------------------------------------------------------------------------
// Instructions
// ---------------------------------------------------------------------------------------------
// The same box to L2 only.  Before the kernel in front has ended, too: L2 is where that kernel's writes arrive.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void bulk_prefetch(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(smem_addr(bar))
               : "memory");
}
// One lane of a converged warp, in a form that the compiler knows to be one: what it issues takes its operands from uniform registers as they are,
// where behind `lane == 0` every one of these instructions waits for a lane to be picked for its operands.
__device__ __forceinline__ bool one_lane() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// Shared-memory descriptors: start address and stride of 8 rows in 16 bytes, version 1, swizzle (2: 128 bytes; 0: none)
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t stride, uint64_t swizzle) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | 1ull << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | swizzle << 61;
}
// 32 lanes x 16 bytes of shared memory to 4 columns, for all four warps' lanes; of a pair (PAIR), each CTA from its own memory
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// Instruction descriptor: e2m1 times e2m1, fp32 sums, both operands along K; the scales' type (1: e8m0) and the bytes of a word of scales to begin with
__host__ __device__ constexpr uint32_t instruction(int M, int N, bool e8m0, int byte) {
  return 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | (e8m0 ? 1u << 23 : 0u) | (uint32_t)(M >> 4) << 24 | (uint32_t)byte << 29 | (uint32_t)byte << 4;
}
#define GNB200_MMA(group, kind)                                                                                                         \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                                                        \
               "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(acc),                      \
               "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(a_scales), "r"(b_scales)                                                        \
               : "memory")
template <int BLOCK, bool PAIR>
__device__ __forceinline__ void multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, uint32_t add) {
  if constexpr (BLOCK == 16 && PAIR)
    GNB200_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (BLOCK == 16)
    GNB200_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (PAIR)
    GNB200_MMA("2", "mxf4.block_scale.scale_vec::2X");
  else
    GNB200_MMA("1", "mxf4.block_scale.scale_vec::2X");
}
#undef GNB200_MMA
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_load16(uint32_t col, float (&f)[16]) {
  uint4 v[4];
  gnb200::tmem_load16(col, v[0], v[1], v[2], v[3]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[4 * k] = __uint_as_float(v[k].x), f[4 * k + 1] = __uint_as_float(v[k].y);
    f[4 * k + 2] = __uint_as_float(v[k].z), f[4 * k + 3] = __uint_as_float(v[k].w);
  }
}
// 32 words; on their way until tmem_wait
__device__ __forceinline__ void tmem_ask32(uint32_t col, float* f) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]), "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31])
      : "r"(col)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_wait(float (&f)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  pin_regs(f);  // (no use of them moves in front)
}
// 16 bytes of shared memory of a CTA of the cluster, at this CTA's address
__device__ __forceinline__ float4 peer_floats(uint32_t addr, unsigned rank) {
  uint32_t there;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
  return v;
}

// ---------------------------------------------------------------------------------------------
// Few tokens: a tile to a CTA, or to a cluster
// ---------------------------------------------------------------------------------------------
// Shared and tensor memory of a CTA.  The scales of a stage have columns of their own: they are written anew only when the stage is,
// behind the barrier that its products have passed.  Half of either memory at most: two CTAs share an SM.
// NT: 128, or enough for all tokens; a tile of tokens begins with a tile of scales, whose columns of tensor memory the products take from the first one on.
template <int NT, int BLOCK>
struct Layout {
  static constexpr int kChunks = kTileK / (4 * BLOCK);  // tiles of scales to a K tile
  static constexpr int kA = kTileM * 128, kB = NT * 128, kScales = kChunks * kScaleTile;
  static constexpr int kStage = (kA + kB + 2 * kScales + 1023) / 1024 * 1024;
  static constexpr int kColumns = 4 * kChunks;  // of tensor memory, for the scales of one operand
  static constexpr int kAcc = NT < 32 ? 32 : NT;
  static constexpr int kBySmem = (108 << 10) / kStage, kByTmem = (256 - kAcc) / (2 * kColumns);
  static constexpr int kStages = kBySmem < kByTmem ? kBySmem : kByTmem;
  static constexpr int kTmem = kAcc + kStages * 2 * kColumns <= 128 ? 128 : 256;
  static constexpr int kSmem = kStages * kStage + 1024;
  static_assert(kStages >= 2 && NT * kTileM * 4 <= kStages * kStage, "the sums of a split K pass through the stages");
};

template <typename T, int NT, int BLOCK>
__global__ void __launch_bounds__(kThreads, 2) linear4_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                              const LinearArgs p) {
  using L = Layout<NT, BLOCK>;
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t full[L::kStages], empty[L::kStages], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  char* const stages = raw + (-smem_addr(raw) & 1023u);  // (swizzled tiles begin on 1024 bytes)
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const unsigned splits = cluster_nctarank(), rank = cluster_ctarank();
  const int m0 = (int)(blockIdx.x / splits) * kTileM, n0 = (int)blockIdx.y * NT;
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    mbar_init(&done, 1);
    gave_up = 0;
    fence_mbar_init_cluster();
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(L::kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  fence_after();
  // (behind the allocation: what comes next waits for this kernel, so this one must not wait for its tensor memory)
  grid_dep_launch_dependents();
  const uint32_t acc = tmem_slot, scales_at = acc + L::kAcc;
  // this CTA's K tiles
  const int ktiles = (p.K + kTileK - 1) / kTileK;
  const int k_begin = (int)((long long)ktiles * rank / splits), k_count = (int)((long long)ktiles * (rank + 1) / splits) - k_begin;
  const uint8_t* const ws = p.w_scales + (long long)(m0 / 128) * p.tiles * kScaleTile;
  if (warp == 4 && one_lane()) {  // the weight's way from memory is the longest: it begins while the kernel that makes the tokens' codes runs
    for (int k = k_begin; k < k_begin + min(k_count, kAhead); ++k) {
      tma_prefetch_2d(&w_map, k * 128, m0);
      bulk_prefetch(ws + (long long)k * L::kScales, min(L::kChunks, p.tiles - k * L::kChunks) * kScaleTile);
    }
  }
  __syncwarp();
  grid_dep_wait();
  bool whole = true;
  if (warp == 4) {
    if (one_lane()) {
      const uint8_t* xs = p.x_scales + (long long)(n0 / 128) * p.tiles * kScaleTile;
      int issued = 0;
      for (; issued < k_count; ++issued) {
        const int s = issued % L::kStages, k = k_begin + issued;
        if (issued >= L::kStages) {
          producer_wait(&empty[s], (issued / L::kStages - 1) & 1, &gave_up, p.wait);
          if (*(volatile int*)&gave_up) break;
        }
        const uint32_t at = smem_addr(stages) + s * L::kStage;
        const int chunks = min(L::kChunks, p.tiles - k * L::kChunks);
        mbar_arrive_expect_tx(&full[s], L::kA + L::kB + 2 * chunks * kScaleTile);
        tma_load_2d(at, &w_map, k * 128, m0, &full[s]);
        tma_load_2d(at + L::kA, &x_map, k * 128, n0, &full[s]);
        bulk_load(at + L::kA + L::kB, ws + (long long)k * L::kScales, chunks * kScaleTile, &full[s]);
        bulk_load(at + L::kA + L::kB + L::kScales, xs + (long long)k * L::kScales, chunks * kScaleTile, &full[s]);
      }
      // (the copies have landed when the CTA ends, given up or not, unless this wait runs out too)
      for (int k = max(0, issued - L::kStages); k < issued; ++k)
        if (!mbar_wait_bounded(&full[k % L::kStages], (k / L::kStages) & 1, p.wait)) gave_up = 1;
    }
    __syncwarp();
  } else if (warp == 5) {
    if (one_lane()) {
      for (int i = 0; i < k_count; ++i) {
        const int s = i % L::kStages, k = k_begin + i;
        producer_wait(&full[s], (i / L::kStages) & 1, &gave_up, p.wait);
        if (*(volatile int*)&gave_up) break;
        fence_after();
        const uint32_t at = smem_addr(stages) + s * L::kStage;
        const uint32_t ws = scales_at + s * 2 * L::kColumns, xs = ws + L::kColumns;
        const int chunks = min(L::kChunks, p.tiles - k * L::kChunks);
        for (int c = 0; c < chunks; ++c) {
          copy_scales<false>(ws + 4 * c, smem_desc(at + L::kA + L::kB + c * kScaleTile, 128, 0));
          copy_scales<false>(xs + 4 * c, smem_desc(at + L::kA + L::kB + L::kScales + c * kScaleTile, 128, 0));
        }
        const int steps = min(4, (p.K - k * kTileK + 63) / 64);
        for (int j = 0; j < steps; ++j) {  // 64 codes of K, 32 bytes of a row
          const int c = BLOCK == 16 ? j : j / 2, byte = BLOCK == 16 ? 0 : j % 2 * 2;
          multiply<BLOCK, false>(acc, smem_desc(at + j * 32, 1024, 2), smem_desc(at + L::kA + j * 32, 1024, 2), instruction(kTileM, NT, BLOCK == 32, byte), ws + 4 * c,
                          xs + 4 * c, i + j > 0);
        }
        commit(&empty[s]);
      }
      commit(&done);
    }
    __syncwarp();
  } else {
    whole = consumer_wait(&done, 0, &gave_up, p.wait);
  }
  __syncthreads();
  if (*(volatile int*)&gave_up) {  // no product runs any more when memory is used anew and given back, unless this wait runs out too
    if (threadIdx.x == 0) mbar_wait_bounded(&done, 0, p.wait);
    __syncthreads();
    whole = false;
  }
  fence_after();
  if (warp < 4) {
    const int count = min(NT, p.tokens - n0);
    const uint32_t own = acc + ((uint32_t)warp << 21);
    float* const red = reinterpret_cast<float*>(stages);
    for (int j = 0; j < count; j += 16) {
      float f[16];
      tmem_load16(own + j, f);
#pragma unroll
      for (int e = 0; e < 16; ++e) red[(j + e) * kTileM + warp * 32 + lane] = whole ? f[e] : kNaN;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (splits > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      cluster_wait();
    } else {
      asm volatile("barrier.sync 1, 128;" ::: "memory");
    }
    // a token to a warp, 4 features a lane; of the tokens of a tile that several CTAs share, each adds its part
    const int feature = m0 + lane * 4, there = p.features - feature;
    const float alpha = (p.x_scale ? *p.x_scale : 1.f) * (p.w_scale ? *p.w_scale : 1.f);
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = p.bias && e < there ? param_at(p.bias, p.bias_dtype, feature + e, 0.f) : 0.f;
    constexpr int AT_ONCE = 2;  // tokens under way
    for (int first = rank + splits * warp; first < count; first += AT_ONCE * 4 * splits) {
      float4 part[AT_ONCE][kMostSplits];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const uint32_t at = smem_addr(red + min(first + k * 4 * (int)splits, count - 1) * kTileM + lane * 4);
#pragma unroll
        for (unsigned q = 0; q < kMostSplits; ++q) part[k][q] = q < splits ? peer_floats(at, q) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int j = first + k * 4 * (int)splits;
        float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (unsigned q = 0; q < kMostSplits; ++q) t[0] += part[k][q].x, t[1] += part[k][q].y, t[2] += part[k][q].z, t[3] += part[k][q].w;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fmaf(t[e], alpha, bias[e]);
        T* const out = static_cast<T*>(p.out) + (long long)(n0 + j) * p.features + feature;
        if (j < count) {
          if (p.stores && there > 0) {
            *reinterpret_cast<Pack<T, 4>*>(out) = pack<T, 4>(t);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < there) out[e] = store_param<T>(t[e]);
          }
        }
      }
    }
  } else if (splits > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    cluster_wait();
  }
  if (splits > 1) {  // (the others have read what this CTA holds)
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    cluster_wait();
  }
  __syncthreads();
  fence_after();
  __syncwarp();
  if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(acc), "r"(L::kTmem) : "memory");
}

// ---------------------------------------------------------------------------------------------
// Many tokens: pairs of CTAs
// ---------------------------------------------------------------------------------------------
// A pair of SMs multiplies 256 tokens (A, 128 of them an SM) by 256 features (B, half of them in either SM's shared memory), so that an SM brings
// half of what a tile of its own of 128 x 256 would take.  Persistent: the loads run ahead into the next tile, whose products begin as soon as
// eight warps have the sums in registers; these round and store them meanwhile, rows of 256 bytes, through a corner of shared memory of each
// warp's own.  Tensor memory holds one tile's sums (256 columns) and the scales of four stages (192), not two tiles' sums: a tile's 13 us at K = 8192 have some
// 1 us in which the sums are on their way out and nothing is multiplied.
// ns a K tile of 256 (8192^3 in blocks of 16, parts left out to time the others): products 303, with the scales' copies 360, with the loads 420.
constexpr int kPairThreads = 320;  // eight warps for the sums, one to load, one to multiply
constexpr int kPairTokens = 256;   // of a pair's tile
constexpr int kPairStages = 4;

template <int BLOCK, int NF>  // NF: features of a pair's tile, 256 or 128
struct PairLayout {
  static constexpr int kChunks = kTileK / (4 * BLOCK);
  static constexpr int kHigh = NF / 128;  // blocks of 128 features
  static constexpr int kA = 128 * 128, kB = NF / 2 * 128, kScales = kChunks * kScaleTile;  // bytes of the operands' halves, of the scales of 128 rows
  static constexpr int kStage = kA + kB + (1 + kHigh) * kScales, kStageAt = (kStage + 1023) / 1024 * 1024;
  static constexpr int kColumns = (1 + kHigh) * 4 * kChunks;  // of tensor memory, for a stage's scales
  static constexpr int kPitch = 256 + 16;           // bytes of a row on its way out: 16-byte accesses of eight lanes meet different banks
  static constexpr int kOut = 32 * kPitch;          // a warp's
  static constexpr int kSmem = kPairStages * kStageAt + 8 * kOut + 1024;
  static_assert(NF + kPairStages * kColumns <= 512, "tensor memory");
};

struct PairArgs {
  LinearArgs l;
  int token_tiles, feature_tiles;
};

__device__ __forceinline__ uint32_t leaders(const void* mine) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(smem_addr(mine)));
  return there;
}
// into this CTA's shared memory, counted on the leader's barrier
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
// half of a stage's bytes that never come
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// on the barriers of both CTAs, when all products so far are done
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
               "h"((uint16_t)3)
               : "memory");
}
// a word of the peer's shared memory, at the place that it has in this CTA's
__device__ __forceinline__ void tell_peer(const int* mine, int rank, int value) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_addr(mine)), "r"(rank ^ 1));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(value) : "memory");
}
__device__ __forceinline__ void commit_leader(uint64_t* bar) {  // on this CTA's alone
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Tiles in the order of their work: bands of 8 tiles of tokens, along the features, so that the pairs that run at a time share what L2 holds.
template <int NF>
__device__ __forceinline__ void tile_at(const PairArgs& p, int t, int& token, int& feature) {
  constexpr int kBand = 8;
  const int per_band = kBand * p.feature_tiles, band = t / per_band, in = t - band * per_band;
  const int high = min(kBand, p.token_tiles - band * kBand);
  token = (band * kBand + in % high) * kPairTokens;
  feature = in / high * NF;
}

template <typename T, int BLOCK, int NF>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    linear4_pair_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap xs_map,
                        const __grid_constant__ CUtensorMap ws_map, const PairArgs p) {
  using L = PairLayout<BLOCK, NF>;
  extern __shared__ char raw[];
  __shared__ __align__(8) uint64_t full[kPairStages], empty[kPairStages], sums, taken, last;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up, peer_gave_up;
  __shared__ PairEnd end;
  char* const stages = raw + (-smem_addr(raw) & 1023u);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    mbar_init(&sums, 1);
    mbar_init(&taken, 16);  // the warps of both CTAs
    mbar_init(&last, 1);
    gave_up = peer_gave_up = 0;
    fence_mbar_init_cluster();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // the peer's barriers are there
  cluster_wait();
  fence_after();
  grid_dep_launch_dependents();
  const uint32_t acc = tmem_slot, scales_at = acc + NF;
  const int ktiles = (p.l.K + kTileK - 1) / kTileK, tiles = p.token_tiles * p.feature_tiles, pairs = (int)gridDim.x / 2, first = (int)blockIdx.x / 2;
  grid_dep_wait();
  if (warp == 8) {
    if (one_lane()) {
      int n = 0;
      for (int t = first; t < tiles; t += pairs) {
        int token, feature;
        tile_at<NF>(p, t, token, feature);
        for (int k = 0; k < ktiles; ++k, ++n) {
          const int s = n % kPairStages;
          if (n >= kPairStages) {
            producer_wait(&empty[s], (n / kPairStages - 1) & 1, &gave_up, p.l.wait);
            if (*(volatile int*)&gave_up) goto stop;
          }
          const uint32_t at = smem_addr(stages) + s * L::kStageAt, bar = leaders(&full[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::kStage);
          tma_load_pair(at, &x_map, k * 128, token + rank * 128, bar);
          tma_load_pair(at + L::kA, &w_map, k * 128, feature + rank * (NF / 2), bar);
          tma_load_pair(at + L::kA + L::kB, &xs_map, k * (L::kScales / 8), token / 128 + rank, bar);
          tma_load_pair(at + L::kA + L::kB + L::kScales, &ws_map, k * (L::kScales / 8), feature / 128, bar);
        }
      }
      // the products' last arrivals at this CTA's barriers; those before were waited for
      for (int k = drain_begin(n, kPairStages); k < n; ++k) producer_wait(&empty[k % kPairStages], (k / kPairStages) & 1, &gave_up, p.l.wait);
    stop:
      end.loads[rank] = n;
    }
    __syncwarp();
  } else if (warp == 9) {
    if (rank == 0 && one_lane()) {
      int n = 0, turn = 0, told = 0;
      for (int t = first; t < tiles; t += pairs, ++turn) {
        for (int k = 0; k < ktiles; ++k, ++n) {
          const int s = n % kPairStages;
          producer_wait(&full[s], (n / kPairStages) & 1, &gave_up, p.l.wait);
          if (*(volatile int*)&gave_up) goto end;
          fence_after();
          const uint32_t at = smem_addr(stages) + s * L::kStageAt;
          const uint32_t xs = scales_at + s * L::kColumns, ws = xs + 4 * L::kChunks;
          const int steps = min(4, (p.l.K - k * kTileK + 63) / 64);
#pragma unroll
          for (int c = 0; c < L::kChunks; ++c) {
            const uint32_t from = at + L::kA + L::kB + c * kScaleTile;
            copy_scales<true>(xs + 4 * c, smem_desc(from, 128, 0));
#pragma unroll
            for (int h = 0; h < L::kHigh; ++h) copy_scales<true>(ws + 4 * (L::kHigh * c + h), smem_desc(from + (1 + h) * L::kScales, 128, 0));
          }
          if (k == 0 && turn > 0) {  // the sums of the tile before are in registers
            producer_wait(&taken, (turn - 1) & 1, &gave_up, p.l.wait);
            if (*(volatile int*)&gave_up) goto end;
            fence_after();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = BLOCK == 16 ? j : j / 2, byte = BLOCK == 16 ? 0 : j % 2 * 2;
            if (j < steps)
              multiply<BLOCK, true>(acc, smem_desc(at + j * 32, 1024, 2), smem_desc(at + L::kA + j * 32, 1024, 2),
                                    instruction(256, NF, BLOCK == 32, byte), xs + 4 * c, ws + 4 * L::kHigh * c, k + j > 0);
          }
          commit_pair(&empty[s]);
        }
        commit_pair(&sums);
        ++told;
      }
    end:
      end.multiplied = n, end.announced = told;
      // (given up, the sums are not announced: both CTAs' warps give up too and store NaN; no product runs any more when the pair ends)
      commit_leader(&last);
      if (!mbar_wait_bounded(&last, 0, p.l.wait)) gave_up = 1;
    }
    __syncwarp();
  } else {
    constexpr int MINE = NF / 2;  // features of a warp
    const uint32_t own = acc + ((uint32_t)(warp & 3) << 21) + (uint32_t)(warp >> 2) * MINE;
    const uint32_t taken_at = leaders(&taken);
    const float alpha = (p.l.x_scale ? *p.l.x_scale : 1.f) * (p.l.w_scale ? *p.l.w_scale : 1.f);
    char* const corner = stages + kPairStages * L::kStageAt + warp * L::kOut;
    constexpr int VE = 16 / sizeof(T), kCols = MINE < 256 / (int)sizeof(T) ? MINE : 256 / (int)sizeof(T);  // columns of a row on its way out
    int turn = 0;
    Turns turns;
    for (int t = first; t < tiles; t += pairs, ++turn) {
      int token, feature;
      tile_at<NF>(p, t, token, feature);
      token += rank * 128 + (warp & 3) * 32;
      feature += (warp >> 2) * MINE;
      bool whole = false;
      if (!turns.gone) {
        for (int tries = 0; tries < 64 && !whole; ++tries) whole = __all_sync(0xffffffffu, mbar_try_wait(&sums, turn & 1));  // (all lanes: one poll less than by way of lane 0)
        if (!whole) whole = consumer_wait(&sums, turn & 1, &gave_up, p.l.wait);
      }
      whole = turns.take(whole);
      fence_after();
      __syncwarp();
      float f[MINE];
#pragma unroll
      for (int j = 0; j < MINE; j += 32) tmem_ask32(own + j, f + j);
      tmem_wait(f);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      if (lane == 0 && whole) arrive_at(taken_at);
      const float factor = whole ? alpha : kNaN;
      if (p.l.bias) {
#pragma unroll
        for (int j = 0; j < MINE; ++j) f[j] = fmaf(f[j], factor, feature + j < p.l.features ? param_at(p.l.bias, p.l.bias_dtype, feature + j, 0.f) : 0.f);
      } else {
        scale_each(f, factor);
      }
#pragma unroll
      for (int from = 0; from < MINE; from += kCols) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kCols; j += VE)
          *reinterpret_cast<Pack<T, VE>*>(corner + lane * L::kPitch + j * sizeof(T)) = pack<T, VE>(*reinterpret_cast<float(*)[VE]>(f + from + j));
        __syncwarp();
        if (p.l.stores) {
          constexpr int kEach = kCols / VE;  // lanes of a row
          const int column = feature + from + lane % kEach * VE;
#pragma unroll 4
          for (int r = lane / kEach; r < 32; r += 32 / kEach) {
            const uint4 v = *reinterpret_cast<const uint4*>(corner + r * L::kPitch + lane % kEach * 16);
            if (token + r < p.l.tokens && column < p.l.features) *reinterpret_cast<uint4*>(static_cast<T*>(p.l.out) + (long long)(token + r) * p.l.features + column) = v;
          }
        } else {
          // Rows that begin anywhere.  The whole 16-byte vectors of the output in this part of each row are put together from words of the corner, as many
          // lanes a row as above; what is left at either end, less than a vector, is stored one by one, a row a lane (all of it so, or the ends along
          // with the vectors: 5000 x 2048 x 5001 74 us, 5000 features 33).
          constexpr int kEach = kCols / VE;
          const int count = min(kCols, p.l.features - feature - from);
          T* const part = static_cast<T*>(p.l.out) + (long long)token * p.l.features + feature + from;
          const auto head_of = [&](const T* row) { return (int)((0 - reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VE); };
#pragma unroll 4
          for (int r = lane / kEach; r < 32; r += 32 / kEach) {
            T* const row = part + (long long)r * p.l.features;
            const int at = head_of(row) + lane % kEach * VE;
            if (at + VE <= count && token + r < p.l.tokens) {
              const uint32_t* const words = reinterpret_cast<const uint32_t*>(corner + r * L::kPitch) + at * (int)sizeof(T) / 4;
              uint4 v = make_uint4(words[0], words[1], words[2], words[3]);
              if (sizeof(T) == 2 && (at & 1)) {
                const uint32_t next = words[4];
                v = make_uint4(__funnelshift_r(v.x, v.y, 16), __funnelshift_r(v.y, v.z, 16), __funnelshift_r(v.z, v.w, 16), __funnelshift_r(v.w, next, 16));
              }
              *reinterpret_cast<uint4*>(row + at) = v;
            }
          }
          if (token + lane < p.l.tokens) {
            T* const row = part + (long long)lane * p.l.features;
            const T* const held = reinterpret_cast<const T*>(corner + lane * L::kPitch);
            const int head = head_of(row), tail = head + max(0, count - head) / VE * VE;
#pragma unroll
            for (int e = 0; e < VE - 1; ++e) {
              if (e < head && e < count) row[e] = held[e];
              if (tail + e < count) row[tail + e] = held[tail + e];
            }
          }
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  const bool mine = *(volatile int*)&gave_up != 0;
  if (mine && threadIdx.x == 0) tell_peer(&peer_gave_up, rank, 1);
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // neither CTA's memory is used by the other's threads any more ...
  cluster_wait();
  // ... nor by what they started: the products have waited for all copies, the loaders and the others for all of the products' arrivals.  Where a wait gave up, that is
  // done here, unless these waits run out too.
  if (mine || *(volatile int*)&peer_gave_up) {
    if (threadIdx.x == 0) {
      tell_peer(&end.loads[rank], rank, end.loads[rank]);
      if (rank == 0) tell_peer(&end.multiplied, rank, end.multiplied), tell_peer(&end.announced, rank, end.announced);
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    cluster_wait();
    if (threadIdx.x == 0) {
      for (int k = drain_begin(end.multiplied, kPairStages); k < end.multiplied; ++k)
        if (!mbar_wait_bounded(&empty[k % kPairStages], (k / kPairStages) & 1, p.l.wait)) break;
      if (end.announced > 0) mbar_wait_bounded(&sums, (end.announced - 1) & 1, p.l.wait);
      for (int k = drain_begin(end.loads[0], kPairStages); rank == 0 && k < drain_end(end.loads[0], end.loads[1]); ++k) {
        const Missing missing = missing_of(k, end.loads[0], end.loads[1]);
        if (missing == kAnnouncement) mbar_arrive_expect_tx(&full[k % kPairStages], L::kStage);
        if (missing == kPeersBytes) mbar_complete_tx(&full[k % kPairStages], L::kStage);
        if (!mbar_wait_bounded(&full[k % kPairStages], (k / kPairStages) & 1, p.l.wait)) break;
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    cluster_wait();
  }
  fence_after();
  __syncwarp();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(acc), "r"(512) : "memory");
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
cudaError_t encode_fn(EncodeTiledFn* out) {
  static std::mutex mu;
  static EncodeTiledFn fn = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t err = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    if (err != cudaSuccess) return err;
    if (q != cudaDriverEntryPointSuccess || !p) return cudaErrorNotSupported;
    fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  *out = fn;
  return cudaSuccess;
}
// rows of K codes in boxes of `box` rows and 128 bytes, zeros outside
cudaError_t codes_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int box) {
  EncodeTiledFn enc = nullptr;
  const cudaError_t err = encode_fn(&enc);
  if (err != cudaSuccess) return err;
  const cuuint64_t dims[2] = {(cuuint64_t)K / 2, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K / 2};
  const cuuint32_t boxes[2] = {128, (cuuint32_t)box}, steps[2] = {1, 1};
  const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// tiles of scales of rows in blocks of 128, as words of 8 bytes: `tiles` of them and `high` blocks of rows a box, zeros outside
cudaError_t scales_map(CUtensorMap* map, const void* base, int64_t rows, int64_t tiles, int box_tiles, int high) {
  EncodeTiledFn enc = nullptr;
  const cudaError_t err = encode_fn(&enc);
  if (err != cudaSuccess) return err;
  const cuuint64_t dims[2] = {(cuuint64_t)tiles * (kScaleTile / 8), (cuuint64_t)((rows + 127) / 128)}, strides[1] = {(cuuint64_t)tiles * kScaleTile};
  const cuuint32_t boxes[2] = {(cuuint32_t)(box_tiles * (kScaleTile / 8)), (cuuint32_t)high}, steps[2] = {1, 1};
  const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<void*>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int BLOCK, int NF>
cudaError_t launch_pairs(const LinearArgs& l, const void* w_codes, const void* x_codes, cudaStream_t stream) {
  using L = PairLayout<BLOCK, NF>;
  auto kernel = &linear4_pair_kernel<T, BLOCK, NF>;
  CUtensorMap x_map, w_map, xs_map, ws_map;
  cudaError_t err = codes_map(&x_map, x_codes, l.tokens, l.K, 128);
  if (err == cudaSuccess) err = codes_map(&w_map, w_codes, l.features, l.K, NF / 2);
  if (err == cudaSuccess) err = scales_map(&xs_map, l.x_scales, l.tokens, l.tiles, L::kChunks, 1);
  if (err == cudaSuccess) err = scales_map(&ws_map, l.w_scales, l.features, l.tiles, L::kChunks, L::kHigh);
  if (err == cudaSuccess) err = ensure_kernel_attributes((const void*)kernel, L::kSmem, false);
  if (err != cudaSuccess) return err;
  PairArgs p = {};
  p.l = l;
  p.token_tiles = (l.tokens + kPairTokens - 1) / kPairTokens, p.feature_tiles = (l.features + NF - 1) / NF;
  p.l.stores = reinterpret_cast<uintptr_t>(l.out) % 16 == 0 && l.features % (16 / (int)sizeof(T)) == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cfg.gridDim = dim3(2);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int pairs = 0;
  err = resident_clusters((const void*)kernel, &cfg, &pairs);
  if (err != cudaSuccess) return err;
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(pairs, (int64_t)p.token_tiles * p.feature_tiles)));
  cfg.numAttrs = chain_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, x_map, w_map, xs_map, ws_map, p);
}

template <typename T, int NT, int BLOCK>
cudaError_t launch_tiles(const LinearArgs& p, const CUtensorMap& w_map, const CUtensorMap& x_map, int splits, cudaStream_t stream) {
  using L = Layout<NT, BLOCK>;
  auto kernel = &linear4_kernel<T, NT, BLOCK>;
  const cudaError_t err = ensure_kernel_attributes((const void*)kernel, L::kSmem, false);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.features + kTileM - 1) / kTileM * splits), (unsigned)((p.tokens + NT - 1) / NT), 1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = chain_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, w_map, x_map, p);
}

template <typename T, int BLOCK>
cudaError_t launch_linear(LinearArgs p, const void* w_codes, const void* x_codes, cudaStream_t stream) {
  const int64_t ktiles = (p.K + kTileK - 1) / kTileK;
  Residency r = {};
  cudaError_t err = residency((const void*)&linear4_kernel<T, 16, BLOCK>, kThreads, 0, &r);  // (asked for the number of SMs)
  if (err != cudaSuccess) return err;
  // Pairs for more than a tile of tokens, in tiles of 128 features where those are one wave (1024 x 4096 x 2048 11.3 us, 256 features 12.2; 777 x 1344 x 4096, two
  // waves, 10.4 and 8.6); but with fewer tiles than two fifths of the pairs and a K that is worth sharing out, clusters (300 x 4096 x 1111 8.9 us, pairs
  // 12.7; 1024 x 1024 x 1024, four K tiles, 7.6 and 5.6).
  if (p.tokens > 128 && p.features > 128) {
    const int64_t high = (p.tokens + kPairTokens - 1) / kPairTokens, tiles = high * ((p.features + 127) / 128), pairs = r.sms / 2;
    if (tiles > pairs) return launch_pairs<T, BLOCK, 256>(p, w_codes, x_codes, stream);
    if (ktiles <= 4 || 5 * tiles >= 2 * pairs) return launch_pairs<T, BLOCK, 128>(p, w_codes, x_codes, stream);
  }
  p.stores = p.features % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % (4 * sizeof(T)) == 0;
  const int NT = p.tokens <= 16 ? 16 : p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : 128;
  CUtensorMap w_map, x_map;
  err = codes_map(&w_map, w_codes, p.features, p.K, kTileM);
  if (err == cudaSuccess) err = codes_map(&x_map, x_codes, p.tokens, p.K, NT);
  if (err != cudaSuccess) return err;
  const int64_t tiles = (int64_t)((p.features + kTileM - 1) / kTileM) * ((p.tokens + NT - 1) / NT);
  // K is shared out by two and by four while all CTAs are resident, two an SM (32 x 8192 x 8192 in clusters of 1, 2, 4, 8: 19.4, 14.4, 13.2, 19.5 us; 16 x 4096 x 16384
  // 13.4, 12.5, 16.5, 25.2), by eight while there is one for two thirds of them (32 x 4096 x 4096 10.7, 7.7, 6.4, 8.0; 4 x 5120 x 1280 11.1, 7.7, 5.5, 4.9).
  int splits = 1;
  while (splits < kMostSplits && splits * 2 <= ktiles && tiles * splits * 2 <= (splits < 4 ? 2 * r.sms : 4 * r.sms / 3)) splits *= 2;
  if (NT == 16) return launch_tiles<T, 16, BLOCK>(p, w_map, x_map, splits, stream);
  if (NT == 32) return launch_tiles<T, 32, BLOCK>(p, w_map, x_map, splits, stream);
  if (NT == 64) return launch_tiles<T, 64, BLOCK>(p, w_map, x_map, splits, stream);
  return launch_tiles<T, 128, BLOCK>(p, w_map, x_map, splits, stream);
}

}  // namespace
}  // namespace gnb200

using namespace gnb200;

extern "C" {

int gnb200_linear_4bit(const void* x_codes, const void* x_scales, const float* x_scale, const void* w_codes, const void* w_scales, const float* w_scale,
                       const void* bias, int64_t tokens, int64_t features, int64_t channels, int block, int bias_dtype, int dtype, void* out, void* stream) {
  const char* name = "gnb200_linear_4bit";
  if (dtype < GNB200_F32 || dtype > GNB200_BF16 || bias_dtype < GNB200_F32 || bias_dtype > GNB200_BF16)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if (block != 16 && block != 32) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: block is 16 or 32 channels (got %d)", name, block);
  if (block == 32 && (x_scale || w_scale))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: blocks of 32 have no scale of the whole tensor", name);
  if (tokens < 0 || features < 0 || channels < 1)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: tokens and features must not be negative and channels be positive (got %lld, %lld, %lld)", name,
                        (long long)tokens, (long long)features, (long long)channels);
  if (tokens == 0 || features == 0) return GNB200_OK;
  // (tiles of tokens are the grid's second axis)
  if (channels > (1 << 30) || features > (1 << 30) || tokens > (int64_t)65535 * 128)
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: more than 2^30 channels or features or 8388480 tokens are not supported (got %lld, %lld, %lld)", name,
                        (long long)channels, (long long)features, (long long)tokens);
  if (!x_codes || !x_scales || !w_codes || !w_scales || !out) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  for (const void* q : {x_codes, x_scales, w_codes, w_scales})
    if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  if (wait_gave_up_on_current_device())
    return report_error(GNB200_ERR_EXCHANGE_TIMEOUT,
                        "%s: a kernel of an earlier call on this device gave up waiting; gnb200_clear_wait_timeouts() re-arms the library", name);
  LinearArgs p = {};
  p.w_scales = static_cast<const uint8_t*>(w_scales), p.x_scales = static_cast<const uint8_t*>(x_scales);
  p.w_scale = w_scale, p.x_scale = x_scale, p.bias = bias, p.out = out, p.bias_dtype = bias_dtype;
  p.tokens = (int)tokens, p.features = (int)features, p.K = (int)four_wide(channels), p.tiles = (int)four_tiles(channels, block);
  cudaError_t err = wait_limit_for_device(&p.wait);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (err == cudaSuccess) {
    const auto typed = [&](auto t) {
      using T = decltype(t);
      return block == 16 ? launch_linear<T, 16>(p, w_codes, x_codes, s) : launch_linear<T, 32>(p, w_codes, x_codes, s);
    };
    err = dtype == GNB200_F32 ? typed(float()) : dtype == GNB200_F16 ? typed(__half()) : typed(__nv_bfloat16());
  }
  if (err != cudaSuccess) return report_error(GNB200_ERR_CUDA, "%s: CUDA error: %s", name, cudaGetErrorString(err));
  return GNB200_OK;
}

}  // extern "C"
