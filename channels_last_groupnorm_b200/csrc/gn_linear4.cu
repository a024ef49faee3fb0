// Product of two matrices in four bits (layout: gn_four.cuh): out[token][feature] = alpha * sum over k of x[token][k] w[feature][k] + bias, sums in
// fp32 in tensor memory, alpha the product of the two tensors' own scales, one rounding at the end.
//
// tcgen05.mma with block scales: the weight is the A operand, so that a tile has 128 features by any number of tokens, and few tokens cost
// little.  A producer thread brings K tiles of 256 codes (128 bytes a row, swizzled) by TMA and their scales by bulk copies; one thread
// copies the scales of a stage to tensor memory and multiplies; four warps take the sums out, a feature a lane, so that a warp's stores
// lie side by side at any width of the output.
// Where a grid of tiles leaves SMs idle the K tiles are shared out over a cluster, whose sums are added over distributed shared memory in
// the order of their ranks.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "../../include/gnb200.h"
#include "gn_async.cuh"
#include "gn_four.cuh"
#include "gn_kernels.h"

namespace gnb200 {
namespace {

constexpr int kTileK = 256;       // codes of a K tile: the 128 bytes of a swizzled row
constexpr int kTileM = 128;       // features of a tile
constexpr int kThreads = 192;     // four warps for the sums, one to load, one to multiply
constexpr int kMostSplits = 8;    // CTAs of a cluster that share a tile's K

struct LinearArgs {
  const uint8_t *w_scales, *x_scales;
  const float *w_scale, *x_scale;  // of the whole tensors, or NULL
  const void* bias;
  void* out;
  int tokens, features, K, tiles;  // tiles: of scales, along K
  int bias_dtype;
  WaitLimit wait;
};

// ---------------------------------------------------------------------------------------------
// Instructions
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(smem_addr(bar))
               : "memory");
}
// Shared-memory descriptors: start address and stride of 8 rows in 16 bytes, version 1, swizzle (2: 128 bytes; 0: none)
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t stride, uint64_t swizzle) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | 1ull << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | swizzle << 61;
}
// 32 lanes x 16 bytes of shared memory to 4 columns, for all four warps' lanes
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// Instruction descriptor: e2m1 times e2m1, fp32 sums, both operands along K; the scales' type (1: e8m0) and the bytes of a word of scales to begin with
__host__ __device__ constexpr uint32_t instruction(int M, int N, bool e8m0, int byte) {
  return 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | (e8m0 ? 1u << 23 : 0u) | (uint32_t)(M >> 4) << 24 | (uint32_t)byte << 29 | (uint32_t)byte << 4;
}
template <int BLOCK>
__device__ __forceinline__ void multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, uint32_t add) {
  if constexpr (BLOCK == 16)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(acc),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(a_scales), "r"(b_scales)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(acc),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(a_scales), "r"(b_scales)
        : "memory");
}
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
__device__ __forceinline__ float peer_float(uint32_t addr, unsigned rank) {
  uint32_t there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

// ---------------------------------------------------------------------------------------------
// Kernel
// ---------------------------------------------------------------------------------------------
// Shared and tensor memory of a CTA.  The scales of a stage have columns of their own: they are written anew only when the stage is,
// behind the barrier that its products have passed.  Half of either memory at most: two CTAs share an SM.
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  grid_dep_wait();
  bool whole = true;
  if (warp == 4) {
    if (lane == 0) {
      const uint8_t* ws = p.w_scales + (long long)(m0 / 128) * p.tiles * kScaleTile;
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
      // (nothing is in flight when the CTA ends, given up or not)
      for (int k = max(0, issued - L::kStages); k < issued; ++k)
        if (!mbar_wait_bounded(&full[k % L::kStages], (k / L::kStages) & 1, p.wait)) gave_up = 1;
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0) {
      for (int i = 0; i < k_count; ++i) {
        const int s = i % L::kStages, k = k_begin + i;
        producer_wait(&full[s], (i / L::kStages) & 1, &gave_up, p.wait);
        if (*(volatile int*)&gave_up) break;
        fence_after();
        const uint32_t at = smem_addr(stages) + s * L::kStage;
        const uint32_t ws = scales_at + s * 2 * L::kColumns, xs = ws + L::kColumns;
        const int chunks = min(L::kChunks, p.tiles - k * L::kChunks);
        for (int c = 0; c < chunks; ++c) {
          copy_scales(ws + 4 * c, smem_desc(at + L::kA + L::kB + c * kScaleTile, 128, 0));
          copy_scales(xs + 4 * c, smem_desc(at + L::kA + L::kB + L::kScales + c * kScaleTile, 128, 0));
        }
        const uint32_t xs_tile = xs + (n0 % 128) / 32;
        const int steps = min(4, (p.K - k * kTileK + 63) / 64);
        for (int j = 0; j < steps; ++j) {  // 64 codes of K, 32 bytes of a row
          const int c = BLOCK == 16 ? j : j / 2, byte = BLOCK == 16 ? 0 : j % 2 * 2;
          multiply<BLOCK>(acc, smem_desc(at + j * 32, 1024, 2), smem_desc(at + L::kA + j * 32, 1024, 2), instruction(kTileM, NT, BLOCK == 32, byte), ws + 4 * c,
                          xs_tile + 4 * c, i + j > 0);
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
  fence_after();
  whole = whole && *(volatile int*)&gave_up == 0;
  if (warp < 4) {
    const int feature = m0 + warp * 32 + lane, count = min(NT, p.tokens - n0);
    const bool inside = feature < p.features;
    const float alpha = (p.x_scale ? *p.x_scale : 1.f) * (p.w_scale ? *p.w_scale : 1.f);
    const float bias = p.bias && inside ? param_at(p.bias, p.bias_dtype, feature, 0.f) : 0.f;
    T* const out = static_cast<T*>(p.out) + (long long)n0 * p.features + feature;
    const uint32_t own = acc + ((uint32_t)warp << 21);
    float* const red = reinterpret_cast<float*>(stages) + warp * 32 + lane;
    for (int j = 0; j < count; j += 16) {
      float f[16];
      tmem_load16(own + j, f);
      if (splits == 1) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (inside && j + e < count) out[(long long)(j + e) * p.features] = store_param<T>(whole ? fmaf(f[e], alpha, bias) : kNaN);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) red[(j + e) * kTileM] = whole ? f[e] : kNaN;
      }
    }
    if (splits > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      cluster_wait();
      for (int j = rank; j < count; j += splits) {
        float t = 0.f;
        for (unsigned q = 0; q < splits; ++q) t += peer_float(smem_addr(red + j * kTileM), q);
        if (inside) out[(long long)j * p.features] = store_param<T>(fmaf(t, alpha, bias));
      }
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      cluster_wait();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  } else if (splits > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    cluster_wait();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    cluster_wait();
  }
  __syncthreads();
  fence_after();
  __syncwarp();
  if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(acc), "r"(L::kTmem) : "memory");
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
cudaError_t launch_linear(const LinearArgs& p, const void* w_codes, const void* x_codes, cudaStream_t stream) {
  const int NT = p.tokens <= 16 ? 16 : p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : 128;
  CUtensorMap w_map, x_map;
  cudaError_t err = codes_map(&w_map, w_codes, p.features, p.K, kTileM);
  if (err == cudaSuccess) err = codes_map(&x_map, x_codes, p.tokens, p.K, NT);
  if (err != cudaSuccess) return err;
  const int64_t tiles = (int64_t)((p.features + kTileM - 1) / kTileM) * ((p.tokens + NT - 1) / NT), ktiles = (p.K + kTileK - 1) / kTileK;
  int splits = 1;
  while (splits < kMostSplits && splits * 2 <= ktiles && tiles * splits * 2 <= 296) splits *= 2;
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
