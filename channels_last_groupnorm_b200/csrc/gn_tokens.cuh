// Building blocks of the kernels on token rows (gn_rms.cu, gn_rotary.cu): vectors of any power-of-two width, sums
// over the lanes or the warps that share a row, parameters of either type, and the number of CTAs that are resident at once.
#pragma once
#include <cuda_fp8.h>

#include <map>
#include <mutex>
#include <tuple>

#include "gn_common.cuh"

namespace gnb200 {

// VE consecutive elements; aligned to their size, or to 16 bytes where they are 32 (8 floats beside 8 halves)
template <typename T, int VE>
__device__ __forceinline__ Pack<T, VE> load_vec(const T* p) {
  Pack<T, VE> v;
  constexpr int kBytes = sizeof(T) * VE;
  if constexpr (kBytes == 32) {
    reinterpret_cast<uint4*>(&v)[0] = reinterpret_cast<const uint4*>(p)[0];
    reinterpret_cast<uint4*>(&v)[1] = reinterpret_cast<const uint4*>(p)[1];
  } else if constexpr (kBytes == 16) {
    *reinterpret_cast<uint4*>(&v) = *reinterpret_cast<const uint4*>(p);
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(&v) = *reinterpret_cast<const uint2*>(p);
  } else {
    static_assert(VE == 1, "vectors of 8, 16 or 32 bytes, or single elements");
    v.v[0] = *p;
  }
  return v;
}
template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, const Pack<T, VE>& v) {
  constexpr int kBytes = sizeof(T) * VE;
  if constexpr (kBytes == 32) {
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<const uint4*>(&v)[0];
    reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<const uint4*>(&v)[1];
  } else if constexpr (kBytes == 16) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&v);
  } else {
    *p = v.v[0];
  }
}

// element i of a parameter vector of type `dtype` (0 fp32, 1 fp16, 2 bf16); `none` where there is no vector
__device__ __forceinline__ float param_at(const void* p, int dtype, long long i, float none) {
  if (p == nullptr) return none;
  if (dtype == 0) return static_cast<const float*>(p)[i];
  if (dtype == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_param_at(void* p, int dtype, long long i, float v) {
  if (dtype == 0)
    static_cast<float*>(p)[i] = v;
  else if (dtype == 1)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// The sum over `lanes` neighbouring lanes (a power of two), the same bits in each: a butterfly adds the same two numbers on both sides.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int delta = lanes >> 1; delta >= 1; delta >>= 1) v += __shfl_xor_sync(0xffffffffu, v, delta);
  return v;
}
// Magnitudes compare like their bit patterns, with NaN above infinity: an integer maximum keeps a NaN, fmaxf would drop it.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  for (int delta = lanes >> 1; delta >= 1; delta >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, delta));
  return v;
}

// Sum over the CTA in a fixed order, one barrier.  `slots`: two rows of 32 floats, used in turn: a thread that writes a row
// again has passed the barrier behind which nobody reads it any more.
__device__ __forceinline__ float cta_sum(float v, float (*slots)[32], int& turn) {
  const int warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  v = lanes_sum(v, 32);
  float* row = slots[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) row[warp] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < nwarps; ++w) t += row[w];
  return t;
}
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* slots) {  // (a barrier of the caller's lies between two calls)
  const int warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) slots[warp] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int w = 0; w < nwarps; ++w) t = max(t, slots[w]);
  return t;
}

// CTAs of `kernel` that the current device holds at once (asked once per kernel, CTA size and device)
inline cudaError_t resident_ctas(const void* kernel, int threads, long long* out) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, int>, long long> known;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(kernel, threads, dev);
  const auto it = known.find(key);
  if (it != known.end()) {
    *out = it->second;
    return cudaSuccess;
  }
  int sms = 0, per_sm = 0;
  err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0);
  if (err != cudaSuccess) return err;
  if (per_sm < 1) return cudaErrorLaunchOutOfResources;
  *out = known[key] = (long long)sms * per_sm;
  return cudaSuccess;
}

// Sums over the rows of up to two sets of C columns, in a fixed order, stored as `dtype` (gn_rms.cu); a programmatic dependent of the
// kernel before it, which writes `part` (`chained`; otherwise in plain stream order)
struct ColumnSums {
  const float* part[2];
  void* out[2];
  int rows[2];
  int C, dtype;
};
cudaError_t launch_column_sums(const ColumnSums& p, int sets, cudaStream_t stream, bool chained);
int report_error(int code, const char* fmt, ...);

}  // namespace gnb200
