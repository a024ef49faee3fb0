// Building blocks of the kernels on token rows (gn_rms.cu, gn_rotary.cu): vectors of any power-of-two width, sums
// over the lanes or the warps that share a row, parameters of either type, and the CTAs that an SM holds at once.
#pragma once
#include <cuda_fp8.h>

#include <array>

#include "gn_common.cuh"

namespace gnb200 {

constexpr int kMostDynamicSmem = 220 << 10;  // of an SM's 227 KB: the kernels have a few KB of static shared memory beside it

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

// VE parameters starting at element i, on the vector path from aligned addresses
template <int VE>
__device__ __forceinline__ void params_at(const void* p, int dtype, long long i, float (&f)[VE]) {
  if constexpr (VE == 1) {
    f[0] = param_at(p, dtype, i, 1.f);
  } else if (dtype == 0) {
    unpack<float, VE>(load_vec<float, VE>(static_cast<const float*>(p) + i), f);
  } else if (dtype == 1) {
    unpack<__half, VE>(load_vec<__half, VE>(static_cast<const __half*>(p) + i), f);
  } else {
    unpack<__nv_bfloat16, VE>(load_vec<__nv_bfloat16, VE>(static_cast<const __nv_bfloat16*>(p) + i), f);
  }
}

// Lane by lane over a vector, two lanes an instruction where there are pairs (the same bits as one by one): a += b, a *= b, a *= s,
// a += b * c (vectors), a += b * c (c a number).
template <int N>
__device__ __forceinline__ void add_each(float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) add2(a[e], a[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] += b[e];
  }
}
template <int N>
__device__ __forceinline__ void mul_each(float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) mul2(a[e], a[e + 1], a[e], a[e + 1], b[e], b[e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] *= b[e];
  }
}
template <int N>
__device__ __forceinline__ void scale_each(float (&a)[N], float s) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) mul2(a[e], a[e + 1], a[e], a[e + 1], s, s);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] *= s;
  }
}
template <int N>
__device__ __forceinline__ void fma_each(float (&a)[N], const float (&b)[N], const float (&c)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) fma2(a[e], a[e + 1], b[e], b[e + 1], c[e], c[e + 1], a[e], a[e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] = fmaf(b[e], c[e], a[e]);
  }
}
template <int N>
__device__ __forceinline__ void axpy_each(float (&a)[N], const float (&b)[N], float c) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) fma2(a[e], a[e + 1], b[e], b[e + 1], c, c, a[e], a[e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] = fmaf(b[e], c, a[e]);
  }
}
// acc += sum of a * b, over even and odd lanes apart
template <int N>
__device__ __forceinline__ void dot_each(float (&acc)[2], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) fma2(acc[0], acc[1], a[e], a[e + 1], b[e], b[e + 1], acc[0], acc[1]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e & 1] = fmaf(a[e], b[e], acc[e & 1]);
  }
}

// The sum over `lanes` neighbouring lanes (a power of two), the same bits in each: a butterfly adds the same two numbers on both sides.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
#pragma unroll
  for (int delta = 16; delta >= 1; delta >>= 1)
    if (lanes > delta) v += __shfl_xor_sync(0xffffffffu, v, delta);
  return v;
}
// (Maxima by shuffles as well: they serve groups of a few lanes, which a reduction over the warp does not.)
// Magnitudes compare like their bit patterns, with NaN above infinity: an integer maximum keeps a NaN, fmaxf would drop it.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// the larger of two magnitudes, or NaN where one is
__device__ __forceinline__ float larger(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
#pragma unroll
  for (int delta = 16; delta >= 1; delta >>= 1)
    if (lanes > delta) v = max(v, __shfl_xor_sync(0xffffffffu, v, delta));
  return v;
}

// Teams of whole warps: a barrier of their own (hardware barriers 1 to 15), and the sum over a team in a fixed order behind one of
// them.  The slots are two rows used in turn: a thread that writes a row again has passed the barrier behind which nobody reads it any
// more.  The places of warps that are not there hold zeros.
constexpr int kMostWarps = 32, kMostTeams = 15;
struct TeamSlots {
  alignas(16) float row[2][kMostWarps];
};
template <bool TEAMS>  // false: the team is the CTA
__device__ __forceinline__ void team_barrier(int threads, int team) {
  if constexpr (TEAMS) {
    __syncwarp();
    asm volatile("barrier.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
  } else {
    __syncthreads();
  }
}
template <bool TEAMS>
__device__ __forceinline__ void clear(TeamSlots& slots, int threads, int team, int first) {
  for (int i = first; i < 2 * kMostWarps; i += threads) slots.row[i / kMostWarps][i % kMostWarps] = 0.f;
  team_barrier<TEAMS>(threads, team);
}
template <bool TEAMS>
__device__ __forceinline__ float team_sum(float v, TeamSlots& slots, int& turn, int threads, int team) {
  v = lanes_sum(v, 32);
  float* row = slots.row[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) row[(threadIdx.x - (TEAMS ? team * threads : 0)) >> 5] = v;
  team_barrier<TEAMS>(threads, team);
  const float4* four = reinterpret_cast<const float4*>(row);
  float4 t = four[0];
  if (threads > 128) {
    const float4 u = four[1];
    t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
  }
  if (threads > 256) {
    const float4 u = four[2], w = four[3];
    t.x += u.x + w.x, t.y += u.y + w.y, t.z += u.z + w.z, t.w += u.w + w.w;
  }
  if (threads > 512) {
    float4 s = four[4];
#pragma unroll
    for (int k = 5; k < kMostWarps / 4; ++k) s.x += four[k].x, s.y += four[k].y, s.z += four[k].z, s.w += four[k].w;
    t.x += s.x, t.y += s.y, t.z += s.z, t.w += s.w;
  }
  return (t.x + t.y) + (t.z + t.w);
}
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* slots) {  // (a barrier of the caller's lies between two calls)
  const int warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  v = lanes_max(v, 32);
  if ((threadIdx.x & 31) == 0) slots[warp] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int w = 0; w < nwarps; ++w) t = max(t, slots[w]);
  return t;
}

// CTAs of `kernel` that one SM holds at once with `smem` bytes of dynamic shared memory, and the SMs of the current device (the question
// also raises the kernel's limit of shared memory)
struct Residency {
  int per_sm, sms;
};
inline cudaError_t ask_residency(const void* kernel, int threads, int smem, Residency* out) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  Residency r = {};
  err = cudaDeviceGetAttribute(&r.sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  if (smem > 0) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostDynamicSmem);
    if (err != cudaSuccess) return err;
  }
  err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&r.per_sm, kernel, threads, smem);
  if (err != cudaSuccess) return err;
  if (r.per_sm < 1) return cudaErrorLaunchOutOfResources;
  *out = r;
  return cudaSuccess;
}
inline cudaError_t residency(const void* kernel, int threads, int smem, Residency* out) {
  // a thread's last answers, one per place of a small table
  struct Known {
    const void* kernel;
    int threads, smem, dev;
    Residency r;
  };
  constexpr int kPlaces = 64;
  static thread_local Known known[kPlaces] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const size_t mix = (reinterpret_cast<uintptr_t>(kernel) >> 4) * 31 + (size_t)threads * 7 + (size_t)(smem >> 4) * 13 + (size_t)dev;
  Known& k = known[mix % kPlaces];
  if (k.kernel != kernel || k.threads != threads || k.smem != smem || k.dev != dev) {
    Residency r;
    err = ask_residency(kernel, threads, smem, &r);
    if (err != cudaSuccess) return err;
    k = Known{kernel, threads, smem, dev, r};
  }
  *out = k.r;
  return cudaSuccess;
}

// The last answers to a question that a program asks again and again with the same few arguments
template <int N>
struct Remembered {
  using Key = std::array<int64_t, N>;
  const size_t* find(const Key& key) const {
    for (int i = 0; i < used; ++i)
      if (keys[i] == key) return &values[i];
    return nullptr;
  }
  size_t keep(const Key& key, size_t value) {
    keys[next] = key;
    values[next] = value;
    if (used < kPlaces) ++used;
    next = (next + 1) % kPlaces;
    return value;
  }
  static constexpr int kPlaces = 16;
  std::array<Key, kPlaces> keys;
  size_t values[kPlaces];
  int used = 0, next = 0;
};

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
