// Rows to four bits and back, and the root-mean-square norm with the residual's addition straight into four bits (formulas and layout:
// gn_four.cuh; the norm is that of gn_rms.cu: s = x + r in fp32, y = s * rsqrt(mean(s^2) + eps) * (offset + w), y not rounded before its codes).
//
// A lane holds 8 channels, neighbouring lanes a block: its largest magnitude by shuffles, one scale, 4 bytes of codes a lane; the scales of
// four blocks become one word.
#include <algorithm>

#include "../../include/gnb200.h"
#include "gn_four.cuh"
#include "gn_kernels.h"

namespace gnb200 {
namespace {

constexpr int VE = 8;  // channels of a lane

struct FourRows {
  uint8_t *codes, *scales;
  const float* tensor_scale;  // g, or NULL for one
  long long rows;
  int C, wide, tiles;
};

// ---------------------------------------------------------------------------------------------
// Codes and scales
// ---------------------------------------------------------------------------------------------
// A code is that of the fp32 quotient y / d, as a division rounds it: with 16-bit inputs y / d lies midway between two codes often enough that
// a quotient one unit off shows.  The reciprocal is the correctly rounded one (a Newton step from the hardware's), the quotient is corrected by
// its remainder (Markstein's theorem).
struct Step {
  float value, inverse;
  uint32_t byte;
};
template <int BLOCK>
__device__ __forceinline__ Step step_of(uint32_t most, float g, float six_g) {
  Step step;
  const bool finite = most < 0x7f800000u;
  if constexpr (BLOCK == 16) {
    const float s = fmaxf(__fdiv_rn(__uint_as_float(most), six_g), 0.001953125f);
    step.byte = finite ? __nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3) : 0x7fu;
    step.value = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)step.byte, __NV_E4M3))) * g;
    float near;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(near) : "f"(step.value));
    step.inverse = fmaf(fmaf(-step.value, near, 1.f), near, near);
  } else {
    const int e = max((int)(most >> 23) - 2, 0);
    step.byte = finite ? (uint32_t)e : 0xffu;
    step.value = 0.f;  // (a product with the inverse, a power of two, is the quotient)
    step.inverse = __uint_as_float((uint32_t)(254 - min(e, 252)) << 23);
  }
  return step;
}
template <int BLOCK>
__device__ __forceinline__ uint32_t codes_of(const float (&y)[VE], const Step& step) {
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < VE; e += 2) {
    float q0, q1;
    mul2(q0, q1, y[e], y[e + 1], step.inverse, step.inverse);
    if constexpr (BLOCK == 16) {
      float r0, r1;
      fma2(r0, r1, q0, q1, step.value, step.value, -y[e], -y[e + 1]);
      fma2(q0, q1, r0, r1, -step.inverse, -step.inverse, q0, q1);
    }
    word |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(q0, q1), __NV_E2M1, cudaRoundNearest) << (4 * e);
  }
  return word;
}
// Codes of the 8 channels y of vector v of a row (zeros where it has none) and the scales that its lanes share; by whole warps.
template <int BLOCK>
__device__ __forceinline__ void put(const FourRows& p, long long row, int v, bool live, const float (&y)[VE], float g, float six_g) {
  constexpr int LANES = BLOCK / VE;
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < VE; ++e) most = larger(most, fabsf(y[e]));
  const Step step = step_of<BLOCK>(lanes_max(magnitude(most), LANES), g, six_g);
  const uint32_t word = codes_of<BLOCK>(y, step);
  const bool inside = v * VE < p.wide;
  if (live && inside) *reinterpret_cast<uint32_t*>(p.codes + (row * (p.wide / VE) + v) * 4) = word;
  const int block = v / LANES;
  uint32_t scales = inside ? step.byte << (8 * (block & 3)) : 0;
  scales |= __shfl_xor_sync(0xffffffffu, scales, LANES);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2 * LANES);
  if (live && v % (4 * LANES) == 0) *reinterpret_cast<uint32_t*>(p.scales + four_scale_at(row, block >> 2, p.tiles)) = scales;
}
// The scales of rows that fill up the last tile, by all threads of the grid.
__device__ __forceinline__ void clear_behind(const FourRows& p, long long thread, long long threads) {
  const int behind = (int)(-p.rows & 127);
  for (long long i = thread; i < (long long)behind * p.tiles; i += threads)
    *reinterpret_cast<uint32_t*>(p.scales + four_scale_at(p.rows + i % behind, i / behind, p.tiles)) = 0;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int v, int C, float (&f)[VE]) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(row)[2 * v], b = reinterpret_cast<const float4*>(row)[2 * v + 1];
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
      unpack<T, VE>(load_vec<T, VE>(row + v * VE), f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = v * VE + e < C ? load_param<T>(row, v * VE + e) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int v, int C, const float (&f)[VE]) {
  if constexpr (VEC) {
    store_vec<T, VE>(row + v * VE, pack<T, VE>(f));
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (v * VE + e < C) row[v * VE + e] = store_param<T>(f[e]);
  }
}
__device__ __forceinline__ void zero(float (&f)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = 0.f;
}

// ---------------------------------------------------------------------------------------------
// Rows to four bits and back
// ---------------------------------------------------------------------------------------------
constexpr int kThreads = 256;

// `lanes` (a power of two) threads share a row's piece; the grid's second axis shares a row out.
template <typename T, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* x, long long x_stride, const FourRows p, int lanes) {
  grid_dep_launch_dependents();
  const int per_cta = kThreads / lanes, lane = threadIdx.x % lanes, vectors = p.tiles * 4 * (BLOCK / VE), step = gridDim.y * lanes;
  const float g = BLOCK == 16 && p.tensor_scale ? *p.tensor_scale : 1.f, six_g = 6.f * g;
  for (long long base = (long long)blockIdx.x * per_cta; base < p.rows; base += (long long)gridDim.x * per_cta) {
    const long long row = base + threadIdx.x / lanes;
    const bool live = row < p.rows;
    const T* from = x + row * x_stride;
    for (int first = blockIdx.y * lanes; first < vectors; first += 2 * step) {
      float y[2][VE];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        zero(y[k]);
        const int v = first + k * step + lane;
        if (live && v * VE < p.C) load8<T, VEC>(from, v, p.C, y[k]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int v = first + k * step + lane;
        put<BLOCK>(p, row, v, live && v < vectors, y[k], g, six_g);
      }
    }
  }
  clear_behind(p, ((long long)blockIdx.y * gridDim.x + blockIdx.x) * kThreads + threadIdx.x, (long long)gridDim.x * gridDim.y * kThreads);
}

__device__ __forceinline__ float scale_value(uint32_t byte, int block) {
  if (block == 16) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
  return byte == 0xff ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);  // (2^-127 is subnormal)
}
template <typename T, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const FourRows p, T* out, int lanes) {
  const int per_cta = kThreads / lanes, lane = threadIdx.x % lanes, step = gridDim.y * lanes;
  const float g = BLOCK == 16 && p.tensor_scale ? *p.tensor_scale : 1.f;
  for (long long row = (long long)blockIdx.x * per_cta + threadIdx.x / lanes; row < p.rows; row += (long long)gridDim.x * per_cta) {
    for (int v = blockIdx.y * lanes + lane; v * VE < p.C; v += step) {
      const uint32_t word = *reinterpret_cast<const uint32_t*>(p.codes + (row * (p.wide / VE) + v) * 4);
      const int block = v / (BLOCK / VE);
      const float scale = scale_value(p.scales[four_scale_at(row, block >> 2, p.tiles) + (block & 3)], BLOCK);
      float f[VE];
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const float2 two = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(word >> (4 * e)), __NV_E2M1)));
        f[e] = two.x * scale * g;
        f[e + 1] = two.y * scale * g;
      }
      store8<T, VEC>(out + row * p.C, v, p.C, f);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Norm
// ---------------------------------------------------------------------------------------------
struct NormArgs {
  const void *x, *residual, *weight;
  void* sum;
  long long x_stride, r_stride;
  int w_dtype;
  float eps, offset, inv_c;
};

// (offset + w) of 8 channels, from addresses on 16 bytes (VEC) or any
template <bool VEC>
__device__ __forceinline__ void weight8(const NormArgs& a, int v, int C, float (&w)[VE]) {
  if constexpr (VEC) {
    if (a.w_dtype == 0) {
      load8<float, true>(static_cast<const float*>(a.weight), v, C, w);
    } else {
      params_at<VE>(a.weight, a.w_dtype, (long long)v * VE, w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = v * VE + e < C ? param_at(a.weight, a.w_dtype, v * VE + e, 1.f) : 0.f;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) w[e] += a.offset;
}

// A row to a warp (WARP) or a CTA, V vectors a thread in registers; V = 0: rows of any length, read twice.
template <typename Tx, typename Ts, int BLOCK, int V, bool WARP, bool VEC>
__global__ void __launch_bounds__(WARP ? 128 : 1024) norm_kernel(const NormArgs a, const FourRows p) {
  constexpr int HELD = V > 0 ? V : 1;
  __shared__ TeamSlots slots;
  grid_dep_launch_dependents();
  const int threads = WARP ? 32 : (int)blockDim.x, at = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const long long row = WARP ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const bool live = row < p.rows;
  const int vectors = p.tiles * 4 * (BLOCK / VE);
  const float g = BLOCK == 16 && p.tensor_scale ? *p.tensor_scale : 1.f, six_g = 6.f * g;
  const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_stride;
  const Ts* r = a.residual ? static_cast<const Ts*>(a.residual) + row * a.r_stride : nullptr;
  if constexpr (!WARP) clear<false>(slots, threads, 0, at);
  auto sum_of = [&](int v, float (&s)[VE]) {
    zero(s);
    if (live && v * VE < p.C) {
      load8<Tx, VEC>(x, v, p.C, s);
      if (r) {
        float f[VE];
        load8<Ts, VEC>(r, v, p.C, f);
        add_each(s, f);
      }
    }
  };
  float s[HELD][VE], sq[2] = {0.f, 0.f};
  if constexpr (V > 0) {
#pragma unroll
    for (int k = 0; k < V; ++k) sum_of(at + k * threads, s[k]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int v = at + k * threads;
      if (r && live && v * VE < p.C) store8<Ts, VEC>(static_cast<Ts*>(a.sum) + row * p.C, v, p.C, s[k]);
      dot_each(sq, s[k], s[k]);
    }
  } else {
    for (int v = at; v * VE < p.C; v += threads) {
      sum_of(v, s[0]);
      dot_each(sq, s[0], s[0]);
    }
  }
  int turn = 0;
  const float all = WARP ? lanes_sum(sq[0] + sq[1], 32) : team_sum<false>(sq[0] + sq[1], slots, turn, threads, 0);
  const float rstd = __frsqrt_rn(fmaf(all, a.inv_c, a.eps));
  auto finish = [&](int v, float (&y)[VE]) {
    if (v * VE < p.C) {
      scale_each(y, rstd);
      if (a.weight) {
        float w[VE];
        weight8<VEC>(a, v, p.C, w);
        mul_each(y, w);
      }
    }
    if constexpr (!VEC) {  // (behind the row a NaN rstd would leave NaN in the zeros)
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (v * VE + e >= p.C) y[e] = 0.f;
    }
    put<BLOCK>(p, row, v, live && v < vectors, y, g, six_g);
  };
  if constexpr (V > 0) {
#pragma unroll
    for (int k = 0; k < V; ++k) finish(at + k * threads, s[k]);
  } else {
    for (int first = 0; first < vectors; first += threads) {
      sum_of(first + at, s[0]);  // (the last look at these: the sum may be the residual's own buffer)
      if (r && (first + at) * VE < p.C) store8<Ts, VEC>(static_cast<Ts*>(a.sum) + row * p.C, first + at, p.C, s[0]);
      finish(first + at, s[0]);
    }
  }
  clear_behind(p, (long long)blockIdx.x * blockDim.x + threadIdx.x, (long long)gridDim.x * blockDim.x);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
template <typename F>
cudaError_t with_type(int dtype, F&& f) {
  if (dtype == GNB200_F32) return f(float());
  if (dtype == GNB200_F16) return f(__half());
  return f(__nv_bfloat16());
}
template <typename F>
cudaError_t with_flag(bool flag, F&& f) {
  return flag ? f(std::true_type()) : f(std::false_type());
}
template <typename F>
cudaError_t with_block(int block, F&& f) {
  return block == 16 ? f(std::integral_constant<int, 16>()) : f(std::integral_constant<int, 32>());
}
bool dtype_ok(int d) { return d == GNB200_F32 || d == GNB200_F16 || d == GNB200_BF16; }
int size_of(int dtype) { return dtype == GNB200_F32 ? 4 : 2; }
bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct Shares {
  int lanes;
  dim3 grid;
};
// Lanes of a row's piece: a row's vectors where they are few, a warp's where there are rows enough to fill the GPU with warps, otherwise the
// CTA; the rest of a row goes round, or to other CTAs while there are SMs without one.
cudaError_t share_out(int64_t rows, int64_t vectors, int least, const void* kernel, Shares* out) {
  Residency r = {};
  const cudaError_t err = residency(kernel, kThreads, 0, &r);
  if (err != cudaSuccess) return err;
  const int64_t resident = (int64_t)r.per_sm * r.sms;
  int lanes = least;
  const int most = rows * 32 >= resident * kThreads ? 32 : kThreads;
  while (lanes < most && lanes < vectors) lanes *= 2;
  const int64_t need = (rows + kThreads / lanes - 1) / (kThreads / lanes), pieces = (vectors + lanes - 1) / lanes;
  out->lanes = lanes;
  out->grid = dim3((unsigned)std::min(need, resident), (unsigned)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(pieces, 65535), resident / need)));
  return cudaSuccess;
}

int launched(const char* name, cudaError_t err) {
  if (err == cudaSuccess) return GNB200_OK;
  return report_error(GNB200_ERR_CUDA, "%s: CUDA error: %s", name, cudaGetErrorString(err));
}

int check_four(const char* name, int64_t rows, int64_t C, int block, const float* tensor_scale) {
  if (block != 16 && block != 32) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: block is 16 or 32 channels (got %d)", name, block);
  if (block == 32 && tensor_scale) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: blocks of 32 have no scale of the whole tensor", name);
  if (rows < 0 || C < 1)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: rows must not be negative and channels be positive (got %lld, %lld)", name, (long long)rows,
                        (long long)C);
  if (C > (1 << 30) || rows >= (int64_t)1 << 31)
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: 2^31 rows or more than 2^30 channels are not supported (got %lld, %lld)", name, (long long)rows, (long long)C);
  return GNB200_OK;
}
FourRows four_rows(int64_t rows, int64_t C, int block, const float* tensor_scale, const void* codes, const void* scales) {
  FourRows p = {};
  p.codes = static_cast<uint8_t*>(const_cast<void*>(codes)), p.scales = static_cast<uint8_t*>(const_cast<void*>(scales)), p.tensor_scale = tensor_scale;
  p.rows = rows, p.C = (int)C, p.wide = (int)four_wide(C), p.tiles = (int)four_tiles(C, block);
  return p;
}

}  // namespace
}  // namespace gnb200

using namespace gnb200;

extern "C" {

size_t gnb200_4bit_code_bytes(int64_t rows, int64_t C) { return rows < 0 || C < 1 ? 0 : (size_t)rows * (size_t)(four_wide(C) / 2); }
size_t gnb200_4bit_scale_bytes(int64_t rows, int64_t C, int block) {
  return rows < 0 || C < 1 || (block != 16 && block != 32) ? 0 : (size_t)four_scale_bytes(rows, C, block);
}

int gnb200_quantize_4bit(const void* x, int64_t x_stride, int64_t rows, int64_t C, int dtype, int block, const float* tensor_scale, void* codes,
                         void* scales, void* stream) {
  const char* name = "gnb200_quantize_4bit";
  if (!dtype_ok(dtype)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if (int rc = check_four(name, rows, C, block, tensor_scale)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!x || !codes || !scales) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!on16(codes) || !on16(scales)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  const FourRows p = four_rows(rows, C, block, tensor_scale, codes, scales);
  const bool vec = on16(x) && C % VE == 0 && (rows == 1 || x_stride * size_of(dtype) % 16 == 0);
  return launched(name, with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_block(block, [&](auto b) {
      return with_flag(vec, [&](auto v) {
        constexpr int BLOCK = decltype(b)::value;
        auto kernel = &quantize_kernel<T, BLOCK, decltype(v)::value>;
        Shares s;
        const cudaError_t err = share_out(rows, (int64_t)p.tiles * 4 * (BLOCK / VE), 4 * (BLOCK / VE), (const void*)kernel, &s);
        if (err != cudaSuccess) return err;
        kernel<<<s.grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const T*>(x), x_stride, p, s.lanes);
        return cudaGetLastError();
      });
    });
  }));
}

int gnb200_dequantize_4bit(const void* codes, const void* scales, int64_t rows, int64_t C, int block, const float* tensor_scale, int dtype, void* out,
                           void* stream) {
  const char* name = "gnb200_dequantize_4bit";
  if (!dtype_ok(dtype)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if (int rc = check_four(name, rows, C, block, tensor_scale)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!out || !codes || !scales) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!on16(codes) || !on16(scales)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  const FourRows p = four_rows(rows, C, block, tensor_scale, codes, scales);
  const bool vec = on16(out) && C % VE == 0;
  return launched(name, with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_block(block, [&](auto b) {
      return with_flag(vec, [&](auto v) {
        auto kernel = &dequantize_kernel<T, decltype(b)::value, decltype(v)::value>;
        Shares s;
        const cudaError_t err = share_out(rows, (C + VE - 1) / VE, 8, (const void*)kernel, &s);
        if (err != cudaSuccess) return err;
        kernel<<<s.grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, static_cast<T*>(out), s.lanes);
        return cudaGetLastError();
      });
    });
  }));
}

int gnb200_rms_fwd_4bit(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows, int64_t C,
                        double eps, double offset, int dtype, int residual_dtype, int weight_dtype, int block, const float* tensor_scale, void* codes,
                        void* scales, void* sum, void* stream) {
  const char* name = "gnb200_rms_fwd_4bit";
  if (!residual) residual_dtype = dtype;
  if (!weight) weight_dtype = dtype;
  if (!dtype_ok(dtype) || !dtype_ok(residual_dtype) || !dtype_ok(weight_dtype))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if ((residual_dtype != dtype && residual_dtype != GNB200_F32) || (weight_dtype != dtype && weight_dtype != GNB200_F32))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: the residual and the weight have the type of x or float32", name);
  if (int rc = check_four(name, rows, C, block, tensor_scale)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!x || !codes || !scales || (residual && !sum)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!on16(codes) || !on16(scales)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  const FourRows p = four_rows(rows, C, block, tensor_scale, codes, scales);
  NormArgs a = {};
  a.x = x, a.residual = residual, a.weight = weight, a.sum = sum, a.x_stride = x_stride, a.r_stride = residual_stride, a.w_dtype = weight_dtype;
  a.eps = (float)eps, a.offset = (float)offset, a.inv_c = (float)(1.0 / (double)C);
  const bool vec = C % VE == 0 && on16(x) && on16(residual) && on16(weight) && on16(sum) &&
                   (rows == 1 || (x_stride * size_of(dtype) % 16 == 0 && (!residual || residual_stride * size_of(residual_dtype) % 16 == 0)));
  const int64_t vectors = (int64_t)p.tiles * 4 * (block / VE);
  // a warp to a row of four vectors a lane at most, where there are rows for the SMs' warps; else a CTA with one or two vectors a thread, four
  // above 16384 channels; longer rows are read twice
  const bool warp = vectors <= 128 && rows >= 148 * 8;
  int V, threads;
  if (warp) {
    V = vectors <= 32 ? 1 : vectors <= 64 ? 2 : 4;
    threads = 128;
  } else {
    V = vectors <= 256 ? 1 : vectors <= 2048 ? 2 : vectors <= 4096 ? 4 : 0;
    threads = V == 0 ? 1024 : (int)((vectors + V - 1) / V + 31) / 32 * 32;
  }
  const int64_t grid = warp ? (rows + 3) / 4 : rows;
  return launched(name, with_type(dtype, [&](auto t) {
    using Tx = decltype(t);
    const auto typed = [&](auto u) {
      using Ts = decltype(u);
      return with_block(block, [&](auto b) {
        return with_flag(vec, [&](auto is_vec) {
          constexpr int BLOCK = decltype(b)::value;
          constexpr bool VEC = decltype(is_vec)::value;
          const auto go = [&](auto kernel) {
            kernel<<<(unsigned)grid, threads, 0, static_cast<cudaStream_t>(stream)>>>(a, p);
            return cudaGetLastError();
          };
          if (warp) {
            if (V == 1) return go(&norm_kernel<Tx, Ts, BLOCK, 1, true, VEC>);
            if (V == 2) return go(&norm_kernel<Tx, Ts, BLOCK, 2, true, VEC>);
            return go(&norm_kernel<Tx, Ts, BLOCK, 4, true, VEC>);
          }
          if (V == 1) return go(&norm_kernel<Tx, Ts, BLOCK, 1, false, VEC>);
          if (V == 2) return go(&norm_kernel<Tx, Ts, BLOCK, 2, false, VEC>);
          if (V == 4) return go(&norm_kernel<Tx, Ts, BLOCK, 4, false, VEC>);
          return go(&norm_kernel<Tx, Ts, BLOCK, 0, false, VEC>);
        });
      });
    };
    if constexpr (!std::is_same<Tx, float>::value)
      if (residual_dtype == GNB200_F32) return typed(float());
    return typed(Tx());
  }));
}

}  // extern "C"
