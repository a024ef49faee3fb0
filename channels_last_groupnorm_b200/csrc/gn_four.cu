// Rows to four bits and back, and the root-mean-square norm with the residual's addition straight into four bits (formulas and layout:
// gn_four.cuh; the norm is that of gn_rms.cu: s = x + r in fp32, y = s * rsqrt(mean(s^2) + eps) * (offset + w), y not rounded before its codes).
//
// A lane holds 16 channels: a block of 16, or half of one of 32, whose largest magnitude a shuffle completes; 8 bytes of codes a lane; the scales
// of four blocks become one word.
#include <algorithm>

#include "../../include/gnb200.h"
#include "gn_four.cuh"
#include "gn_kernels.h"

namespace gnb200 {
namespace {

constexpr int VE = 16;  // channels of a lane
template <int BLOCK>
constexpr int kLanes = BLOCK / VE;  // lanes of a block

struct FourRows {
  uint8_t *codes, *scales;
  const float* tensor_scale;  // g, or NULL for one
  long long rows;
  int C, wide, tiles;
};

// Codes of the 16 channels y of vector v of a row (zeros where it has none) and the scales that its lanes share; by whole warps.
template <int BLOCK>
__device__ __forceinline__ void put(const FourRows& p, long long row, int v, bool live, const float (&y)[VE], const TensorScale& t) {
  constexpr int LANES = kLanes<BLOCK>;
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < VE; ++e) most = larger(most, fabsf(y[e]));
  if constexpr (LANES > 1) most = larger(most, __shfl_xor_sync(0xffffffffu, most, 1));
  const FourStep step = four_step<BLOCK>(most, t);
  const uint2 words = make_uint2(codes8<BLOCK>(y, step), codes8<BLOCK>(y + 8, step));
  const bool inside = v * VE < p.wide;
  if (live && inside) *reinterpret_cast<uint2*>(p.codes + (row * (p.wide / VE) + v) * 8) = words;
  const int block = v / LANES;
  uint32_t scales = inside ? step.byte << (8 * (block & 3)) : 0;
  scales |= __shfl_xor_sync(0xffffffffu, scales, LANES);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2 * LANES);
  if (live && v % (4 * LANES) == 0) put_scales(p.scales, row, p.rows, block >> 2, p.tiles, scales);
}
// ---------------------------------------------------------------------------------------------
// 16 channels of a row
// ---------------------------------------------------------------------------------------------
// A tensor's bytes: vectors that reach beyond a row may be read as long as they stay in these.
struct Bounds {
  const char *begin, *end;
};
// Aligned (VEC, rows of whole 8 channels), or from any address: then the 16-byte vectors that the channels lie in are read whole and shifted into place,
// three of them for 16 bits where element by element it were 16 loads (9001 x 1111 bf16 to four bits 66 us so); element by element at the ends of a
// row and where a vector would reach out of the tensor.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* row, int v, int C, const Bounds& bounds, float (&f)[VE]) {
  constexpr int N = VE * (int)sizeof(T) / 16;  // vectors
  const T* at = row + v * VE;
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float part[16 / sizeof(T)];
      if (v * VE + k * (int)(16 / sizeof(T)) < C) {
        unpack16<T, 16 / sizeof(T)>(reinterpret_cast<const uint4*>(at)[k], part);
      } else {
#pragma unroll
        for (int e = 0; e < (int)(16 / sizeof(T)); ++e) part[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < (int)(16 / sizeof(T)); ++e) f[k * (16 / sizeof(T)) + e] = part[e];
    }
  } else {
    const uintptr_t a = reinterpret_cast<uintptr_t>(at);
    const char* const from = reinterpret_cast<const char*>(a & ~(uintptr_t)15);
    if (v * VE + VE <= C && from >= bounds.begin && from + 16 * (N + 1) <= bounds.end) {
      uint32_t w[4 * (N + 1)];
#pragma unroll
      for (int k = 0; k <= N; ++k) {
        const uint4 q = reinterpret_cast<const uint4*>(from)[k];
        w[4 * k] = q.x, w[4 * k + 1] = q.y, w[4 * k + 2] = q.z, w[4 * k + 3] = q.w;
      }
      const bool two = a & 8, one = a & 4, half = a & 2;
#pragma unroll
      for (int k = 0; k < 4 * N + 2; ++k) w[k] = two ? w[k + 2] : w[k];
#pragma unroll
      for (int k = 0; k < 4 * N + 1; ++k) w[k] = one ? w[k + 1] : w[k];
#pragma unroll
      for (int k = 0; k < 4 * N; ++k) {
        if constexpr (sizeof(T) == 4) {
          f[k] = __uint_as_float(w[k]);
        } else {
          const uint32_t pair = __funnelshift_r(w[k], w[k + 1], half ? 16 : 0);
          float part[2];
          unpack<T, 2>(*reinterpret_cast<const Pack<T, 2>*>(&pair), part);
          f[2 * k] = part[0], f[2 * k + 1] = part[1];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = v * VE + e < C ? load_param<T>(at, e) : 0.f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store16(T* row, int v, int C, const float (&f)[VE]) {
  constexpr int W = 16 / sizeof(T);
  T* at = row + v * VE;
#pragma unroll
  for (int k = 0; k < VE / W; ++k) {
    float part[W];
#pragma unroll
    for (int e = 0; e < W; ++e) part[e] = f[k * W + e];
    if constexpr (VEC) {
      if (v * VE + k * W < C) store_vec<T, W>(at + k * W, pack<T, W>(part));
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (v * VE + k * W + e < C) at[k * W + e] = store_param<T>(part[e]);
    }
  }
}
__device__ __forceinline__ void zero(float (&f)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = 0.f;
}

// 16 channels as they lie in an aligned row
template <typename T>
struct Raw {
  uint4 q[sizeof(T)];
  __device__ __forceinline__ void load(const T* row, int v, int C) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T); ++k) {
      q[k] = make_uint4(0, 0, 0, 0);
      if (v * VE + k * (int)(16 / sizeof(T)) < C) q[k] = reinterpret_cast<const uint4*>(row + v * VE)[k];
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[VE]) const {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < (int)sizeof(T); ++k) {
      float part[W];
      unpack16<T, W>(q[k], part);
#pragma unroll
      for (int e = 0; e < W; ++e) f[k * W + e] = part[e];
    }
  }
};

// ---------------------------------------------------------------------------------------------
// Rows to four bits and back
// ---------------------------------------------------------------------------------------------
constexpr int kThreads = 256;

// 2^shift threads share a row's piece; the grid's second axis shares a row out.  Aligned rows: a lane asks for its next 16 channels before it works on these.
template <typename T, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* x, long long x_stride, const Bounds bounds, const FourRows p, int shift) {
  grid_dep_launch_dependents();
  const int lanes = 1 << shift, per_cta = kThreads >> shift, lane = threadIdx.x & (lanes - 1), vectors = p.tiles * 4 * kLanes<BLOCK>, step = gridDim.y << shift;
  const TensorScale t(BLOCK == 16 ? p.tensor_scale : nullptr);
  const long long rows_step = (long long)gridDim.x * per_cta;
  const int begin = blockIdx.y << shift;
  long long base = (long long)blockIdx.x * per_cta, row = base + (threadIdx.x >> shift);  // (base and first: the same for the warp)
  int first = begin;
  Raw<T> next;
  const auto ask = [&]() {
    if (VEC && row < p.rows && (first + lane) * VE < p.C) next.load(x + row * x_stride, first + lane, p.C);
  };
  ask();
  while (base < p.rows) {
    const long long here = row;
    const int v = first + lane;
    const bool live = here < p.rows;
    float y[VE];
    zero(y);
    if (live && v * VE < p.C) {
      if constexpr (VEC)
        next.unpack(y);
      else
        load16<T, false>(x + here * x_stride, v, p.C, bounds, y);
    }
    first += step;
    if (first >= vectors) first = begin, base += rows_step, row += rows_step;
    if (base < p.rows) ask();
    put<BLOCK>(p, here, v, live && v < vectors, y, t);
  }
  clear_behind(p.scales, p.rows, p.tiles, (blockIdx.y * gridDim.x + blockIdx.x) * kThreads + threadIdx.x, gridDim.x * gridDim.y * kThreads);
}

__device__ __forceinline__ void values_of(uint32_t word, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 two = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(word >> (4 * e)), __NV_E2M1)));
    f[e] = two.x, f[e + 1] = two.y;
  }
}
// VEC: output rows of whole 16-byte vectors on their boundaries.
template <typename T, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const FourRows p, T* out, int shift) {
  const int lanes = 1 << shift, per_cta = kThreads >> shift, lane = threadIdx.x & (lanes - 1), step = gridDim.y << shift;
  const float g = BLOCK == 16 && p.tensor_scale ? *p.tensor_scale : 1.f;
  const auto scale_at = [&](long long row, int channel) {
    const int block = channel / BLOCK;
    return scale_value(p.scales[four_scale_at(row, block >> 2, p.tiles) + (block & 3)], BLOCK);
  };
  for (long long row = (long long)blockIdx.x * per_cta + (threadIdx.x >> shift); row < p.rows; row += (long long)gridDim.x * per_cta) {
    const uint8_t* const codes = p.codes + row * (p.wide / 2);
    T* const to = out + row * p.C;
    if constexpr (VEC) {
      // a vector of the output a lane, so that a warp's stores lie side by side (16 codes a lane: 16384 x 8192 bf16 90 us); two under way
      constexpr int W = 16 / sizeof(T);
      for (int v = (blockIdx.y << shift) + lane; v * W < p.C; v += 2 * step) {
        uint32_t word[2];
        float scale[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = (v + k * step) * W;
          word[k] = 0, scale[k] = 0.f;
          if (at < p.C) {
            word[k] = W == 8 ? *reinterpret_cast<const uint32_t*>(codes + at / 2) : *reinterpret_cast<const uint16_t*>(codes + at / 2);
            scale[k] = scale_at(row, at);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = (v + k * step) * W;
          float f[8], o[W];
          values_of(word[k], f);
#pragma unroll
          for (int e = 0; e < W; ++e) o[e] = f[e];
          scale_each(o, scale[k]);
          if constexpr (BLOCK == 16) scale_each(o, g);
          if (at < p.C) store_vec<T, W>(to + at, pack<T, W>(o));
        }
      }
    } else {
      // in the frame of the output's 16-byte vectors, whose first and last have elements of the rows beside this one; 8 codes from any one on
      constexpr int W = 16 / sizeof(T);
      const int skew = (int)(reinterpret_cast<uintptr_t>(to) / sizeof(T) % W), count = (p.C + skew + W - 1) / W, words = p.wide / 8;
      for (int v = (blockIdx.y << shift) + lane; v < count; v += step) {
        const int c = v * W - skew, at = c < 0 ? -1 : c / 8;
        const uint32_t* const w = reinterpret_cast<const uint32_t*>(codes);
        const uint32_t below = at >= 0 ? w[at] : 0, above = at + 1 < words ? w[at + 1] : 0;
        float f[8];
        values_of(__funnelshift_r(below, above, 4 * (c & 7)), f);
        const int border = ((c + W - 1) / BLOCK) * BLOCK;  // channels from here on have the last one's scale
        const float last = scale_at(row, min(c + W - 1, p.C - 1)), first = c >= 0 && c < border ? scale_at(row, c) : last;
        const bool whole = c >= 0 && c + W <= p.C;
        float o[W];
#pragma unroll
        for (int e = 0; e < W; ++e) o[e] = f[e] * (c + e < border ? first : last) * g;
        if (whole) {
          store_vec<T, W>(to + c, pack<T, W>(o));
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e)
            if ((unsigned)(c + e) < (unsigned)p.C) to[c + e] = store_param<T>(o[e]);
        }
      }
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
  Bounds x_bounds, r_bounds;
  int w_dtype;
  float eps, offset, inv_c;
};

// (offset + w) of 16 channels, from addresses on 16 bytes (VEC) or any
template <bool VEC>
__device__ __forceinline__ void weight16(const NormArgs& a, int v, int C, float (&w)[VE]) {
  if constexpr (VEC) {
    const Bounds none = {};
    if (a.w_dtype == 0)
      load16<float, true>(static_cast<const float*>(a.weight), v, C, none, w);
    else if (a.w_dtype == 1)
      load16<__half, true>(static_cast<const __half*>(a.weight), v, C, none, w);
    else
      load16<__nv_bfloat16, true>(static_cast<const __nv_bfloat16*>(a.weight), v, C, none, w);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = v * VE + e < C ? param_at(a.weight, a.w_dtype, v * VE + e, 1.f) : 0.f;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) w[e] += a.offset;
}

// A row to a warp (WARP) or a CTA, V vectors a thread in registers; V = 0: rows of any length, read twice.  The CTAs that are resident walk over the
// rows; of an aligned row with one vector a thread the next one's vectors are asked for before this one's sum.
template <typename Tx, typename Ts, int BLOCK, int V, bool WARP, bool VEC, bool RES>
__global__ void __launch_bounds__(WARP ? 128 : V == 1 ? 512 : 1024) norm_kernel(const NormArgs a, const FourRows p) {
  constexpr int HELD = V > 0 ? V : 1;
  constexpr bool AHEAD = VEC && V == 1;
  __shared__ TeamSlots slots;
  grid_dep_launch_dependents();
  const int threads = WARP ? 32 : (int)blockDim.x, at = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const int per_cta = WARP ? (int)blockDim.x >> 5 : 1;
  const int vectors = p.tiles * 4 * kLanes<BLOCK>;
  if constexpr (!WARP) clear<false>(slots, threads, 0, at);
  const TensorScale t(BLOCK == 16 ? p.tensor_scale : nullptr);
  int turn = 0;
  Raw<Tx> next_x;
  Raw<Ts> next_r;
  const auto ask = [&](long long row) {
    if (row < p.rows && at * VE < p.C) {
      next_x.load(static_cast<const Tx*>(a.x) + row * a.x_stride, at, p.C);
      if constexpr (RES) next_r.load(static_cast<const Ts*>(a.residual) + row * a.r_stride, at, p.C);
    }
  };
  long long row = (long long)blockIdx.x * per_cta + (WARP ? (int)threadIdx.x >> 5 : 0);
  if constexpr (AHEAD) ask(row);
  for (; row < p.rows; row += (long long)gridDim.x * per_cta) {  // (whole warps)
    const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_stride;
    const Ts* r = RES ? static_cast<const Ts*>(a.residual) + row * a.r_stride : nullptr;
    auto sum_of = [&](int v, float (&s)[VE]) {
      zero(s);
      if (v * VE < p.C) {
        if constexpr (AHEAD)
          next_x.unpack(s);
        else
          load16<Tx, VEC>(x, v, p.C, a.x_bounds, s);
        if constexpr (RES) {
          float f[VE];
          if constexpr (AHEAD)
            next_r.unpack(f);
          else
            load16<Ts, VEC>(r, v, p.C, a.r_bounds, f);
          add_each(s, f);
        }
      }
    };
    float s[HELD][VE], sq[2] = {0.f, 0.f};
    if constexpr (V > 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) sum_of(at + k * threads, s[k]);
      if constexpr (AHEAD) ask(row + (long long)gridDim.x * per_cta);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int v = at + k * threads;
        if (RES && v * VE < p.C) store16<Ts, VEC>(static_cast<Ts*>(a.sum) + row * p.C, v, p.C, s[k]);
        dot_each(sq, s[k], s[k]);
      }
    } else {
      for (int v = at; v * VE < p.C; v += threads) {
        sum_of(v, s[0]);
        dot_each(sq, s[0], s[0]);
      }
    }
    const float all = WARP ? lanes_sum(sq[0] + sq[1], 32) : team_sum<false>(sq[0] + sq[1], slots, turn, threads, 0);
    const float rstd = __frsqrt_rn(fmaf(all, a.inv_c, a.eps));
    auto finish = [&](int v, float (&y)[VE]) {
      if (v * VE < p.C) {
        scale_each(y, rstd);
        if (a.weight) {
          float w[VE];
          weight16<VEC>(a, v, p.C, w);
          mul_each(y, w);
        }
        if (v * VE + VE > p.C) {  // (behind the row a NaN rstd would leave NaN in the zeros)
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (v * VE + e >= p.C) y[e] = 0.f;
        }
      }
      put<BLOCK>(p, row, v, v < vectors, y, t);
    };
    if constexpr (V > 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) finish(at + k * threads, s[k]);
    } else {
      for (int first = 0; first < vectors; first += threads) {
        sum_of(first + at, s[0]);  // (the last look at these: the sum may be the residual's own buffer)
        if (RES && (first + at) * VE < p.C) store16<Ts, VEC>(static_cast<Ts*>(a.sum) + row * p.C, first + at, p.C, s[0]);
        finish(first + at, s[0]);
      }
    }
  }
  clear_behind(p.scales, p.rows, p.tiles, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
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
Bounds bounds_of(const void* p, int64_t rows, int64_t stride, int64_t C, int size) {
  const char* const begin = static_cast<const char*>(p);
  return p && stride >= 0 ? Bounds{begin, begin + ((rows - 1) * stride + C) * size} : Bounds{};
}

struct Shares {
  int shift;
  dim3 grid;
};
// Lanes of a row's piece: a row's vectors where they are few, a warp's where there are rows enough to fill the GPU with warps, otherwise the
// CTA; the rest of a row goes round, or to other CTAs while there are SMs without one.
cudaError_t share_out(int64_t rows, int64_t vectors, int least, const void* kernel, Shares* out) {
  Residency r = {};
  const cudaError_t err = residency(kernel, kThreads, 0, &r);
  if (err != cudaSuccess) return err;
  const int64_t resident = (int64_t)r.per_sm * r.sms;
  const int most = rows * 32 >= resident * kThreads ? 5 : 8;
  int shift = 0;
  while (1 << shift < least || (shift < most && 1 << shift < vectors)) ++shift;
  const int64_t need = (rows + (kThreads >> shift) - 1) / (kThreads >> shift), pieces = (vectors + (1 << shift) - 1) >> shift;
  out->shift = shift;
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
  const int width = 16 / size_of(dtype);
  const bool vec = on16(x) && C % width == 0 && (rows == 1 || x_stride % width == 0);
  return launched(name, with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_block(block, [&](auto b) {
      return with_flag(vec, [&](auto v) {
        constexpr int BLOCK = decltype(b)::value;
        auto kernel = &quantize_kernel<T, BLOCK, decltype(v)::value>;
        Shares s;
        const cudaError_t err = share_out(rows, (int64_t)p.tiles * 4 * kLanes<BLOCK>, 4 * kLanes<BLOCK>, (const void*)kernel, &s);
        if (err != cudaSuccess) return err;
        kernel<<<s.grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const T*>(x), x_stride, bounds_of(x, rows, x_stride, C, sizeof(T)), p, s.shift);
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
  const int width = 16 / size_of(dtype);
  const bool vec = on16(out) && C % width == 0;
  return launched(name, with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_block(block, [&](auto b) {
      return with_flag(vec, [&](auto v) {
        auto kernel = &dequantize_kernel<T, decltype(b)::value, decltype(v)::value>;
        Shares s;
        const cudaError_t err = share_out(rows, C / width + 1, 4, (const void*)kernel, &s);
        if (err != cudaSuccess) return err;
        kernel<<<s.grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, static_cast<T*>(out), s.shift);
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
  const FourNorm n = {x, residual, weight, sum, p.codes, p.scales, tensor_scale, rows, x_stride, residual_stride, (int)C, block, dtype, residual_dtype, weight_dtype, eps, offset};
  const cudaError_t how = launch_rms_4bit(n, static_cast<cudaStream_t>(stream));
  if (how != cudaErrorInvalidValue) return launched(name, how);
  NormArgs a = {};
  a.x = x, a.residual = residual, a.weight = weight, a.sum = sum, a.x_stride = x_stride, a.r_stride = residual_stride, a.w_dtype = weight_dtype;
  a.eps = (float)eps, a.offset = (float)offset, a.inv_c = (float)(1.0 / (double)C);
  a.x_bounds = bounds_of(x, rows, x_stride, C, size_of(dtype)), a.r_bounds = bounds_of(residual, rows, residual_stride, C, size_of(residual_dtype));
  const bool vec = C % 8 == 0 && on16(x) && on16(residual) && on16(weight) && on16(sum) &&
                   (rows == 1 || (x_stride * size_of(dtype) % 16 == 0 && (!residual || residual_stride * size_of(residual_dtype) % 16 == 0)));
  const int64_t vectors = (int64_t)p.tiles * 4 * (block / VE);
  // a warp to a row of four vectors a lane at most, where there are rows for the SMs' warps; else a CTA with one vector a thread, two above 8192
  // channels; longer rows are read twice
  const bool warp = vectors <= 128 && rows >= 148 * 8;
  int V, threads;
  if (warp) {
    V = vectors <= 32 ? 1 : vectors <= 64 ? 2 : 4;
    threads = 128;
  } else {
    V = vectors <= 512 ? 1 : vectors <= 2048 ? 2 : 0;
    threads = V == 0 ? 1024 : (int)((vectors + V - 1) / V + 31) / 32 * 32;
  }
  return launched(name, with_type(dtype, [&](auto t) {
    using Tx = decltype(t);
    const auto typed = [&](auto u, auto is_res) {
      using Ts = decltype(u);
      return with_block(block, [&](auto b) {
        return with_flag(vec, [&](auto is_vec) {
          constexpr int BLOCK = decltype(b)::value;
          constexpr bool VEC = decltype(is_vec)::value, RES = decltype(is_res)::value;
          const auto go = [&](void (*kernel)(const NormArgs, const FourRows)) {
            Residency r = {};
            const cudaError_t err = residency((const void*)kernel, threads, 0, &r);
            if (err != cudaSuccess) return err;
            const int64_t need = warp ? (rows + 3) / 4 : rows;
            kernel<<<(unsigned)std::min<int64_t>(need, (int64_t)r.per_sm * r.sms), threads, 0, static_cast<cudaStream_t>(stream)>>>(a, p);
            return cudaGetLastError();
          };
          if (warp) {
            if (V == 1) return go(&norm_kernel<Tx, Ts, BLOCK, 1, true, VEC, RES>);
            if (V == 2) return go(&norm_kernel<Tx, Ts, BLOCK, 2, true, VEC, RES>);
            return go(&norm_kernel<Tx, Ts, BLOCK, 4, true, VEC, RES>);
          }
          if (V == 1) return go(&norm_kernel<Tx, Ts, BLOCK, 1, false, VEC, RES>);
          if (V == 2) return go(&norm_kernel<Tx, Ts, BLOCK, 2, false, VEC, RES>);
          return go(&norm_kernel<Tx, Ts, BLOCK, 0, false, VEC, RES>);
        });
      });
    };
    if (!residual) return typed(Tx(), std::false_type());
    if constexpr (!std::is_same<Tx, float>::value)
      if (residual_dtype == GNB200_F32) return typed(float(), std::true_type());
    return typed(Tx(), std::true_type());
  }));
}

}  // extern "C"
