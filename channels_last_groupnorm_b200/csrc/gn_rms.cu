// Root-mean-square norm of token rows with the residual's addition: forward, forward with an 8-bit output and
// scales, backward.
//
//   s = x + r                      added in fp32, stored rounded once to r's type; the norm takes the unrounded sum
//   y = s * rstd * (offset + w)    rstd = 1 / sqrt(mean(s^2) + eps) over the C channels of a row
//   q = y / scale                  scale = max(|y|) / largest code, per row or per block of channels; at least 2^-126
//   d = ds + rstd * (g - n * mean(g * n))   with n = s * rstd, g = dy * (offset + w): the gradient of x and of r
//   dw = sum over rows of dy * n
//
// Every element is read and written once: a row's elements stay in registers between the sum over the row and the
// output.  Rows of up to four vectors a lane belong to a group of lanes of one warp (shuffles only), longer ones to a CTA (one barrier
// a sum); longer ones still are read twice, element by element (`any`).  The grid holds the CTAs that are resident at once; each keeps its
// channels' weights in registers, walks over the rows and asks for its next row before it reduces the present one.
#include <algorithm>

#include "../../include/gnb200.h"
#include "gn_kernels.h"
#include "gn_tokens.cuh"

namespace gnb200 {
namespace {

constexpr int kWarpThreads = 128;  // CTA size of the kernels with one group of lanes per row
constexpr int kMostThreads = 512;  // CTA size limit of the kernels with one CTA per row
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126: its reciprocal is finite, a block of zeros gets codes of zero

struct RmsFwd {
  const void *x, *residual, *weight;
  void *y, *sum;  // y: or the codes
  float *rstd, *scale;
  long long rows, x_stride, r_stride;
  int C, lanes, w_dtype, block, blocks, format;
  float eps, offset, inv_c;
};

// ---------------------------------------------------------------------------------------------
// 8-bit codes
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float scale_of(uint32_t most, int format) {
  const float largest = format == GNB200_E4M3 ? 448.f : 127.f;
  const float s = __uint_as_float(most) / largest;
  return s < kSmallestScale ? kSmallestScale : s;  // (a NaN stays)
}
template <int VE>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&f)[VE], float inverse, int format) {
  Pack<uint8_t, VE> c;
  if (format == GNB200_E4M3) {
    if constexpr (VE % 2 == 0) {
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const __nv_fp8x2_storage_t two =
            __nv_cvt_float2_to_fp8x2(make_float2(f[e] * inverse, f[e + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
        c.v[e] = (uint8_t)(two & 0xff);
        c.v[e + 1] = (uint8_t)(two >> 8);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) c.v[e] = (uint8_t)__nv_cvt_float_to_fp8(f[e] * inverse, __NV_SATFINITE, __NV_E4M3);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) c.v[e] = (uint8_t)(int8_t)max(-127, min(127, __float2int_rn(f[e] * inverse)));
  }
  if constexpr (VE == 8)
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&c);
  else if constexpr (VE == 4)
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(&c);
  else
    *p = c.v[0];
}

// ---------------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------------
template <typename T, int VE, int V>
__device__ __forceinline__ void fetch(Pack<T, VE> (&out)[V], const T* row, int first, int step, int nvec) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = first + v * step;
    if (at < nvec) out[v] = load_vec<T, VE>(row + (long long)at * VE);
  }
}

// (offset + w) of this thread's channels
template <int VE, int V>
__device__ __forceinline__ void fetch_weight(float (&w)[V][VE], const void* p, int dtype, float offset, int first, int step, int nvec) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = first + v * step;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[v][e] = 1.f;
    if (p != nullptr && at < nvec) {
#pragma unroll
      for (int e = 0; e < VE; ++e) w[v][e] = offset + param_at(p, dtype, (long long)at * VE + e, 1.f);
    }
  }
}

template <typename Tx, typename Ts, int VE, int V, bool WARP, bool Q>
__global__ void __launch_bounds__(WARP ? kWarpThreads : kMostThreads) rms_fwd_kernel(const RmsFwd p) {
  __shared__ float slots[2][32];
  __shared__ uint32_t most[VE == 1 && Q ? V * (kMostThreads / 32) : 32];
  const int lanes = WARP ? p.lanes : (int)blockDim.x;
  const int first = WARP ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
  const int nvec = p.C / VE;
  const long long per_cta = WARP ? kWarpThreads / lanes : 1;
  const long long step = per_cta * gridDim.x;
  long long row = blockIdx.x * per_cta + (WARP ? (int)threadIdx.x / lanes : 0);
  const Tx* x = static_cast<const Tx*>(p.x);
  const Ts* r = static_cast<const Ts*>(p.residual);
  Pack<Tx, VE> xv[V];
  Pack<Ts, VE> rv[V];
  if (row < p.rows) {
    fetch<Tx, VE, V>(xv, x + row * p.x_stride, first, lanes, nvec);
    if (r) fetch<Ts, VE, V>(rv, r + row * p.r_stride, first, lanes, nvec);
  }
  float w[V][VE];
  fetch_weight<VE, V>(w, p.weight, p.w_dtype, p.offset, first, lanes, nvec);
  int turn = 0;
  // (every thread of a warp takes the same number of turns: the shuffles want all lanes)
  for (long long base = blockIdx.x * per_cta; base < p.rows; base += step, row += step) {
    const bool live = row < p.rows;
    float s[V][VE];
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (live && first + v * lanes < nvec) {
        unpack<Tx, VE>(xv[v], s[v]);
        if (r) {
          float f[VE];
          unpack<Ts, VE>(rv[v], f);
#pragma unroll
          for (int e = 0; e < VE; ++e) s[v][e] += f[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) s[v][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) sq = fmaf(s[v][e], s[v][e], sq);
    }
    const long long next = row + step;
    if (next < p.rows) {
      fetch<Tx, VE, V>(xv, x + next * p.x_stride, first, lanes, nvec);
      if (r) fetch<Ts, VE, V>(rv, r + next * p.r_stride, first, lanes, nvec);
    }
    if (r && live) {
      Ts* out = static_cast<Ts*>(p.sum) + row * p.C;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (first + v * lanes < nvec) store_vec<Ts, VE>(out + (first + v * lanes) * VE, pack<Ts, VE>(s[v]));
    }
    sq = WARP ? lanes_sum(sq, lanes) : cta_sum(sq, slots, turn);
    const float rstd = 1.f / sqrtf(fmaf(sq, p.inv_c, p.eps));
    if (p.rstd && live && first == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < VE; ++e) s[v][e] = s[v][e] * rstd * w[v][e];
    if constexpr (!Q) {
      if (live) {
        Tx* out = static_cast<Tx*>(p.y) + row * p.C;
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (first + v * lanes < nvec) store_vec<Tx, VE>(out + (first + v * lanes) * VE, pack<Tx, VE>(s[v]));
      }
    } else {
      uint8_t* out = static_cast<uint8_t*>(p.y) + row * p.C;
      uint32_t m[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        m[v] = 0;
        if (first + v * lanes < nvec) {  // (beyond the row a NaN rstd would leave NaN in the zeros)
#pragma unroll
          for (int e = 0; e < VE; ++e) m[v] = max(m[v], magnitude(s[v][e]));
        }
      }
      if (p.block == 0) {
        uint32_t all = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) all = max(all, m[v]);
        all = WARP ? lanes_max(all, lanes) : cta_max(all, most);
        const float scale = scale_of(all, p.format), inverse = 1.f / scale;
        if (live && first == 0) p.scale[row] = scale;
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (live && first + v * lanes < nvec) store_codes<VE>(out + (first + v * lanes) * VE, s[v], inverse, p.format);
      } else if constexpr (VE > 1) {
        // a block's vectors lie in neighbouring lanes: block / VE of them, at most a warp's
        const int share = p.block / VE, among = min(share, WARP ? lanes : 32);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int at = first + v * lanes;
          const float scale = scale_of(lanes_max(m[v], among), p.format), inverse = 1.f / scale;
          if (live && at < nvec) {
            if (at % share == 0) p.scale[row * p.blocks + at / share] = scale;
            store_codes<VE>(out + at * VE, s[v], inverse, p.format);
          }
        }
      } else {
        // single elements: a block is one, two or four warps' worth; entry i of `most` is that of channels 32 i to 32 i + 31
        const int nwarps = lanes >> 5, warp = first >> 5, share = p.block / 32;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const uint32_t mv = __reduce_max_sync(0xffffffffu, m[v]);
          if ((first & 31) == 0) most[v * nwarps + warp] = mv;
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int at = first + v * lanes;
          if (at < nvec) {
            const int from = at / p.block * share, to = min(from + share, V * nwarps);
            uint32_t all = 0;
            for (int i = from; i < to; ++i) all = max(all, most[i]);
            const float scale = scale_of(all, p.format);
            if (at % p.block == 0) p.scale[row * p.blocks + at / p.block] = scale;
            store_codes<1>(out + at, s[v], 1.f / scale, p.format);
          }
        }
      }
    }
  }
}

// Rows of any length: one CTA per row, element by element, read once for the sum and once more for each thing that needs it.
template <typename Tx, typename Ts, bool Q>
__global__ void __launch_bounds__(kMostThreads) rms_fwd_any_kernel(const RmsFwd p) {
  __shared__ float slots[2][32];
  __shared__ uint32_t most[32];
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const Tx* x = static_cast<const Tx*>(p.x) + row * p.x_stride;
    const Ts* r = p.residual ? static_cast<const Ts*>(p.residual) + row * p.r_stride : nullptr;
    auto sum_at = [&](int i) {
      float s = load_param<Tx>(x, i);
      if (r) s += load_param<Ts>(r, i);
      return s;
    };
    float sq = 0.f;
    for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
      const float s = sum_at(i);
      sq = fmaf(s, s, sq);
      if (r) static_cast<Ts*>(p.sum)[row * p.C + i] = store_param<Ts>(s);
    }
    sq = cta_sum(sq, slots, turn);
    const float rstd = 1.f / sqrtf(fmaf(sq, p.inv_c, p.eps));
    if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
    auto y_at = [&](int i) { return sum_at(i) * rstd * (p.weight ? p.offset + param_at(p.weight, p.w_dtype, i, 1.f) : 1.f); };
    if constexpr (!Q) {
      for (int i = threadIdx.x; i < p.C; i += blockDim.x) static_cast<Tx*>(p.y)[row * p.C + i] = store_param<Tx>(y_at(i));
    } else {
      uint8_t* out = static_cast<uint8_t*>(p.y) + row * p.C;
      if (p.block == 0) {
        uint32_t m = 0;
        for (int i = threadIdx.x; i < p.C; i += blockDim.x) m = max(m, magnitude(y_at(i)));
        const float scale = scale_of(cta_max(m, most), p.format), inverse = 1.f / scale;
        if (threadIdx.x == 0) p.scale[row] = scale;
        for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
          const float f[1] = {y_at(i)};
          store_codes<1>(out + i, f, inverse, p.format);
        }
      } else {  // one warp per block of at most 128 channels
        const int lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
        for (int b = threadIdx.x >> 5; b < p.blocks; b += nwarps) {
          float f[4][1];
          uint32_t m = 0;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int in = lane + 32 * v, i = b * p.block + in;
            f[v][0] = in < p.block && i < p.C ? y_at(i) : 0.f;
            m = max(m, magnitude(f[v][0]));
          }
          const float scale = scale_of(__reduce_max_sync(0xffffffffu, m), p.format), inverse = 1.f / scale;
          if (lane == 0) p.scale[row * p.blocks + b] = scale;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int in = lane + 32 * v, i = b * p.block + in;
            if (in < p.block && i < p.C) store_codes<1>(out + i, f[v], inverse, p.format);
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------------
struct RmsBwd {
  const void *dy, *dsum, *sum, *addend, *weight;  // s = sum, or sum + addend (dy's type) where the stored sum was rounded to 16 bits
  const float* rstd;
  void *dx, *dsum_out;  // the same gradient in dy's type and, where sum has another type, in sum's
  float* part;          // one row of C floats per CTA, or NULL
  long long rows, dy_stride, ds_stride, s_stride, a_stride;
  int C, lanes, w_dtype;
  float offset, inv_c;
};

template <typename Tx, typename Ts, int VE, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpThreads : kMostThreads) rms_bwd_kernel(const RmsBwd p) {
  __shared__ float slots[2][32];
  const int lanes = WARP ? p.lanes : (int)blockDim.x;
  const int first = WARP ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
  const int nvec = p.C / VE;
  const long long per_cta = WARP ? kWarpThreads / lanes : 1;
  const long long step = per_cta * gridDim.x;
  long long row = blockIdx.x * per_cta + (WARP ? (int)threadIdx.x / lanes : 0);
  grid_dep_launch_dependents();
  const Tx* dy = static_cast<const Tx*>(p.dy);
  const Tx* add = static_cast<const Tx*>(p.addend);
  const Ts *ds = static_cast<const Ts*>(p.dsum), *sum = static_cast<const Ts*>(p.sum);
  Pack<Tx, VE> yv[V], av[V];
  Pack<Ts, VE> sv[V], dv[V];
  float rn = 0.f;
  auto ask = [&](long long at) {
    fetch<Tx, VE, V>(yv, dy + at * p.dy_stride, first, lanes, nvec);
    fetch<Ts, VE, V>(sv, sum + at * p.s_stride, first, lanes, nvec);
    if (add) fetch<Tx, VE, V>(av, add + at * p.a_stride, first, lanes, nvec);
    if (ds) fetch<Ts, VE, V>(dv, ds + at * p.ds_stride, first, lanes, nvec);
    rn = p.rstd[at];
  };
  if (row < p.rows) ask(row);
  float w[V][VE], dw[V][VE];
  fetch_weight<VE, V>(w, p.weight, p.w_dtype, p.offset, first, lanes, nvec);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < VE; ++e) dw[v][e] = 0.f;
  int turn = 0;
  for (long long base = blockIdx.x * per_cta; base < p.rows; base += step, row += step) {
    const bool live = row < p.rows;
    const float rstd = rn;
    float g[V][VE], n[V][VE], d[V][VE];
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int e = 0; e < VE; ++e) g[v][e] = n[v][e] = d[v][e] = 0.f;
      if (live && first + v * lanes < nvec) {
        unpack<Tx, VE>(yv[v], g[v]);
        unpack<Ts, VE>(sv[v], n[v]);
        if (add) {
          float f[VE];
          unpack<Tx, VE>(av[v], f);
#pragma unroll
          for (int e = 0; e < VE; ++e) n[v][e] += f[e];
        }
        if (ds) unpack<Ts, VE>(dv[v], d[v]);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          n[v][e] *= rstd;
          dw[v][e] = fmaf(g[v][e], n[v][e], dw[v][e]);
          g[v][e] *= w[v][e];
          dot = fmaf(g[v][e], n[v][e], dot);
        }
      }
    }
    if (row + step < p.rows) ask(row + step);
    const float c = (WARP ? lanes_sum(dot, lanes) : cta_sum(dot, slots, turn)) * p.inv_c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (live && first + v * lanes < nvec) {
        const long long at = row * p.C + (first + v * lanes) * VE;
#pragma unroll
        for (int e = 0; e < VE; ++e) d[v][e] = fmaf(rstd, fmaf(-n[v][e], c, g[v][e]), d[v][e]);
        store_vec<Tx, VE>(static_cast<Tx*>(p.dx) + at, pack<Tx, VE>(d[v]));
        if constexpr (!std::is_same<Tx, Ts>::value)
          if (p.dsum_out) store_vec<Ts, VE>(static_cast<Ts*>(p.dsum_out) + at, pack<Ts, VE>(d[v]));
      }
    }
  }
  if (p.part == nullptr) return;
  float* part = p.part + (long long)blockIdx.x * p.C;
  if constexpr (!WARP) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (first + v * lanes < nvec) {
#pragma unroll
        for (int e = 0; e < VE; ++e) part[(first + v * lanes) * VE + e] = dw[v][e];
      }
  } else {
    // the groups of lanes hold the same channels: added in order, one vector at a time
    __shared__ float share[kWarpThreads * VE];
    const int groups = kWarpThreads / lanes;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VE; ++e) share[(threadIdx.x / lanes * VE + e) * lanes + first] = dw[v][e];
      __syncthreads();
      for (int i = threadIdx.x; i < lanes * VE; i += kWarpThreads) {
        const int lane = i / VE, e = i % VE, channel = (lane + v * lanes) * VE + e;
        float t = 0.f;
        for (int g = 0; g < groups; ++g) t += share[(g * VE + e) * lanes + lane];
        if (channel < p.C) part[channel] = t;
      }
    }
  }
}

template <typename Tx, typename Ts>
__global__ void __launch_bounds__(kMostThreads) rms_bwd_any_kernel(const RmsBwd p) {
  __shared__ float slots[2][32];
  int turn = 0;
  grid_dep_launch_dependents();
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const Tx* dy = static_cast<const Tx*>(p.dy) + row * p.dy_stride;
    const Ts* sum = static_cast<const Ts*>(p.sum) + row * p.s_stride;
    const Ts* ds = p.dsum ? static_cast<const Ts*>(p.dsum) + row * p.ds_stride : nullptr;
    const Tx* add = p.addend ? static_cast<const Tx*>(p.addend) + row * p.a_stride : nullptr;
    const float rstd = p.rstd[row];
    auto g_at = [&](int i) { return load_param<Tx>(dy, i) * (p.weight ? p.offset + param_at(p.weight, p.w_dtype, i, 1.f) : 1.f); };
    auto n_at = [&](int i) { return (load_param<Ts>(sum, i) + (add ? load_param<Tx>(add, i) : 0.f)) * rstd; };
    float dot = 0.f;
    for (int i = threadIdx.x; i < p.C; i += blockDim.x) dot = fmaf(g_at(i), n_at(i), dot);
    const float c = cta_sum(dot, slots, turn) * p.inv_c;
    for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
      const float d = fmaf(rstd, fmaf(-n_at(i), c, g_at(i)), ds ? load_param<Ts>(ds, i) : 0.f);
      static_cast<Tx*>(p.dx)[row * p.C + i] = store_param<Tx>(d);
      if constexpr (!std::is_same<Tx, Ts>::value)
        if (p.dsum_out) static_cast<Ts*>(p.dsum_out)[row * p.C + i] = store_param<Ts>(d);
    }
  }
  if (p.part == nullptr) return;
  // (a second look at the CTA's own rows, one channel per thread)
  for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
    float t = 0.f;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
      float s = load_param<Ts>(static_cast<const Ts*>(p.sum) + row * p.s_stride, i);
      if (p.addend) s += load_param<Tx>(static_cast<const Tx*>(p.addend) + row * p.a_stride, i);
      t = fmaf(load_param<Tx>(static_cast<const Tx*>(p.dy) + row * p.dy_stride, i), s * p.rstd[row], t);
    }
    p.part[(long long)blockIdx.x * p.C + i] = t;
  }
}

// One warp-wide column block of 32 channels per CTA; the rows are dealt out to its warps, whose sums are added in order.
constexpr int kSumWarps = 16;
__global__ void __launch_bounds__(32 * kSumWarps) column_sums_kernel(const ColumnSums p) {
  __shared__ float share[kSumWarps][32];
  const int per_set = (p.C + 31) / 32, set = (int)blockIdx.x / per_set;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = ((int)blockIdx.x - set * per_set) * 32 + lane;
  const float* part = p.part[set];
  const int rows = p.rows[set];
  grid_dep_wait();
  float t = 0.f;
  if (c < p.C) {
#pragma unroll 4
    for (int r = warp; r < rows; r += kSumWarps) t += part[(long long)r * p.C + c];
  }
  share[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && c < p.C) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < kSumWarps; ++i) t += share[i][lane];
    store_param_at(p.out[set], p.dtype, c, t);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
struct RmsGeom {
  int ve, v, lanes, threads;  // lanes: per row, 0 = one CTA per row; ve = 0: the kernels for rows of any length
};

RmsGeom rms_geometry(int64_t C, int dtype, bool aligned) {
  const int full = dtype == GNB200_F32 ? 4 : 8;
  RmsGeom g = {};
  g.ve = aligned && C % full == 0 ? full : 1;
  const int64_t nvec = C / g.ve;
  if (g.ve > 1 && nvec <= 32 * 4) {
    g.lanes = 1;
    while (g.lanes < 32 && g.lanes < nvec) g.lanes *= 2;
    g.v = nvec <= g.lanes ? 1 : nvec <= 2 * g.lanes ? 2 : 4;
    g.threads = kWarpThreads;
    return g;
  }
  const int most = 32 / g.ve;  // vectors a thread
  int v = g.ve == 1 ? 4 : 2;
  while (v < most && nvec > (int64_t)v * kMostThreads) v = g.ve == 1 ? (v == 4 ? 16 : 32) : 2 * v;
  if (nvec > (int64_t)v * kMostThreads) return RmsGeom{0, 0, 0, kMostThreads};
  g.v = v;
  g.threads = (int)((nvec + v - 1) / v + 31) / 32 * 32;
  return g;
}

// The CTAs of a call: no more than are resident at once, no more than there are rows
cudaError_t rms_grid(const void* kernel, const RmsGeom& g, int64_t rows, unsigned* grid) {
  long long most = 0;
  const cudaError_t err = resident_ctas(kernel, g.threads, &most);
  if (err != cudaSuccess) return err;
  const int64_t per_cta = g.lanes ? kWarpThreads / g.lanes : 1;
  const int64_t need = (rows + per_cta - 1) / per_cta;
  *grid = (unsigned)(need < most ? need : most);
  return cudaSuccess;
}

// calls f with the types of a call: x's, the sum's
template <typename F>
cudaError_t with_types(int dtype, int sum_dtype, F&& f) {
  if (dtype == GNB200_F32) return f(float(), float());
  if (dtype == GNB200_F16) return sum_dtype == GNB200_F32 ? f(__half(), float()) : f(__half(), __half());
  return sum_dtype == GNB200_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
}
template <int N>
using Int = std::integral_constant<int, N>;
// ... and with the geometry's numbers: elements a vector, vectors a thread, one group of lanes per row?
template <int FULL, typename F>
cudaError_t with_geometry(const RmsGeom& g, F&& f) {
  if (g.ve == 1) {
    if (g.v == 4) return f(Int<1>(), Int<4>(), std::false_type());
    if (g.v == 16) return f(Int<1>(), Int<16>(), std::false_type());
    return f(Int<1>(), Int<32>(), std::false_type());
  }
  if (g.lanes) {
    if (g.v == 1) return f(Int<FULL>(), Int<1>(), std::true_type());
    if (g.v == 2) return f(Int<FULL>(), Int<2>(), std::true_type());
    return f(Int<FULL>(), Int<4>(), std::true_type());
  }
  if (g.v == 2) return f(Int<FULL>(), Int<2>(), std::false_type());
  if constexpr (FULL == 4) {
    if (g.v == 8) return f(Int<FULL>(), Int<8>(), std::false_type());
  }
  return f(Int<FULL>(), Int<4>(), std::false_type());
}

template <typename Call>
cudaError_t launch_rows(void (*kernel)(Call), const RmsGeom& g, unsigned grid, const Call& p, cudaStream_t stream) {
  kernel<<<grid, g.threads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <bool Q>
cudaError_t launch_rms_fwd(RmsFwd p, int dtype, int sum_dtype, bool aligned, cudaStream_t stream) {
  const RmsGeom g = rms_geometry(p.C, dtype, aligned);
  p.lanes = g.lanes;
  return with_types(dtype, sum_dtype, [&](auto tx, auto ts) {
    using Tx = decltype(tx);
    using Ts = decltype(ts);
    auto go = [&](void (*kernel)(const RmsFwd)) {
      unsigned grid = 0;
      const cudaError_t err = rms_grid((const void*)kernel, g, p.rows, &grid);
      return err != cudaSuccess ? err : launch_rows(kernel, g, grid, p, stream);
    };
    if (g.ve == 0) return go(&rms_fwd_any_kernel<Tx, Ts, Q>);
    return with_geometry<16 / (int)sizeof(Tx)>(g, [&](auto ve, auto v, auto warp) {
      return go(&rms_fwd_kernel<Tx, Ts, decltype(ve)::value, decltype(v)::value, decltype(warp)::value, Q>);
    });
  });
}

// `grid_only`: the number of CTAs, that is of rows of partial sums, is all that is wanted
cudaError_t launch_rms_bwd(RmsBwd p, int dtype, int sum_dtype, bool aligned, cudaStream_t stream, unsigned* grid, bool grid_only) {
  const RmsGeom g = rms_geometry(p.C, dtype, aligned);
  p.lanes = g.lanes;
  return with_types(dtype, sum_dtype, [&](auto tx, auto ts) {
    using Tx = decltype(tx);
    using Ts = decltype(ts);
    auto go = [&](void (*kernel)(const RmsBwd)) {
      const cudaError_t err = rms_grid((const void*)kernel, g, p.rows, grid);
      if (g.ve == 0) *grid = std::min(*grid, (unsigned)std::max(1, (1 << 24) / p.C));  // 64 MB of partial sums at most, or one row
      return err != cudaSuccess || grid_only ? err : launch_rows(kernel, g, *grid, p, stream);
    };
    if (g.ve == 0) return go(&rms_bwd_any_kernel<Tx, Ts>);
    return with_geometry<16 / (int)sizeof(Tx)>(g, [&](auto ve, auto v, auto warp) {
      return go(&rms_bwd_kernel<Tx, Ts, decltype(ve)::value, decltype(v)::value, decltype(warp)::value>);
    });
  });
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool dtype_ok(int d) { return d == GNB200_F32 || d == GNB200_F16 || d == GNB200_BF16; }

int check_rows(const char* name, int64_t rows, int64_t C, int dtype, int sum_dtype, int w_dtype) {
  if (!dtype_ok(dtype) || !dtype_ok(sum_dtype) || !dtype_ok(w_dtype))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if ((sum_dtype != dtype && sum_dtype != GNB200_F32) || (w_dtype != dtype && w_dtype != GNB200_F32))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: the residual and the weight have the type of x or float32", name);
  if (rows < 0 || C < 1)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: rows must not be negative and channels be positive (got %lld, %lld)", name,
                        (long long)rows, (long long)C);
  if (C > (1 << 30))
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: rows of more than 2^30 channels are not supported (got %lld)", name, (long long)C);
  return GNB200_OK;
}
int launched(const char* name, cudaError_t err) {
  if (err == cudaSuccess) return GNB200_OK;
  return report_error(GNB200_ERR_CUDA, "%s: CUDA error: %s", name, cudaGetErrorString(err));
}

}  // namespace

cudaError_t launch_column_sums(const ColumnSums& p, int sets, cudaStream_t stream, bool chained) {
  return launch_chained(&column_sums_kernel, (unsigned)((p.C + 31) / 32 * sets), dim3(32 * kSumWarps), 0, stream, chained && chain_enabled(), p);
}

}  // namespace gnb200

using namespace gnb200;

extern "C" {

static int rms_forward(const char* name, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                       int64_t rows, int64_t C, double eps, double offset, int dtype, int residual_dtype, int weight_dtype, void* y,
                       void* sum, float* rstd, bool codes, int block, int format, float* scale, void* stream) {
  if (!residual) residual_dtype = dtype;
  if (!weight) weight_dtype = dtype;
  if (int rc = check_rows(name, rows, C, dtype, residual_dtype, weight_dtype)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!x || !y || (residual && !sum) || (codes && !scale))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (codes && block != 0 && block != 32 && block != 64 && block != 128)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: block is 0 (one scale per row), 32, 64 or 128 channels (got %d)", name, block);
  if (codes && format != GNB200_E4M3 && format != GNB200_INT8)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown format code %d (0=e4m3, 1=int8)", name, format);
  RmsFwd p = {};
  p.x = x, p.residual = residual, p.weight = weight, p.y = y, p.sum = sum, p.rstd = rstd, p.scale = scale;
  p.rows = rows, p.x_stride = x_stride, p.r_stride = residual_stride;
  p.C = (int)C, p.w_dtype = weight_dtype, p.block = block, p.blocks = block ? (int)((C + block - 1) / block) : 1, p.format = format;
  p.eps = (float)eps, p.offset = (float)offset, p.inv_c = (float)(1.0 / (double)C);
  const int full = dtype == GNB200_F32 ? 4 : 8;
  const bool aligned = on16(x) && on16(residual) && on16(y) && on16(sum) && x_stride % full == 0 && (!residual || residual_stride % full == 0);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launched(name, codes ? launch_rms_fwd<true>(p, dtype, residual_dtype, aligned, s)
                              : launch_rms_fwd<false>(p, dtype, residual_dtype, aligned, s));
}

int gnb200_rms_fwd(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows,
                   int64_t C, double eps, double offset, int dtype, int residual_dtype, int weight_dtype, void* y, void* sum, float* rstd,
                   void* stream) {
  return rms_forward("gnb200_rms_fwd", x, x_stride, residual, residual_stride, weight, rows, C, eps, offset, dtype, residual_dtype,
                     weight_dtype, y, sum, rstd, false, 0, 0, nullptr, stream);
}

int gnb200_rms_fwd_8bit(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows,
                        int64_t C, double eps, double offset, int dtype, int residual_dtype, int weight_dtype, int block, int format,
                        void* q, float* scale, void* sum, void* stream) {
  return rms_forward("gnb200_rms_fwd_8bit", x, x_stride, residual, residual_stride, weight, rows, C, eps, offset, dtype, residual_dtype,
                     weight_dtype, q, sum, nullptr, true, block, format, scale, stream);
}

size_t gnb200_rms_bwd_workspace_bytes(int64_t rows, int64_t C, int dtype, int sum_dtype) {
  if (check_rows("gnb200_rms_bwd_workspace_bytes", rows, C, dtype, sum_dtype, dtype) != GNB200_OK || rows == 0) return 0;
  RmsBwd p = {};
  p.rows = rows, p.C = (int)C;
  size_t most = 0;
  for (int aligned = 0; aligned < 2; ++aligned) {  // whichever kernel the pointers will ask for
    unsigned grid = 0;
    if (launch_rms_bwd(p, dtype, sum_dtype, aligned != 0, nullptr, &grid, true) != cudaSuccess) return 0;
    const size_t need = (size_t)grid * (size_t)C * sizeof(float);
    most = need > most ? need : most;
  }
  return most;
}

int gnb200_rms_bwd(const void* dy, int64_t dy_stride, const void* dsum, int64_t dsum_stride, const void* sum, int64_t sum_stride,
                   const void* addend, int64_t addend_stride, const void* weight, const float* rstd, int64_t rows, int64_t C, double offset, int dtype, int sum_dtype,
                   int weight_dtype, void* dx, void* dsum_out, void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "gnb200_rms_bwd";
  if (!weight) weight_dtype = dtype;
  if (int rc = check_rows(name, rows, C, dtype, sum_dtype, weight_dtype)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dweight && !weight) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: a gradient of the weight without a weight", name);
  if (rows == 0) {
    if (!dweight) return GNB200_OK;
    return launched(name, cudaMemsetAsync(dweight, 0, (size_t)C * (weight_dtype == GNB200_F32 ? 4 : 2), s));
  }
  if (!dy || !sum || !rstd || !dx) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (dsum_out && sum_dtype == dtype)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: dsum_out is for a sum of another type than dy", name);
  RmsBwd p = {};
  p.dy = dy, p.dsum = dsum, p.sum = sum, p.addend = addend, p.weight = weight, p.rstd = rstd, p.dx = dx, p.dsum_out = dsum_out;
  p.rows = rows, p.dy_stride = dy_stride, p.ds_stride = dsum_stride, p.s_stride = sum_stride, p.a_stride = addend_stride;
  p.C = (int)C, p.w_dtype = weight_dtype, p.offset = (float)offset, p.inv_c = (float)(1.0 / (double)C);
  const int full = dtype == GNB200_F32 ? 4 : 8;
  const bool aligned = on16(dy) && on16(dsum) && on16(sum) && on16(addend) && on16(dx) && on16(dsum_out) &&
                       dy_stride % full == 0 && sum_stride % full == 0 && (!dsum || dsum_stride % full == 0) &&
                       (!addend || addend_stride % full == 0);
  unsigned grid = 0;
  if (dweight) {
    cudaError_t err = launch_rms_bwd(p, dtype, sum_dtype, aligned, s, &grid, true);
    if (err != cudaSuccess) return launched(name, err);
    const size_t need = (size_t)grid * (size_t)C * sizeof(float);
    if (!workspace || workspace_bytes < need)
      return report_error(GNB200_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu are needed", name, workspace ? workspace_bytes : (size_t)0, need);
    p.part = static_cast<float*>(workspace);
  }
  cudaError_t err = launch_rms_bwd(p, dtype, sum_dtype, aligned, s, &grid, false);
  if (err == cudaSuccess && dweight) err = launch_column_sums(ColumnSums{{p.part}, {dweight}, {(int)grid}, (int)C, weight_dtype}, 1, s, true);
  return launched(name, err);
}

}  // extern "C"
