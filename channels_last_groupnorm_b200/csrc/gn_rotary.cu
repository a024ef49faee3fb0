// Rotary positions with several axes (time, height, width, ...) on queries and keys, with or without the
// root-mean-square norm of each head in front: forward and backward.
//
//   n = x * rstd * (offset + w), rstd = 1 / sqrt(mean over the head of x^2 + eps)      (n = x without a weight)
//   pair i of a head turns by angle_i = position[axis of i] * inv_freq[i]; pairs beyond the rotated ones stay:
//   (a, b) -> (a cos - b sin, b cos + a sin)     pair i: channels (i, i + pairs), or (2 i, 2 i + 1) where interleaved
// Backward: the gradient turns by -angle, g; then, with n without its weight,
//   dx = rstd * (g (offset + w) - n * mean(g (offset + w) n)),  dw = sum over tokens and heads of g * n.
//
// Both tensors are read and written once.  A warp takes a token's heads, or a share of them: it computes the token's
// angles once, in its own piece of shared memory, and 32 / lanes heads at a time pass through registers, each in `lanes` lanes.  A
// lane holds both channels of its pairs (two vectors), so the rotation exchanges nothing and the norm one butterfly.  The
// product of position and frequency is formed and reduced to a fraction of a turn in fp64, so that the angle of a position of a
// million is as exact as that of the first; per token that is a few instructions beside hundreds of channels.
#include <algorithm>

#include "../../include/gnb200.h"
#include "gn_kernels.h"
#include "gn_tokens.cuh"

namespace gnb200 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMostHead = 512;
constexpr int kMostAxes = 8;

struct Rotary {
  const void *in[2], *x[2], *weight[2];  // q, k: in = the tensor to turn (backward: the gradient); x: backward of the norm, what the forward got
  void* out[2];
  float* part[2];  // backward of the norm: one row of D floats per CTA
  long long in_stride[2][3], x_stride[2][3];  // batch, token, head; out is contiguous
  int heads[2], per_task[2], tasks_per_token[2];
  unsigned ctas[2];
  long long tokens;
  int S, D, pairs, lanes;
  const void* positions;
  long long pos_stride[3];  // batch, token, axis
  int pos_type;
  const float* inv_freq;
  int axes, last[kMostAxes];  // last[a]: one past the pairs of axis a
  int w_dtype[2];
  float eps, offset, inv_d, sign;
};

// cos and sin of this token's angles, into the warp's shared memory
__device__ __forceinline__ void token_angles(const Rotary& p, long long b, long long s, float2* out) {
  const long long at = b * p.pos_stride[0] + s * p.pos_stride[1];
  for (int i = threadIdx.x & 31; i < p.pairs; i += 32) {
    int axis = 0;
    while (axis + 1 < p.axes && i >= p.last[axis]) ++axis;
    const long long from = at + axis * p.pos_stride[2];
    double position;
    if (p.pos_type == GNB200_POS_I64)
      position = (double)static_cast<const long long*>(p.positions)[from];
    else if (p.pos_type == GNB200_POS_I32)
      position = (double)static_cast<const int*>(p.positions)[from];
    else
      position = (double)static_cast<const float*>(p.positions)[from];
    double turns = position * (double)p.inv_freq[i] * 0.15915494309189535;  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif((float)(2.0 * turns), &sn, &cs);
    out[i] = make_float2(cs, p.sign * sn);
  }
  __syncwarp();
}

// Where a lane's slot of two vectors stands in the head.  Slots 0 .. pairs / VE - 1 are turned, the others pass.  WHOLE: the head is
// turned from end to end and every lane has one slot.
template <int VE, bool INTER, bool WHOLE>
struct Slot {
  int a, b;
  bool has_a, has_b, turns;
  __device__ __forceinline__ Slot(int s, int pairs, int D) {
    const int rotated = pairs / VE;
    turns = WHOLE || s < rotated;
    if (turns) {
      a = INTER ? 2 * s * VE : s * VE;
      b = INTER ? a + VE : pairs + s * VE;
    } else {
      a = 2 * pairs + 2 * (s - rotated) * VE;
      b = a + VE;
    }
    has_a = WHOLE || a < D;
    has_b = WHOLE || b < D;
  }
};

// (a, b) -> (a aa + b ab, b bb + a ba) for the pairs of f, the slot's two vectors
template <int VE, bool INTER>
__device__ __forceinline__ void turn(float (&f)[2 * VE], const float (&aa)[VE], const float (&ab)[VE], const float (&bb)[VE], const float (&ba)[VE]) {
  if constexpr (!INTER && VE % 2 == 0) {
#pragma unroll
    for (int e = 0; e < VE; e += 2) {
      float u0, u1, v0, v1;
      mul2(u0, u1, f[VE + e], f[VE + e + 1], ab[e], ab[e + 1]);
      mul2(v0, v1, f[e], f[e + 1], ba[e], ba[e + 1]);
      fma2(f[e], f[e + 1], f[e], f[e + 1], aa[e], aa[e + 1], u0, u1);
      fma2(f[VE + e], f[VE + e + 1], f[VE + e], f[VE + e + 1], bb[e], bb[e + 1], v0, v1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int i = INTER ? 2 * e : e, j = INTER ? 2 * e + 1 : VE + e;
      const float a = f[i], b = f[j];
      f[i] = fmaf(a, aa[e], b * ab[e]);
      f[j] = fmaf(b, bb[e], a * ba[e]);
    }
  }
}

template <typename T, int VE>
__device__ __forceinline__ void unpack_two(const Pack<T, VE>& a, const Pack<T, VE>& b, float (&f)[2 * VE]) {
  float g[VE];
  unpack<T, VE>(a, g);
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = g[e];
  unpack<T, VE>(b, g);
#pragma unroll
  for (int e = 0; e < VE; ++e) f[VE + e] = g[e];
}

// SLOTS: slots a lane.  BACK: backward of the norm (a backward without one is a forward with the angles' sign changed).
template <typename T, int VE, int SLOTS, bool WHOLE, bool INTER, bool NORM, bool BACK>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary p) {
  __shared__ float2 angles[kWarps][kMostHead / 2];
  using Where = Slot<VE, INTER, WHOLE>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane & (p.lanes - 1), group = lane / p.lanes, groups = 32 / p.lanes;
  const int t = blockIdx.x >= p.ctas[0];  // q or k
  const unsigned cta = blockIdx.x - (t ? p.ctas[0] : 0);
  if constexpr (BACK) grid_dep_launch_dependents();
  float w[NORM ? SLOTS : 1][2 * VE], dw[BACK ? SLOTS : 1][2 * VE];
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const Where slot(l + j * p.lanes, p.pairs, p.D);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        w[j][e] = slot.has_a ? p.offset + param_at(p.weight[t], p.w_dtype[t], slot.a + e, 1.f) : 0.f;
        w[j][VE + e] = slot.has_b ? p.offset + param_at(p.weight[t], p.w_dtype[t], slot.b + e, 1.f) : 0.f;
        if constexpr (BACK) dw[j][e] = dw[j][VE + e] = 0.f;
      }
    }
  }
  const T* const tensor = static_cast<const T*>(p.in[t]);
  const T* const xtensor = static_cast<const T*>(p.x[t]);
  const long long head_stride = p.in_stride[t][2], xhead_stride = BACK ? p.x_stride[t][2] : 0;
  const int per_token = p.tasks_per_token[t], per_task = p.per_task[t], heads = p.heads[t];
  const long long tasks = p.tokens * per_token;
  for (long long task = (long long)cta * kWarps + warp; task < tasks; task += (long long)p.ctas[t] * kWarps) {
    const long long token = per_token == 1 ? task : task / per_token, b = p.S == p.tokens ? 0 : token / p.S, s = token - b * p.S;
    const int from = (int)(task - token * per_token) * per_task, to = min(from + per_task, heads);
    const T* in = tensor + b * p.in_stride[t][0] + s * p.in_stride[t][1];
    const T* xs = BACK ? xtensor + b * p.x_stride[t][0] + s * p.x_stride[t][1] : nullptr;
    // the heads of one turn of the warp; a group beyond the last head takes the last one again and stores nothing
    Pack<T, VE> va[SLOTS], vb[SLOTS], xa[BACK ? SLOTS : 1], xb[BACK ? SLOTS : 1];
    auto ask = [&](int base) {
      const int head = min(base + group, to - 1);
      const T* row = in + head * head_stride;
      const T* xrow = xs + head * xhead_stride;
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const Where slot(l + j * p.lanes, p.pairs, p.D);
        if (slot.has_a) va[j] = load_vec<T, VE>(row + slot.a);
        if (slot.has_b) vb[j] = load_vec<T, VE>(row + slot.b);
        if constexpr (BACK) {
          if (slot.has_a) xa[j] = load_vec<T, VE>(xrow + slot.a);
          if (slot.has_b) xb[j] = load_vec<T, VE>(xrow + slot.b);
        }
      }
    };
    ask(from);
    __syncwarp();
    token_angles(p, b, s, angles[warp]);
    // The rotation's coefficients; the norm's weights are part of them forward, where nothing needs the rotated values without.
    float aa[SLOTS][VE], ab[SLOTS][VE], bb[SLOTS][VE], ba[SLOTS][VE];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const int slot = l + j * p.lanes;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float2 v = WHOLE || (slot + 1) * VE <= p.pairs ? angles[warp][slot * VE + e] : make_float2(1.f, 0.f);
        if constexpr (NORM && !BACK) {
          const int i = INTER ? 2 * e : e, k = INTER ? 2 * e + 1 : VE + e;
          aa[j][e] = v.x * w[j][i], ab[j][e] = -v.y * w[j][k], bb[j][e] = v.x * w[j][k], ba[j][e] = v.y * w[j][i];
        } else {
          aa[j][e] = bb[j][e] = v.x, ab[j][e] = -v.y, ba[j][e] = v.y;
        }
      }
    }
    T* out = static_cast<T*>(p.out[t]) + token * heads * p.D;
    for (int base = from; base < to; base += groups) {
      const int head = base + group;
      const bool live = head < to;
      float f[SLOTS][2 * VE], n[BACK ? SLOTS : 1][2 * VE];
      float sq[2] = {0.f, 0.f}, dot[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const Where slot(l + j * p.lanes, p.pairs, p.D);
        unpack_two<T, VE>(va[j], vb[j], f[j]);
        if constexpr (BACK) unpack_two<T, VE>(xa[j], xb[j], n[j]);
        if constexpr (!WHOLE) {
#pragma unroll
          for (int e = 0; e < 2 * VE; ++e) {
            if (!(e < VE ? slot.has_a : slot.has_b)) {
              f[j][e] = 0.f;
              if constexpr (BACK) n[j][e] = 0.f;
            }
          }
        }
        if constexpr (NORM && !BACK) dot_each(sq, f[j], f[j]);
        if (slot.turns) {
          turn<VE, INTER>(f[j], aa[j], ab[j], bb[j], ba[j]);
        } else if constexpr (NORM && !BACK) {
          mul_each(f[j], w[j]);
        }
        if constexpr (BACK) dot_each(sq, n[j], n[j]);
      }
      if (base + groups < to) ask(base + groups);
      if constexpr (NORM) {
        const float rstd = __frsqrt_rn(fmaf(lanes_sum(sq[0] + sq[1], p.lanes), p.inv_d, p.eps));
        if constexpr (BACK) {
#pragma unroll
          for (int j = 0; j < SLOTS; ++j) {
            scale_each(n[j], rstd);
            if (live) fma_each(dw[j], f[j], n[j]);
            mul_each(f[j], w[j]);
            dot_each(dot, f[j], n[j]);
          }
          const float c = -lanes_sum(dot[0] + dot[1], p.lanes) * p.inv_d;
#pragma unroll
          for (int j = 0; j < SLOTS; ++j) axpy_each(f[j], n[j], c);
        }
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) scale_each(f[j], rstd);
      }
      if (live) {
        T* row = out + (long long)head * p.D;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
          const Where slot(l + j * p.lanes, p.pairs, p.D);
          float g[VE];
          if (slot.has_a) {
#pragma unroll
            for (int e = 0; e < VE; ++e) g[e] = f[j][e];
            store_vec<T, VE>(row + slot.a, pack<T, VE>(g));
          }
          if (slot.has_b) {
#pragma unroll
            for (int e = 0; e < VE; ++e) g[e] = f[j][VE + e];
            store_vec<T, VE>(row + slot.b, pack<T, VE>(g));
          }
        }
      }
    }
  }
  if constexpr (BACK) {
    // the groups of a warp and the warps of the CTA hold the same channels: added in a fixed order
    float(*share)[kMostHead] = reinterpret_cast<float(*)[kMostHead]>(&angles[0][0]);  // a warp's angles are as long as a head
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const Where slot(l + j * p.lanes, p.pairs, p.D);
#pragma unroll
      for (int e = 0; e < 2 * VE; ++e) {
        float v = dw[j][e];
        for (int delta = 16; delta >= p.lanes; delta >>= 1) v += __shfl_xor_sync(0xffffffffu, v, delta);
        if (group == 0 && (e < VE ? slot.has_a : slot.has_b)) share[warp][(e < VE ? slot.a + e : slot.b + e - VE)] = v;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.D; i += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v += share[k][i];
      p.part[t][(long long)cta * p.D + i] = v;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
struct RotaryGeom {
  int ve, slots, lanes;
  bool whole;
};
// ve: the widest vectors that the head, the pairs and (`widest`, by alignment) the tensors allow
RotaryGeom rotary_geometry(int D, int pairs, int widest, int widest_full) {
  RotaryGeom g = {widest, 1, 1, false};
  while (g.ve > 1 && (D % g.ve || pairs % g.ve)) g.ve = g.ve == 8 ? 4 : 1;
  const int count = pairs / g.ve + ((D - 2 * pairs) / g.ve + 1) / 2;
  while (g.lanes < 32 && g.lanes < count) g.lanes *= 2;
  while (g.slots * g.lanes < count) g.slots *= 2;
  if (g.ve == 1) g.slots = g.slots <= 2 ? 2 : 8;
  g.whole = 2 * pairs == D && g.ve == widest_full && g.slots == 1 && pairs == g.ve * g.lanes;
  return g;
}

template <int N>
using Int = std::integral_constant<int, N>;
template <typename T, typename F>
cudaError_t with_rotary_geometry(const RotaryGeom& g, F&& f) {
  if (g.whole) return f(Int<16 / (int)sizeof(T)>(), Int<1>(), std::true_type());
  if constexpr (sizeof(T) == 2) {
    if (g.ve == 8) return f(Int<8>(), Int<1>(), std::false_type());
  }
  if (g.ve == 4) return g.slots == 1 ? f(Int<4>(), Int<1>(), std::false_type()) : f(Int<4>(), Int<2>(), std::false_type());
  return g.slots == 2 ? f(Int<1>(), Int<2>(), std::false_type()) : f(Int<1>(), Int<8>(), std::false_type());
}

// How the tokens' heads are dealt out: warps take whole tokens where there are enough of them, else shares of a token's heads.
cudaError_t rotary_split(const void* kernel, const RotaryGeom& g, Rotary& p) {
  Residency r;
  const cudaError_t err = residency(kernel, kThreads, 0, &r);
  if (err != cudaSuccess) return err;
  const long long most = (long long)r.per_sm * r.sms;
  const int groups = 32 / g.lanes, all = p.heads[0] + p.heads[1];
  long long want[2] = {0, 0};
  for (int t = 0; t < 2; ++t) {
    if (!p.heads[t]) continue;
    const int turns = (p.heads[t] + groups - 1) / groups;  // of a warp, for a token
    const long long share = std::max(1LL, most * kWarps * p.heads[t] / all / std::max(1LL, p.tokens));
    const int tasks = (int)std::min<long long>(turns, share);
    p.per_task[t] = (turns + tasks - 1) / tasks * groups;
    p.tasks_per_token[t] = (p.heads[t] + p.per_task[t] - 1) / p.per_task[t];
    want[t] = (p.tokens * p.tasks_per_token[t] + kWarps - 1) / kWarps;
  }
  if (want[0] + want[1] > most) {
    for (int t = 0; t < 2; ++t)
      if (p.heads[t]) want[t] = std::max(1LL, std::min(want[t], most * p.heads[t] / all));
  }
  p.ctas[0] = (unsigned)want[0];
  p.ctas[1] = (unsigned)want[1];
  return cudaSuccess;
}

// plan_only: p.ctas is all that is wanted
cudaError_t launch_rotary(Rotary& p, int dtype, int widest, bool inter, bool norm, bool back, bool plan_only, cudaStream_t stream) {
  const RotaryGeom g = rotary_geometry(p.D, p.pairs, widest, dtype == GNB200_F32 ? 4 : 8);
  p.lanes = g.lanes;
  auto go = [&](void (*kernel)(const Rotary)) {
    const cudaError_t err = rotary_split((const void*)kernel, g, p);
    if (err != cudaSuccess || plan_only) return err;
    kernel<<<p.ctas[0] + p.ctas[1], kThreads, 0, stream>>>(p);
    return cudaGetLastError();
  };
  auto typed = [&](auto type) {
    using T = decltype(type);
    return with_rotary_geometry<T>(g, [&](auto ve, auto slots, auto whole) {
      constexpr int VE = decltype(ve)::value, S = decltype(slots)::value;
      constexpr bool W = decltype(whole)::value;
      if (inter) {
        if (back) return go(&rotary_kernel<T, VE, S, W, true, true, true>);
        return norm ? go(&rotary_kernel<T, VE, S, W, true, true, false>) : go(&rotary_kernel<T, VE, S, W, true, false, false>);
      }
      if (back) return go(&rotary_kernel<T, VE, S, W, false, true, true>);
      return norm ? go(&rotary_kernel<T, VE, S, W, false, true, false>) : go(&rotary_kernel<T, VE, S, W, false, false, false>);
    });
  };
  if (dtype == GNB200_F32) return typed(float());
  if (dtype == GNB200_F16) return typed(__half());
  return typed(__nv_bfloat16());
}

// widest vector, in elements, that a tensor's address and strides allow
int widest_of(const void* p, const int64_t* strides, int size, int ve) {
  for (; ve > 1; ve = ve == 8 ? 4 : 1) {
    bool ok = reinterpret_cast<uintptr_t>(p) % (ve * size) == 0;
    for (int i = 0; strides && i < 3; ++i) ok = ok && strides[i] % ve == 0;
    if (ok) return ve;
  }
  return 1;
}

int check_rotary(const char* name, const gnb200_rotary_args* a) {
  if (!a) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  const bool types = (a->dtype == GNB200_F32 || a->dtype == GNB200_F16 || a->dtype == GNB200_BF16) &&
                     (!a->q_weight || a->q_weight_dtype == a->dtype || a->q_weight_dtype == GNB200_F32) &&
                     (!a->k_weight || a->k_weight_dtype == a->dtype || a->k_weight_dtype == GNB200_F32);
  if (!types) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: dtype codes are 0=f32, 1=f16, 2=bf16; weights have the tensors' or 0", name);
  if (a->pos_type != GNB200_POS_I32 && a->pos_type != GNB200_POS_I64 && a->pos_type != GNB200_POS_F32)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown position type %d", name, a->pos_type);
  if (a->batch < 0 || a->tokens < 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads + a->k_heads < 1 || a->head_dim < 2)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: sizes must not be negative, heads and channels be there", name);
  if (a->head_dim > kMostHead)
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: heads of more than %d channels are not supported (got %lld)", name, kMostHead,
                        (long long)a->head_dim);
  if (a->q_heads > (1 << 20) || a->k_heads > (1 << 20) || a->batch > (1LL << 31) || a->tokens >= (1LL << 31))
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: more than 2^20 heads or 2^31 tokens", name);
  if (a->axes < 1 || a->axes > kMostAxes)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: 1 to %d axes (got %d)", name, kMostAxes, a->axes);
  int64_t pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0 || a->sections[i] > kMostHead)
      return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: section %d of %d pairs", name, i, a->sections[i]);
    pairs += a->sections[i];
  }
  if (pairs < 1 || 2 * pairs > a->head_dim)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: %lld pairs do not fit heads of %lld channels", name, (long long)pairs,
                        (long long)a->head_dim);
  return GNB200_OK;
}

// The part of the call that forward and backward share; false where there is nothing to do.
bool fill(const gnb200_rotary_args* a, Rotary& p) {
  if (a->batch == 0 || a->tokens == 0) return false;
  p.tokens = a->batch * a->tokens;
  p.S = (int)a->tokens;
  p.D = (int)a->head_dim;
  p.heads[0] = (int)a->q_heads;
  p.heads[1] = (int)a->k_heads;
  p.axes = a->axes;
  for (int i = 0; i < a->axes; ++i) p.last[i] = p.pairs += a->sections[i];
  p.positions = a->positions;
  p.pos_type = a->pos_type;
  for (int i = 0; i < 3; ++i) p.pos_stride[i] = a->pos_stride[i];
  p.inv_freq = a->inv_freq;
  p.weight[0] = a->q_weight, p.weight[1] = a->k_weight;
  p.w_dtype[0] = a->q_weight_dtype, p.w_dtype[1] = a->k_weight_dtype;
  p.eps = (float)a->eps, p.offset = (float)a->offset, p.inv_d = (float)(1.0 / (double)p.D);
  p.sign = 1.f;
  return true;
}
int launched(const char* name, cudaError_t err) {
  if (err == cudaSuccess) return GNB200_OK;
  return report_error(GNB200_ERR_CUDA, "%s: CUDA error: %s", name, cudaGetErrorString(err));
}

}  // namespace
}  // namespace gnb200

using namespace gnb200;

extern "C" {

int gnb200_rotary_fwd(const gnb200_rotary_args* a, const void* q, const int64_t* q_stride, const void* k, const int64_t* k_stride,
                      void* q_out, void* k_out, void* stream) {
  const char* name = "gnb200_rotary_fwd";
  if (int rc = check_rotary(name, a)) return rc;
  Rotary p = {};
  if (!fill(a, p)) return GNB200_OK;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* strides[2] = {q_stride, k_stride};
  if (!a->positions || !a->inv_freq) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  const int size = a->dtype == GNB200_F32 ? 4 : 2;
  // the tensors with a norm and those without are two launches where one has a weight and the other none
  bool with_norm[2] = {a->q_weight != nullptr, a->k_weight != nullptr};
  for (int t = 0; t < 2; ++t) {
    if (!p.heads[t]) continue;
    if (!in[t] || !out[t] || !strides[t]) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    p.in[t] = in[t], p.out[t] = out[t];
    for (int i = 0; i < 3; ++i) p.in_stride[t][i] = strides[t][i];
  }
  const bool together = !p.heads[0] || !p.heads[1] || with_norm[0] == with_norm[1];
  for (int first = 0; first < (together ? 1 : 2); ++first) {
    Rotary call = p;
    if (!together) call.heads[1 - first] = 0;
    int widest = 16 / size;
    for (int t = 0; t < 2; ++t)
      if (call.heads[t]) widest = std::min({widest, widest_of(in[t], strides[t], size, widest), widest_of(out[t], nullptr, size, widest)});
    const bool norm = call.heads[0] ? with_norm[0] : with_norm[1];
    if (int rc = launched(name, launch_rotary(call, a->dtype, widest, a->interleaved != 0, norm, false, false, static_cast<cudaStream_t>(stream))))
      return rc;
  }
  return GNB200_OK;
}

// every kernel that the call may take, by the tensors' alignment: the largest number of partial rows
size_t gnb200_rotary_bwd_workspace_bytes(const gnb200_rotary_args* a) {
  if (check_rotary("gnb200_rotary_bwd_workspace_bytes", a) != GNB200_OK || (!a->q_weight && !a->k_weight)) return 0;
  Rotary p = {};
  if (!fill(a, p)) return 0;
  size_t most = 0;
  for (int which = 1; which < 4; ++which) {  // q, k, both
    for (int widest = 16 / (a->dtype == GNB200_F32 ? 4 : 2); widest >= 1; widest = widest == 8 ? 4 : widest == 4 ? 1 : 0) {
      Rotary call = p;
      if (!(which & 1)) call.heads[0] = 0;
      if (!(which & 2)) call.heads[1] = 0;
      if (call.heads[0] + call.heads[1] == 0) continue;
      if (launch_rotary(call, a->dtype, widest, a->interleaved != 0, true, true, true, nullptr) != cudaSuccess) return 0;
      most = std::max(most, ((size_t)call.ctas[0] + call.ctas[1]) * (size_t)p.D * sizeof(float));
    }
  }
  return most;
}

int gnb200_rotary_bwd(const gnb200_rotary_args* a, const void* dq, const int64_t* dq_stride, const void* dk, const int64_t* dk_stride,
                      const void* q, const int64_t* q_stride, const void* k, const int64_t* k_stride, void* dq_out, void* dk_out,
                      void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "gnb200_rotary_bwd";
  if (int rc = check_rotary(name, a)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int size = a->dtype == GNB200_F32 ? 4 : 2;
  void* dweight[2] = {dq_weight, dk_weight};
  const void* weight[2] = {a->q_weight, a->k_weight};
  const int w_dtype[2] = {a->q_weight_dtype, a->k_weight_dtype};
  Rotary p = {};
  const bool some = fill(a, p);
  const int64_t heads[2] = {a->q_heads, a->k_heads};
  for (int t = 0; t < 2; ++t) {
    if (weight[t] && heads[t] && !dweight[t]) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    if (!some && weight[t] && heads[t])
      if (int rc = launched(name, cudaMemsetAsync(dweight[t], 0, (size_t)a->head_dim * (w_dtype[t] == GNB200_F32 ? 4 : 2), s))) return rc;
  }
  if (!some) return GNB200_OK;
  p.sign = -1.f;
  const void *in[2] = {dq, dk}, *x[2] = {q, k};
  void* out[2] = {dq_out, dk_out};
  const int64_t *in_stride[2] = {dq_stride, dk_stride}, *x_stride[2] = {q_stride, k_stride};
  if (!a->positions || !a->inv_freq) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  for (int t = 0; t < 2; ++t) {
    if (!p.heads[t]) continue;
    if (!in[t] || !in_stride[t] || !out[t] || (weight[t] && (!x[t] || !x_stride[t])))
      return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    p.in[t] = in[t], p.x[t] = x[t], p.out[t] = out[t];
    for (int i = 0; i < 3; ++i) {
      p.in_stride[t][i] = in_stride[t][i];
      if (weight[t]) p.x_stride[t][i] = x_stride[t][i];
    }
  }
  const bool norm[2] = {weight[0] != nullptr, weight[1] != nullptr};
  const bool together = !p.heads[0] || !p.heads[1] || norm[0] == norm[1];
  for (int first = 0; first < (together ? 1 : 2); ++first) {
    Rotary call = p;
    if (!together) call.heads[1 - first] = 0;
    const bool back = call.heads[0] ? norm[0] : norm[1];
    int widest = 16 / size;
    for (int t = 0; t < 2; ++t) {
      if (!call.heads[t]) continue;
      widest = std::min({widest, widest_of(in[t], in_stride[t], size, widest), widest_of(out[t], nullptr, size, widest)});
      if (back) widest = std::min(widest, widest_of(x[t], x_stride[t], size, widest));
    }
    const bool inter = a->interleaved != 0;
    if (back) {
      cudaError_t err = launch_rotary(call, a->dtype, widest, inter, true, true, true, s);
      if (err != cudaSuccess) return launched(name, err);
      const size_t need = ((size_t)call.ctas[0] + call.ctas[1]) * (size_t)p.D * sizeof(float);
      if (!workspace || workspace_bytes < need)
        return report_error(GNB200_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu are needed", name, workspace ? workspace_bytes : (size_t)0, need);
      call.part[0] = static_cast<float*>(workspace);
      call.part[1] = call.part[0] + (size_t)call.ctas[0] * p.D;
    }
    if (int rc = launched(name, launch_rotary(call, a->dtype, widest, inter, back, back, false, s))) return rc;
    if (!back) continue;
    ColumnSums sums[2] = {};
    int sets = 0, launches = 0;
    for (int t = 0; t < 2; ++t) {  // one launch, or two where the weights have different types
      if (!call.heads[t]) continue;
      if (sets && sums[0].dtype != w_dtype[t]) launches = 1, sets = 0;
      ColumnSums& c = sums[launches];
      c.part[sets] = call.part[t], c.out[sets] = dweight[t], c.rows[sets] = (int)call.ctas[t];
      c.C = p.D, c.dtype = w_dtype[t];
      ++sets;
    }
    if (launches) {
      if (int rc = launched(name, launch_column_sums(sums[0], 1, s, true))) return rc;
      if (int rc = launched(name, launch_column_sums(sums[1], 1, s, false))) return rc;
    } else if (int rc = launched(name, launch_column_sums(sums[0], sets, s, true))) {
      return rc;
    }
  }
  return GNB200_OK;
}

}  // extern "C"
