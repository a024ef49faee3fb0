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
// lane holds both channels of its pairs (two vectors), so the rotation exchanges nothing and the norm one butterfly (two in the backward, at
// once).  Angles are formed in turns from two floats, so that the angle of a position of ten million is as exact as that of the first.
//
// Bound by HBM with many heads: 16384 tokens of 32 + 32 heads of 128, bf16, with norm 87 us = 6.2 TB/s (94 % of a copy's rate), without 87 us,
// backward with norm (four tensors read, two written) 130 us = 6.2 TB/s.  With few heads by instructions: a token's angles, coefficients and
// addresses cost as much as four turns of the warp (2 x 4096 tokens of 20 + 20 heads of 64 with norm 17.7 us, 16384 of 4 + 4 of 128
// 24 us, 1.4 and 2.4 times their bytes' time).  A single token takes 3.2 us: launch, first load, one turn.
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
  int tokens, S, D, pairs, lanes;
  unsigned div_mul, div_shift;  // token / S for token < 2^31: (umulhi(token, mul) + token) >> shift
  const void* positions;
  long long pos_stride[3];  // batch, token, axis
  int pos_type;
  const float* inv_freq;
  int axes, last[kMostAxes];  // last[a]: one past the pairs of axis a
  int w_dtype[2];
  float eps, offset, inv_d, sign;
};

constexpr double kPerTurn = 0.15915494309189535;  // 1 / (2 pi)

// What a CTA knows of its pairs: inv_freq / (2 pi) as the sum of two floats, and the axis.
struct PairTable {
  float2 turns[kMostHead / 2];
  uint8_t axis[kMostHead / 2];
};
__device__ __forceinline__ void fill_pairs(const Rotary& p, PairTable& table) {
  for (int i = threadIdx.x; i < p.pairs; i += kThreads) {
    const double turns = (double)p.inv_freq[i] * kPerTurn;
    const float hi = (float)turns;
    table.turns[i] = make_float2(hi, (float)(turns - (double)hi));
    int axis = 0;
    while (axis + 1 < p.axes && i >= p.last[axis]) ++axis;
    table.axis[i] = (uint8_t)axis;
  }
}

// A lane's share of a token's positions: those of pairs lane and lane + 32 (asked for a token ahead; further ones as they are needed).
struct Positions {
  long long raw[2];
};
__device__ __forceinline__ long long position_at(const Rotary& p, long long at) {
  if (p.pos_type == GNB200_POS_I64) return static_cast<const long long*>(p.positions)[at];
  return static_cast<const int*>(p.positions)[at];  // (or the bits of a float)
}
__device__ __forceinline__ void ask_positions(const Rotary& p, const PairTable& table, int b, int s, Positions& out) {
  const long long at = p.pos_stride[0] * b + p.pos_stride[1] * s;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = (int)(threadIdx.x & 31) + 32 * k;
    if (i < p.pairs) out.raw[k] = position_at(p, at + table.axis[i] * p.pos_stride[2]);
  }
}

// cos and sin of pair i's angle.  It is formed in turns, whole ones dropped: position * hi in fp32, what its rounding lost (an fma gives it
// exactly) and position * lo.  That holds for positions that fp32 holds exactly; larger ones are multiplied in fp64.  fast: the hardware's
// sine and cosine, off by 2^-21 on the remaining half turns, where all results are rounded to 16 bits.
__device__ __forceinline__ float2 angle_of(const Rotary& p, const PairTable& table, int i, long long raw, bool fast) {
  const float2 freq = table.turns[i];
  const bool is_float = p.pos_type == GNB200_POS_F32;
  const float position = is_float ? __int_as_float((int)raw) : (float)(int)raw;
  const bool exact = is_float ? fabsf(position) < 16777216.f : (raw < 16777216 && raw > -16777216);
  float part;
  if (exact) {
    const float turns = position * freq.x;
    part = (turns - rintf(turns)) + fmaf(position, freq.y, fmaf(position, freq.x, -turns));
  } else {
    const double turns = (is_float ? (double)position : (double)raw) * ((double)p.inv_freq[i] * kPerTurn);
    part = (float)(turns - rint(turns));
  }
  float sn, cs;
  if (fast) {
    part -= rintf(part);  // (the two parts' sum may have passed half a turn)
    const float radians = part * 6.28318531f;
    sn = __sinf(radians);
    cs = __cosf(radians);
  } else {
    sincospif(2.f * part, &sn, &cs);
  }
  return make_float2(cs, p.sign * sn);
}

// cos and sin of a token's angles, into the warp's shared memory
__device__ __forceinline__ void token_angles(const Rotary& p, const PairTable& table, int b, int s, const Positions& known, bool fast, float2* out) {
  const int lane = threadIdx.x & 31;
  __syncwarp();  // (nobody reads the token before any more)
  if (lane < p.pairs) out[lane] = angle_of(p, table, lane, known.raw[0], fast);
  if (lane + 32 < p.pairs) out[lane + 32] = angle_of(p, table, lane + 32, known.raw[1], fast);
  if (p.pairs > 64) {
    const long long at = p.pos_stride[0] * b + p.pos_stride[1] * s;
    for (int i = lane + 64; i < p.pairs; i += 32) out[i] = angle_of(p, table, i, position_at(p, at + table.axis[i] * p.pos_stride[2]), fast);
  }
  __syncwarp();
}

// The heads ahead.  16-byte vectors travel to the warp's ring of stages in shared memory, one stage a turn of the warp, where a lane
// finds what it copied itself; shorter ones to registers, one turn ahead.
template <typename T, int VE>
constexpr bool kRing = sizeof(T) * VE == 16;
template <bool RING, int STAGES, int VECTORS>  // VECTORS: a lane's, of a turn
struct Ring {
  static constexpr int kStages = RING ? STAGES : 1;
  uint4 at[RING ? kWarps : 1][kStages][RING ? VECTORS : 1][RING ? 32 : 1];
};

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
      a = INTER && VE == 1 ? 2 * s : s * VE;
      b = INTER && VE == 1 ? 2 * s + 1 : pairs + s * VE;
    } else {
      a = 2 * pairs + 2 * (s - rotated) * VE;
      b = a + VE;
    }
    has_a = WHOLE || a < D;
    has_b = WHOLE || b < D;
  }
  // the pair that is turned by the slot's coefficient e; its channels are those of elements first(e) and second(e) of the slot
  __device__ __forceinline__ int pair(int e) const {
    if constexpr (!INTER) return a + e;
    if constexpr (VE == 1) return a / 2;
    return e < VE / 2 ? a / 2 + e : b / 2 + e - VE / 2;
  }
  static __device__ __forceinline__ constexpr int first(int e) { return INTER ? 2 * e : e; }
  static __device__ __forceinline__ constexpr int second(int e) { return INTER ? 2 * e + 1 : VE + e; }
  __device__ __forceinline__ int channel(int i) const { return i < VE ? a + i : b + i - VE; }
};

// a task's token, and its place
__device__ __forceinline__ int token_of(const Rotary& p, int task, int per_token, int& b, int& s) {
  const int token = per_token == 1 ? task : task / per_token;
  b = (int)((__umulhi((unsigned)token, p.div_mul) + (unsigned)token) >> p.div_shift);
  s = token - b * p.S;
  return token;
}
__device__ __forceinline__ long long place(const long long (&strides)[3], int b, int s, int head) {
  return strides[0] * b + strides[1] * s + strides[2] * head;
}
// Reciprocal root mean square.  The fast one is off by two units of fp32's last place, below what results of 16 bits show.
__device__ __forceinline__ float rms_inverse(float mean_square, bool fast) {
  return fast ? rsqrtf(mean_square) : __frsqrt_rn(mean_square);
}

// cos and sin of the slot's pairs, two pairs a load (they lie together, on 16 bytes)
template <int VE, typename Slot>
__device__ __forceinline__ void read_angles(const float2* angles, const Slot& slot, float2 (&v)[VE]) {
  if constexpr (VE == 1) {
    v[0] = angles[slot.pair(0)];
  } else {
#pragma unroll
    for (int e = 0; e < VE; e += 2) {
      const float4 two = *reinterpret_cast<const float4*>(&angles[slot.pair(e)]);
      v[e] = make_float2(two.x, two.y);
      v[e + 1] = make_float2(two.z, two.w);
    }
  }
}
template <int VE>
__device__ __forceinline__ void read_weights(const float* w, float* out) {
  if constexpr (VE == 1) {
    out[0] = w[0];
  } else {
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
      const float4 four = *reinterpret_cast<const float4*>(w + e);
      out[e] = four.x, out[e + 1] = four.y, out[e + 2] = four.z, out[e + 3] = four.w;
    }
  }
}

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

template <typename T, int VE>
__device__ __forceinline__ void store_two(T* row, int a, int b, bool has_a, bool has_b, const float (&f)[2 * VE]) {
  float g[VE];
  if (has_a) {
#pragma unroll
    for (int e = 0; e < VE; ++e) g[e] = f[e];
    store_vec<T, VE>(row + a, pack<T, VE>(g));
  }
  if (has_b) {
#pragma unroll
    for (int e = 0; e < VE; ++e) g[e] = f[VE + e];
    store_vec<T, VE>(row + b, pack<T, VE>(g));
  }
}

// SLOTS: slots a lane.  Forward, and backward where there is no norm (the angles' sign changed).  A task is a token's heads of q and then of
// k, or a share of both, so that the angles serve both; a warp's turn takes the next `groups` of them.
template <typename T, int VE, int SLOTS, bool WHOLE, bool INTER, bool NORM>
__global__ void __launch_bounds__(kThreads) rotary_fwd_kernel(const Rotary p) {
  __shared__ alignas(16) float2 angles[kWarps][kMostHead / 2];
  __shared__ PairTable table;
  __shared__ alignas(16) float weights[NORM ? 2 : 1][NORM ? kMostHead : 1];
  constexpr bool RING = kRing<T, VE>;
  __shared__ Ring<RING, 2, 2 * SLOTS> ring;
  constexpr int STAGES = decltype(ring)::kStages;
  using Where = Slot<VE, INTER, WHOLE>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane & (p.lanes - 1), group = lane / p.lanes, groups = 32 / p.lanes;
  const int per_token = p.tasks_per_token[0];
  const int tasks = p.tokens * per_token, step = (int)gridDim.x * kWarps;
  // the heads of q (t = 0) or k that are a task's
  const auto heads_from = [&](int task, int token, int t) { return min((task - token * per_token) * p.per_task[t], p.heads[t]); };
  const auto heads_to = [&](int from, int t) { return min(from + p.per_task[t], p.heads[t]); };

  // What is asked for next: the warp's next turn of a task's heads of q, then of k; row: this lane's head.
  const int first_task = (int)blockIdx.x * kWarps + warp;
  int asked = first_task, ask_t = 0, ask_head = 0, ask_to = 0, ask_stage = 0, ask_token = 0, ask_b = 0, ask_s = 0;
  const T* row = nullptr;
  long long row_step = 0;
  const auto open = [&]() {
    const int from = heads_from(asked, ask_token, ask_t);
    ask_to = heads_to(from, ask_t);
    ask_head = from + group;
    row = static_cast<const T*>(p.in[ask_t]) + place(p.in_stride[ask_t], ask_b, ask_s, ask_head);
    row_step = groups * p.in_stride[ask_t][2];
  };
  const auto advance = [&]() {  // to the next heads that there are
    do {
      ask_t ^= 1;
      if (ask_t == 0) {
        asked += step;
        if (asked >= tasks) return;
        ask_token = token_of(p, asked, per_token, ask_b, ask_s);
      }
      open();
    } while (ask_head - group >= ask_to);
  };
  Pack<T, VE> va[SLOTS], vb[SLOTS];
  const auto ask = [&]() {
    if (ask_head < ask_to && asked < tasks) {
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const Where slot(l + j * p.lanes, p.pairs, p.D);
        if constexpr (RING) {
          if (slot.has_a) cp_async16(smem_addr(&ring.at[warp][ask_stage][2 * j][lane]), row + slot.a);
          if (slot.has_b) cp_async16(smem_addr(&ring.at[warp][ask_stage][2 * j + 1][lane]), row + slot.b);
        } else {
          if (slot.has_a) va[j] = load_vec<T, VE>(row + slot.a);
          if (slot.has_b) vb[j] = load_vec<T, VE>(row + slot.b);
        }
      }
    }
    if constexpr (RING) {
      cp_async_commit();
      ask_stage = (ask_stage + 1) % STAGES;
    }
    row += row_step;
    ask_head += groups;
    if (ask_head - group >= ask_to && asked < tasks) advance();
  };
  if (asked < tasks) {
    ask_token = token_of(p, asked, per_token, ask_b, ask_s);
    open();
    if (ask_head - group >= ask_to) advance();
  }
#pragma unroll
  for (int i = 0; i < STAGES; ++i) ask();
  fill_pairs(p, table);
  if constexpr (NORM) {
    for (int i = threadIdx.x; i < 2 * p.D; i += kThreads) {
      const int t = i >= p.D, at = i - t * p.D;
      if (p.heads[t]) weights[t][at] = p.offset + param_at(p.weight[t], p.w_dtype[t], at, 1.f);
    }
  }
  __syncthreads();
  Positions positions = {};
  int b = 0, s = 0, token = 0, stage = 0;
  if (first_task < tasks) {
    token = token_of(p, first_task, per_token, b, s);
    ask_positions(p, table, b, s, positions);
  }
  for (int task = first_task; task < tasks; task += step) {
    token_angles(p, table, b, s, positions, sizeof(T) == 2, angles[warp]);
    const int now = token;
    if (task + step < tasks) {
      token = token_of(p, task + step, per_token, b, s);
      ask_positions(p, table, b, s, positions);
    }
    float aa[SLOTS][VE], ab[SLOTS][VE], bb[SLOTS][VE], ba[SLOTS][VE];
    bool have = false;
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const int from = heads_from(task, now, t), to = heads_to(from, t);
      if (from >= to) continue;
      if (NORM || !have) {
        // The rotation's coefficients, the norm's weights among them.
        have = true;
        const float* w = weights[NORM ? t : 0];
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
          const Where slot(l + j * p.lanes, p.pairs, p.D);
          float2 v[VE];
          if (slot.turns) read_angles<VE>(angles[warp], slot, v);
          if constexpr (NORM) {
            float wi[2 * VE] = {};
            if (slot.has_a) read_weights<VE>(w + slot.a, wi);
            if (slot.has_b) read_weights<VE>(w + slot.b, wi + VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              if (slot.turns) {
                const float first = wi[Where::first(e)], second = wi[Where::second(e)];
                aa[j][e] = v[e].x * first, ab[j][e] = -v[e].y * second, bb[j][e] = v[e].x * second, ba[j][e] = v[e].y * first;
              } else {  // (the weights alone)
                aa[j][e] = wi[e], bb[j][e] = wi[VE + e], ab[j][e] = ba[j][e] = 0.f;
              }
            }
          } else if (slot.turns) {
#pragma unroll
            for (int e = 0; e < VE; ++e) aa[j][e] = bb[j][e] = v[e].x, ab[j][e] = -v[e].y, ba[j][e] = v[e].y;
          }
        }
      }
      T* out = static_cast<T*>(p.out[t]) + ((long long)now * p.heads[t] + from + group) * p.D;
      const int out_step = groups * p.D;
      for (int head = from + group; head - group < to; head += groups, out += out_step) {
        if constexpr (RING) cp_async_wait<STAGES - 1>();
        float f[SLOTS][2 * VE];
        float sq[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
          const Where slot(l + j * p.lanes, p.pairs, p.D);
          if constexpr (RING) {
            va[j] = load_vec<T, VE>(reinterpret_cast<const T*>(&ring.at[warp][stage][2 * j][lane]));
            vb[j] = load_vec<T, VE>(reinterpret_cast<const T*>(&ring.at[warp][stage][2 * j + 1][lane]));
          }
          unpack_two<T, VE>(va[j], vb[j], f[j]);
          if constexpr (!WHOLE) {
#pragma unroll
            for (int e = 0; e < 2 * VE; ++e)
              if (!(e < VE ? slot.has_a : slot.has_b)) f[j][e] = 0.f;
          }
          if constexpr (NORM) dot_each(sq, f[j], f[j]);
          if (slot.turns) {
            turn<VE, INTER>(f[j], aa[j], ab[j], bb[j], ba[j]);
          } else if constexpr (NORM) {
#pragma unroll
            for (int e = 0; e < VE; ++e) f[j][e] *= aa[j][e], f[j][VE + e] *= bb[j][e];
          }
        }
        if constexpr (RING) stage = (stage + 1) % STAGES;
        ask();
        if constexpr (NORM) {
          const float rstd = rms_inverse(fmaf(lanes_sum(sq[0] + sq[1], p.lanes), p.inv_d, p.eps), sizeof(T) == 2);
#pragma unroll
          for (int j = 0; j < SLOTS; ++j) scale_each(f[j], rstd);
        }
        if (head < to) {  // (a group beyond the last head has nothing to store)
#pragma unroll
          for (int j = 0; j < SLOTS; ++j) {
            const Where slot(l + j * p.lanes, p.pairs, p.D);
            store_two<T, VE>(out, slot.a, slot.b, slot.has_a, slot.has_b, f[j]);
          }
        }
      }
    }
  }
}

// Backward of the norm.  A CTA takes heads of q or of k alone, since a lane's sums for the weight's gradient stand in registers.
template <typename T, int VE, int SLOTS, bool WHOLE, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_bwd_kernel(const Rotary p) {
  __shared__ alignas(16) float2 angles[kWarps][kMostHead / 2];
  __shared__ PairTable table;
  constexpr bool RING = kRing<T, VE>;
  __shared__ Ring<RING, 2, 4 * SLOTS> ring;
  constexpr int STAGES = decltype(ring)::kStages;
  using Where = Slot<VE, INTER, WHOLE>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane & (p.lanes - 1), group = lane / p.lanes, groups = 32 / p.lanes;
  const int t = blockIdx.x >= p.ctas[0];  // q or k
  const unsigned cta = blockIdx.x - (t ? p.ctas[0] : 0);
  grid_dep_launch_dependents();
  const int per_token = p.tasks_per_token[t], per_task = p.per_task[t], heads = p.heads[t];
  // (the gradient of an fp32 weight is a sum of the same terms that stays in 32 bits: 16384 tokens of 32 + 32 heads 134 us, fast 130)
  const bool fast = sizeof(T) == 2 && p.w_dtype[t] != GNB200_F32;
  const int tasks = p.tokens * per_token, step = (int)p.ctas[t] * kWarps;
  // what is asked for next: the warp's next turn of a task's heads; in, xs: this lane's head of the gradient and of the input
  const int first_task = (int)cta * kWarps + warp;
  const long long in_step = groups * p.in_stride[t][2], xs_step = groups * p.x_stride[t][2];
  int asked = first_task, ask_head = 0, ask_to = 0, ask_stage = 0;
  const T *in = nullptr, *xs = nullptr;
  const auto open = [&]() {
    int b, s;
    const int token = token_of(p, asked, per_token, b, s), from = (asked - token * per_token) * per_task;
    ask_head = from + group;
    ask_to = min(from + per_task, heads);
    in = static_cast<const T*>(p.in[t]) + place(p.in_stride[t], b, s, ask_head);
    xs = static_cast<const T*>(p.x[t]) + place(p.x_stride[t], b, s, ask_head);
  };
  Pack<T, VE> v[SLOTS][4];  // of a slot: the gradient's two vectors, the input's two
  const auto ask = [&]() {
    if (ask_head < ask_to && asked < tasks) {
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const Where slot(l + j * p.lanes, p.pairs, p.D);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i % 2 ? slot.has_b : slot.has_a) {
            const T* from = (i / 2 ? xs : in) + (i % 2 ? slot.b : slot.a);
            if constexpr (RING)
              cp_async16(smem_addr(&ring.at[warp][ask_stage][4 * j + i][lane]), from);
            else
              v[j][i] = load_vec<T, VE>(from);
          }
        }
      }
    }
    if constexpr (RING) {
      cp_async_commit();
      ask_stage = (ask_stage + 1) % STAGES;
    }
    in += in_step;
    xs += xs_step;
    ask_head += groups;
    if (ask_head - group >= ask_to && asked < tasks) {
      asked += step;
      if (asked < tasks) open();
    }
  };
  if (asked < tasks) open();
#pragma unroll
  for (int i = 0; i < STAGES; ++i) ask();
  fill_pairs(p, table);
  __syncthreads();
  float w[SLOTS][2 * VE], dw[SLOTS][2 * VE];
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    const Where slot(l + j * p.lanes, p.pairs, p.D);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      w[j][e] = slot.has_a ? p.offset + param_at(p.weight[t], p.w_dtype[t], slot.a + e, 1.f) : 0.f;
      w[j][VE + e] = slot.has_b ? p.offset + param_at(p.weight[t], p.w_dtype[t], slot.b + e, 1.f) : 0.f;
      dw[j][e] = dw[j][VE + e] = 0.f;
    }
  }
  Positions positions = {};
  int b = 0, s = 0, token = 0, stage = 0;
  if (first_task < tasks) {
    token = token_of(p, first_task, per_token, b, s);
    ask_positions(p, table, b, s, positions);
  }
  for (int task = first_task; task < tasks; task += step) {
    token_angles(p, table, b, s, positions, fast, angles[warp]);
    const int from = (task - token * per_token) * per_task, to = min(from + per_task, heads);
    T* out = static_cast<T*>(p.out[t]) + ((long long)token * heads + from + group) * p.D;
    const int out_step = groups * p.D;
    if (task + step < tasks) {
      token = token_of(p, task + step, per_token, b, s);
      ask_positions(p, table, b, s, positions);
    }
    float aa[SLOTS][VE], ab[SLOTS][VE], bb[SLOTS][VE], ba[SLOTS][VE];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const Where slot(l + j * p.lanes, p.pairs, p.D);
      if (slot.turns) {
        float2 c[VE];
        read_angles<VE>(angles[warp], slot, c);
#pragma unroll
        for (int e = 0; e < VE; ++e) aa[j][e] = bb[j][e] = c[e].x, ab[j][e] = -c[e].y, ba[j][e] = c[e].y;
      }
    }
    for (int head = from + group; head - group < to; head += groups, out += out_step) {
      const bool live = head < to;  // (a group beyond the last head adds and stores nothing)
      if constexpr (RING) cp_async_wait<STAGES - 1>();
      float f[SLOTS][2 * VE], n[SLOTS][2 * VE];
      float sq[2] = {0.f, 0.f}, dot[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const Where slot(l + j * p.lanes, p.pairs, p.D);
        if constexpr (RING) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[j][i] = load_vec<T, VE>(reinterpret_cast<const T*>(&ring.at[warp][stage][4 * j + i][lane]));
        }
        unpack_two<T, VE>(v[j][0], v[j][1], f[j]);
        unpack_two<T, VE>(v[j][2], v[j][3], n[j]);
        if constexpr (!WHOLE) {
#pragma unroll
          for (int e = 0; e < 2 * VE; ++e) {
            if (!(e < VE ? slot.has_a : slot.has_b)) f[j][e] = n[j][e] = 0.f;
          }
        }
        if (slot.turns) turn<VE, INTER>(f[j], aa[j], ab[j], bb[j], ba[j]);
        dot_each(sq, n[j], n[j]);
      }
      if constexpr (RING) stage = (stage + 1) % STAGES;
      ask();
      // both sums at once: mean(g w n) = rstd * mean(g w x)
      float gw[SLOTS][2 * VE];
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
#pragma unroll
        for (int e = 0; e < 2 * VE; ++e) gw[j][e] = f[j][e];
        mul_each(gw[j], w[j]);
        dot_each(dot, gw[j], n[j]);
      }
      const float all_sq = lanes_sum(sq[0] + sq[1], p.lanes), all_dot = lanes_sum(dot[0] + dot[1], p.lanes);
      const float rstd = rms_inverse(fmaf(all_sq, p.inv_d, p.eps), fast), c = -all_dot * rstd * p.inv_d;
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        scale_each(n[j], rstd);
        if (live) fma_each(dw[j], f[j], n[j]);
        axpy_each(gw[j], n[j], c);
        scale_each(gw[j], rstd);
      }
      if (live) {
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
          const Where slot(l + j * p.lanes, p.pairs, p.D);
          store_two<T, VE>(out, slot.a, slot.b, slot.has_a, slot.has_b, gw[j]);
        }
      }
    }
  }
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

// How the tokens' heads are dealt out: warps take whole tokens where there are enough of them, else shares of a token's heads.  Forward q and
// k share the tasks; backward each has CTAs in proportion to a token's turns of the warp, and two more for the angles and all else that a token
// takes (16384 tokens, 32 and 8 heads of 128: 134 us in proportion to the heads, 98 with them).
// Forward calls with many heads are bound by memory: four CTAs an SM keep 32 KB of heads ahead, and more of them only disturb one another.
// With few heads a token's angles count for more, with a norm its coefficients too, and every warp helps.  16384 tokens, bf16, us with four CTAs and
// with five, by a token's turns of the warp:
//   heads of 128, norm    6: 41.3, 38.9    8: 49.5, 47.4    9: 54.2, 53.3    10: 58.6, 58.5 and 59.9    12: 67.6, 73.9    16: 87.9, 98.9
//   without               6: 36.1, 36.5    7: 40.7, 42.3    8: 45.2, 48.8    10: 55.5, 60.7    12: 65.3, 71.8    16: 88.0, 94.0
//   heads of 64, norm     6: 36.1, 35.7    8: 45.8, 48.0    10: 55.4, 61.4;   of 256    8: 54.0, 50.8    10: 63.0, 61.1    12: 71.4, 71.2    16: 90.8, 99.8
//   without               6: 34.7, 36.1    8: 44.6, 49.0;                      of 256    6: 37.4, 36.9    8: 46.9, 49.1
constexpr int kTokenTurns = 2, kManyTurns = 7, kManyTurnsWithNorm = 10;
cudaError_t rotary_split(const void* kernel, const RotaryGeom& g, bool ring, bool norm, bool back, Rotary& p) {
  Residency r;
  const cudaError_t err = residency(kernel, kThreads, 0, &r);
  if (err != cudaSuccess) return err;
  const int groups = 32 / g.lanes;
  long long want[2] = {0, 0}, turns[2] = {0, 0}, weight[2] = {0, 0};
  for (int t = 0; t < 2; ++t) {
    if (!p.heads[t]) continue;
    turns[t] = (p.heads[t] + groups - 1) / groups;  // of a warp, for a token
    weight[t] = turns[t] + kTokenTurns;
  }
  if (ring && !back && turns[0] + turns[1] >= (norm ? kManyTurnsWithNorm : kManyTurns)) r.per_sm = std::min(r.per_sm, 4);
  const long long most = (long long)r.per_sm * r.sms;
  for (int t = 0; t < 2; ++t) {
    if (!p.heads[t]) continue;
    const long long warps = back ? most * kWarps * weight[t] / (weight[0] + weight[1]) : most * kWarps;
    const long long tasks = std::min(turns[t], std::max(1LL, warps / std::max(1, p.tokens)));
    p.per_task[t] = (int)((turns[t] + tasks - 1) / tasks) * groups;
    p.tasks_per_token[t] = (p.heads[t] + p.per_task[t] - 1) / p.per_task[t];
    want[t] = ((long long)p.tokens * p.tasks_per_token[t] + kWarps - 1) / kWarps;
  }
  if (!back) {
    p.tasks_per_token[0] = std::max(p.tasks_per_token[0], p.tasks_per_token[1]);
    want[0] = std::min(most, std::max(want[0], want[1]));
    want[1] = 0;
  } else if (want[0] + want[1] > most) {
    for (int t = 0; t < 2; ++t)
      if (want[t]) want[t] = std::max(1LL, std::min(want[t], most * weight[t] / (weight[0] + weight[1])));
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
    const cudaError_t err = rotary_split((const void*)kernel, g, g.ve == (dtype == GNB200_F32 ? 4 : 8), norm, back, p);
    if (err != cudaSuccess || plan_only) return err;
    kernel<<<p.ctas[0] + p.ctas[1], kThreads, 0, stream>>>(p);
    return cudaGetLastError();
  };
  auto typed = [&](auto type) {
    using T = decltype(type);
    return with_rotary_geometry<T>(g, [&](auto ve, auto slots, auto whole) {
      constexpr int VE = decltype(ve)::value, S = decltype(slots)::value;
      constexpr bool W = decltype(whole)::value;
      if (back) return inter ? go(&rotary_bwd_kernel<T, VE, S, W, true>) : go(&rotary_bwd_kernel<T, VE, S, W, false>);
      if (norm) return inter ? go(&rotary_fwd_kernel<T, VE, S, W, true, true>) : go(&rotary_fwd_kernel<T, VE, S, W, false, true>);
      return inter ? go(&rotary_fwd_kernel<T, VE, S, W, true, false>) : go(&rotary_fwd_kernel<T, VE, S, W, false, false>);
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
  if (a->q_heads > (1 << 20) || a->k_heads > (1 << 20) || a->tokens >= (1LL << 30) || a->batch >= (1LL << 30) ||
      a->batch * a->tokens >= (1LL << 30))
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: more than 2^20 heads or 2^30 tokens", name);
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
  p.tokens = (int)(a->batch * a->tokens);
  p.S = (int)a->tokens;
  while ((1LL << p.div_shift) < p.S) ++p.div_shift;
  p.div_mul = (unsigned)(((1ULL << 32) * ((1ULL << p.div_shift) - (unsigned)p.S)) / (unsigned)p.S + 1);
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
  static thread_local Remembered<8> known;  // the answer depends on nothing but these and the device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const Remembered<8>::Key key = {p.tokens, p.D, p.pairs, p.heads[0], p.heads[1], a->interleaved != 0, a->dtype, dev};
  if (const size_t* v = known.find(key)) return *v;
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
  return known.keep(key, most);
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
