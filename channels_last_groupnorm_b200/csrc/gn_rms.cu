// Root-mean-square norm of token rows with the residual's addition: forward, forward with an 8-bit output and
// scales, backward.
//
//   s = x + r                      added in fp32, stored rounded once to r's type; the norm takes the unrounded sum
//   y = s * rstd * (offset + w)    rstd = 1 / sqrt(mean(s^2) + eps) over the C channels of a row
//   q = y / scale                  scale = max(|y|) / largest code, per row or per block of channels; at least 2^-126
//   d = ds + rstd * (g - n * mean(g * n))   with n = s * rstd, g = dy * (offset + w): the gradient of x and of r
//   dw = sum over rows of dy * n
//
// Every element is read and written once: a row's elements stay in registers (backward: in shared memory) between the sum over the row and
// the output, and the only traffic beside them is a row of partial sums per CTA in the backward.  Bound by HBM where there are rows enough:
// 16384 x 4096 bf16 with the residual, forward 89 us = 6.0 TB/s, backward (four tensors read, one written) 107 us = 6.3 TB/s, 92 and
// 96 % of a copy's rate; 8192 x 8192 bf16 over an fp32 stream to 8 bits 115 us = 6.4 TB/s.  A call of one row takes 2.2 us, of 8 rows in
// 8 bits 3: launch, first load and one reduction.  With 4-bit codes (gn_four.cuh): 8192 x 8192 bf16 over an fp32 stream 115 us in blocks of 32, 120 of 16, over bf16 73 = 6.0 TB/s, 2048 x 4096
// over fp32 20, odd rows 36 (9001 x 1111).
//
// Rows of up to four vectors a lane belong to a group of lanes of one warp (shuffles only), longer ones to a CTA, or in the backward to a
// team of warps, of which a CTA has several so that fewer partial rows are left to add up; rows longer than those (more than 16384
// channels, odd ones a little fewer) are read two or three times, element by element (`any`).  The backward of short and odd widths is
// bound by instructions and by idle lanes, not by HBM: 30000 x 320 bf16 27 us for 14.6 of traffic, 9000 x 1112 28 for 15.3, 4000 x 1280
// fp32 19.5 for 12.5.  The grid holds the CTAs that are resident at once; each keeps its channels' weights in registers, walks over the
// rows and asks for the next ones early: into registers while these are few (one row, 64 bytes a thread), otherwise by cp.async into a ring
// of rows in shared memory, which costs two more instructions a vector but no registers (8192 x 8192 to 8 bits 136 -> 121 us; the backward
// of 16384 x 4096 125 -> 106, whose spills it ended; the forward of 16384 x 4096 stays in registers: 88 against 93).
#include <algorithm>
#include <initializer_list>

#include "../../include/gnb200.h"
#include "gn_four.cuh"
#include "gn_kernels.h"
#include "gn_rows.h"
#include "gn_tokens.cuh"

namespace gnb200 {
namespace {

constexpr int kWarpThreads = 128;  // CTA size of the kernels with one group of lanes per row
constexpr int kMostThreads = 512;  // CTA size of the kernels for rows of any length
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126: its reciprocal is finite, a block of zeros gets codes of zero

struct RmsFwd {
  const void *x, *residual, *weight;
  void *y, *sum;  // y: or the codes
  float *rstd, *scale;
  long long rows, x_stride, r_stride;
  int C, lanes, stages, stage_bytes, w_dtype, block, blocks, format;
  float eps, offset, inv_c;
  int edge;  // rows at either end that Frame::readable looks at
};
static_assert(sizeof(RmsFwd) <= 128, "above that the compiler's copy of the arguments changes the kernels' registers: 16384 x 2560 bf16 54.5 -> 58.8 us");

// ---------------------------------------------------------------------------------------------
// 8-bit codes
// ---------------------------------------------------------------------------------------------
// A code is that of y / scale rounded as a division rounds it, so that codes and y / scale agree wherever they are formed: the product
// q = y * inverse with the correctly rounded reciprocal is at most one unit of its last place off, and q - inverse * (q * scale - y), the
// remainder taken exactly by an fma, is the rounded quotient (Markstein's theorem; y below 2^-126 aside).  The reciprocal: one Newton
// step from the hardware's, which is a unit off at most (the same bits as __frcp_rn for every mantissa, without its branch for other ranges).  Two
// fma an element; the product alone gave one code in 100 000 of the neighbouring value, where bf16 inputs put y / scale midway between
// two codes.  2048 x 4096 bf16 in blocks of 128: product alone 10.7 us, so 11.2, with __frcp_rn 11.7; 8192 x 8192 over fp32 118.5 and 115.
struct Scale {
  float value, inverse;
  float back;  // value; 0 where it is infinite: what is finite over infinity is zero, not the remainder's NaN
};
__device__ __forceinline__ Scale scale_of(uint32_t most, int format) {
  const float s = __uint_as_float(most) * (format == GNB200_E4M3 ? 1.f / 448.f : 1.f / 127.f);
  Scale scale;
  scale.value = s < kSmallestScale ? kSmallestScale : s;  // (a NaN stays)
  float near;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(near) : "f"(scale.value));
  const bool infinite = near == 0.f;
  scale.inverse = infinite ? 0.f : fmaf(fmaf(-scale.value, near, 1.f), near, near);
  scale.back = infinite ? 0.f : scale.value;
  return scale;
}
__device__ __forceinline__ float over(float y, float inverse, float back) {
  const float q = y * inverse;
  return fmaf(-inverse, fmaf(q, back, -y), q);
}
template <int VE>
__device__ __forceinline__ void over_each(float (&f)[VE], const Scale& scale) {
  const float inverse = scale.inverse, back = scale.back, less = -inverse;
#pragma unroll
  for (int e = 0; e < VE; e += 2) {
    float q0, q1, r0, r1;
    mul2(q0, q1, f[e], f[e + 1], inverse, inverse);
    fma2(r0, r1, q0, q1, back, back, -f[e], -f[e + 1]);
    fma2(f[e], f[e + 1], r0, r1, less, less, q0, q1);
  }
}
__device__ __forceinline__ uint32_t code_of(float v, int format) {
  if (format == GNB200_E4M3) return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)max(-127, min(127, __float2int_rn(v))) & 0xffu;
}
// VE codes of quotients, four a word
template <int VE>
__device__ __forceinline__ void codes_of(const float (&v)[VE], int format, uint32_t (&w)[VE / 4]) {
#pragma unroll
  for (int k = 0; k < VE / 4; ++k) {
    const float* g = v + 4 * k;
    if (format == GNB200_E4M3) {
      const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(g[0], g[1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(g[2], g[3]), __NV_SATFINITE, __NV_E4M3);
      w[k] = __byte_perm(low, high, 0x5410);
    } else {
      int n[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) n[e] = max(-127, min(127, __float2int_rn(g[e])));
      w[k] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Rows as vectors
// ---------------------------------------------------------------------------------------------
// RAGGED rows start between the boundaries of 16 bytes, or end there.  They are taken in a frame that begins at the boundary before: vector i
// holds channels i * VE - skew and on, the first and the last one in part.  All tensors of a call have the same frame (checked by the
// host), and the step from one of a thread's rows to the next is a multiple of VE rows, so that the skew, and with it the channels of a thread, stay:
// its weights and sums are in registers as they are for aligned rows.  Device us, element by element and so: 9000 rows of 1111 bf16 with a
// residual, forward 27.0 and 21.1, backward 42.3 and 40.2; 3000 of 12345, backward 210 and 154; 4000 of 12345 fp16 over fp32, 8-bit output with
// blocks, 592 and 224.  Twice the instructions of aligned rows bound them: the sums' way through shared memory, and the edges.
template <int VE, bool RAGGED>
struct Frame {
  int skew, nvec, C;
  __device__ __forceinline__ Frame(uint32_t row_elements, int channels) {
    C = channels;
    skew = RAGGED ? (int)(row_elements % VE) : 0;
    nvec = RAGGED ? (C + skew + VE - 1) / VE : C / VE;
  }
  __device__ __forceinline__ bool whole(int i) const { return !RAGGED || (i * VE >= skew && (i + 1) * VE - skew <= C); }
  __device__ __forceinline__ int channel(int i) const { return i * VE - skew; }  // of the vector's first element; may lie before the row
  __device__ __forceinline__ bool has(int i, int e) const { return !RAGGED || (unsigned)(channel(i) + e) < (unsigned)C; }
  // elements outside of the row become zero
  __device__ __forceinline__ void cut(float (&f)[VE], int i) const {
    if constexpr (RAGGED) {
      if (!whole(i)) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (!has(i, e)) f[e] = 0.f;
      }
    }
  }
  // Whether vector i may be read as a whole, with elements of the rows beside it: in the tensor's first and last rows (not `inner`, by
  // edge_rows()) only where it lies in the row.  What may not is fetched where it is used.
  __device__ __forceinline__ bool readable(int i, bool inner) const { return !RAGGED || inner || whole(i); }
  template <typename T>
  __device__ __forceinline__ Pack<T, VE> fetch(const T* row, int i) const {
    Pack<T, VE> v;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      v.v[e] = store_param<T>(0.f);
      if (has(i, e)) v.v[e] = row[i * VE + e];
    }
    return v;
  }
  // Sums over a ragged row go through shared memory, so that each lane adds the same channels in the same order wherever the row stands:
  // written as vectors of the frame, read a channel a lane.  (In planes of channel mod VE: 27002 x 1111 bf16 69 us instead of 58, its backward 116 instead of 95.)
  __device__ __forceinline__ void lay_out(float* line, int i, const float (&f)[VE]) const {
#pragma unroll
    for (int e = 0; e < VE; e += 4) *reinterpret_cast<float4*>(line + i * VE + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
  }
  // channels first + step * (v VE + 0, 1, ...); zeros behind the row
  __device__ __forceinline__ void take(const float* line, int v, int first, int step, float (&f)[VE]) const {
    const int from = first + v * VE * step;
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = from + e * step < C ? line[skew + from + e * step] : 0.f;
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, int i, const float (&f)[VE]) const {
    if (whole(i)) {
      store_vec<T, VE>(row + i * VE, pack<T, VE>(f));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (has(i, e)) row[i * VE + e] = store_param<T>(f[e]);
    }
  }
};

// Bytes of a tensor's row in a stage
__host__ __device__ constexpr int segment_bytes(int C, int ve, int size, bool ragged) { return ragged ? (C + 2 * ve - 2) / ve * ve * size : C * size; }

// ... and of the line of its sum
__host__ __device__ constexpr int line_bytes(int C, int ve, bool ragged) { return segment_bytes(C, ve, ragged ? 4 : 0, ragged); }

// Copies a row to its stage, 16 bytes a lane; of the tensor's first and last rows (not `inner`) its own elements alone, so that nothing
// outside of the tensor is read.
template <typename T, int VE, int V, bool RAGGED>
__device__ __forceinline__ void ask_row(char* stage, const T* row, const Frame<VE, RAGGED>& frame, int first, int step, bool inner) {
  const uint32_t dst = smem_addr(stage);
  constexpr int kParts = sizeof(T) * VE / 16;  // 32 bytes where 8 floats stand beside 8 halves
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = first + v * step;
    if (i < frame.nvec) {
      if (frame.readable(i, inner)) {
#pragma unroll
        for (int k = 0; k < kParts; ++k) cp_async16(dst + (i * kParts + k) * 16, reinterpret_cast<const char*>(row) + (i * kParts + k) * 16);
      } else {
        for (int e = 0; e < VE; ++e)
          if (frame.has(i, e)) reinterpret_cast<T*>(stage)[i * VE + e] = row[i * VE + e];
      }
    }
  }
}

// (offset + w) of this thread's channels
template <int VE, int V, bool RAGGED>
__device__ __forceinline__ void fetch_weight(float (&w)[V][VE], const void* p, int dtype, float offset, const Frame<VE, RAGGED>& frame, int first,
                                             int step) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = first + v * step;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[v][e] = 1.f;
    if (p != nullptr && i < frame.nvec) {
      if constexpr (RAGGED) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (frame.has(i, e)) w[v][e] = param_at(p, dtype, frame.channel(i) + e, 1.f);
      } else {
        params_at<VE>(p, dtype, i * VE, w[v]);
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) w[v][e] += offset;
    }
  }
}

// the codes of vector i of the row whose frame begins at `row`
template <int VE, bool RAGGED>
__device__ __forceinline__ void store_codes(uint8_t* row, const Frame<VE, RAGGED>& frame, int i, const float (&quotients)[VE], int format) {
  uint32_t w[VE / 4];
  codes_of<VE>(quotients, format, w);
  if (frame.whole(i)) {
    if constexpr (VE == 8)
      *reinterpret_cast<uint2*>(row + i * VE) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(row + i * VE) = w[0];
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (frame.has(i, e)) row[i * VE + e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
  }
}

// How the rows are dealt out: this thread's place in its row's group, the group's rows and its stages.
// A group is a power-of-two number of lanes of one warp (WARP), a team of whole warps (TEAMS) or the CTA.
template <bool WARP, bool TEAMS>
struct Place {
  int lanes, first, group;
  long long per_cta, base, row, step;
  char* stages;
  float* line;
  __device__ __forceinline__ Place(int row_lanes, int stage_bytes, int nstages, int line_bytes, char* smem) {
    lanes = WARP || TEAMS ? row_lanes : (int)blockDim.x;
    group = WARP || TEAMS ? (int)threadIdx.x / lanes : 0;
    first = (int)threadIdx.x - group * lanes;
    per_cta = WARP || TEAMS ? (int)blockDim.x / lanes : 1;
    base = blockIdx.x * per_cta + (WARP ? 0 : group);  // (a warp's groups take their turns together, teams each for themselves)
    row = blockIdx.x * per_cta + group;
    step = per_cta * gridDim.x;
    stages = smem + (long long)group * (stage_bytes * nstages + line_bytes);
    line = reinterpret_cast<float*>(stages + stage_bytes * nstages);
  }
  // what the group's other lanes wrote becomes visible
  __device__ __forceinline__ void meet() const {
    if constexpr (WARP)
      __syncwarp();
    else
      team_barrier<TEAMS>(lanes, group);
  }
  // what the group's other lanes read may be written again behind the row's sum: a team has that sum's barrier, lanes of a warp only shuffles,
  // which order no memory
  __device__ __forceinline__ void part() const {
    if constexpr (WARP) __syncwarp();
  }
};

// ---------------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------------
// What a thread holds of the row that comes next: registers where a few vectors do, otherwise the stages.
template <typename Tx, typename Ts, int VE, int V, int THREADS>
constexpr bool kStaged = THREADS > kWarpThreads && (THREADS > 512 || V * VE * (sizeof(Tx) + sizeof(Ts)) > 64);
constexpr int kMostBlocks = 512;  // of the rows that these kernels take
enum Output { kPlain = 0, kCodes8 = 1, kCodes4Of16 = 2, kCodes4Of32 = 3 };  // (4-bit codes in blocks of 16 or 32)
__host__ __device__ constexpr bool is_four(int out) { return out >= kCodes4Of16; }

// THREADS: the CTA's at most; kWarpThreads where a row has a group of lanes, otherwise a row has the CTA
// OUT: y in x's type, 8-bit codes, 4-bit codes (`rstd` is the tensor's scale then, `scale` the tiles, `blocks` how many lie along a row).  Blocks of 4-bit codes
// begin at channel 0: of a ragged row they are taken out of the line that its sum went through.
// (4-bit codes: the compiler is held to two CTAs of 512 threads, three or five of 128; 0 leaves it free as no second bound does; left to itself it took 100 registers for the 50 of before a smaller change, and
// 8192 x 8192 over fp32 158 us in place of 127.)
template <typename Tx, typename Ts, int VE, int V, int THREADS, int OUT, bool RES, bool RAGGED>
__global__ void __launch_bounds__(THREADS, !is_four(OUT) || THREADS == 1024 ? 0 : THREADS == 512 ? 2 : V == 4 ? 3 : 5) rms_fwd_kernel(const RmsFwd p) {
  constexpr bool WARP = THREADS == kWarpThreads, STAGED = kStaged<Tx, Ts, VE, V, THREADS>;
  extern __shared__ __align__(16) char smem[];
  __shared__ TeamSlots slots;
  __shared__ uint32_t most[32];
  __shared__ uint2 blocks[OUT == kCodes8 && RAGGED ? kMostBlocks : 1];  // maxima of a block's own vectors, of the channels before them
  const Place<WARP, false> at(p.lanes, p.stage_bytes, p.stages, line_bytes(p.C, VE, RAGGED), smem);
  if constexpr (is_four(OUT)) grid_dep_launch_dependents();  // (the product that takes the codes)
  const int lanes = at.lanes, first = at.first;
  const Tx* next_x = static_cast<const Tx*>(p.x) + at.row * p.x_stride;  // the next row to be asked for
  const Ts* next_r = RES ? static_cast<const Ts*>(p.residual) + at.row * p.r_stride : nullptr;
  const Frame<VE, RAGGED> frame((uint32_t)(reinterpret_cast<uintptr_t>(next_x) / sizeof(Tx)), p.C);
  const int nvec = frame.nvec, r_at = segment_bytes(p.C, VE, sizeof(Tx), RAGGED);
  next_x -= frame.skew;
  if (RES) next_r -= frame.skew;
  const long long x_step = at.step * p.x_stride, r_step = RES ? at.step * p.r_stride : 0;
  long long asked = at.row;
  int ask_stage = 0, stage = 0;
  Pack<Tx, VE> xv[STAGED ? 1 : V];
  Pack<Ts, VE> rv[STAGED || !RES ? 1 : V];
  auto ask = [&]() {
    if (asked < p.rows) {
      const bool inner = asked >= p.edge && asked < p.rows - p.edge;
      if constexpr (STAGED) {
        char* s = at.stages + ask_stage * p.stage_bytes;
        ask_row<Tx, VE, V, RAGGED>(s, next_x, frame, first, lanes, inner);
        if constexpr (RES) ask_row<Ts, VE, V, RAGGED>(s + r_at, next_r, frame, first, lanes, inner);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int i = first + v * lanes;
          if (i < nvec && frame.readable(i, inner)) {
            xv[v] = load_vec<Tx, VE>(next_x + i * VE);
            if constexpr (RES) rv[v] = load_vec<Ts, VE>(next_r + i * VE);
          }
        }
      }
    }
    if constexpr (STAGED) {
      cp_async_commit();
      ask_stage = ask_stage + 1 == p.stages ? 0 : ask_stage + 1;
    }
    next_x += x_step;
    next_r += r_step;
    asked += at.step;
  };
  ask();
  if constexpr (STAGED)
    for (int i = 1; i < p.stages; ++i) ask();
  float w[V][VE];
  Frame<VE, RAGGED> weights = frame;
  if constexpr (is_four(OUT)) weights.skew = 0, weights.nvec = (p.C + VE - 1) / VE;
  fetch_weight<VE, V, RAGGED>(w, p.weight, p.w_dtype, p.offset, weights, first, lanes);
  if constexpr (!WARP) clear<false>(slots, lanes, 0, first);
  int turn = 0;
  long long row = at.row;
  // (every thread of a warp takes the same number of turns: the shuffles want all lanes)
  for (long long base = at.base; base < p.rows; base += at.step, row += at.step) {
    const bool live = !WARP || row < p.rows;
    const char* here = nullptr;
    if constexpr (STAGED) {
      cp_async_wait_dyn8(p.stages - 1);
      here = at.stages + stage * p.stage_bytes;
      stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
    const long long out_at = row * p.C - frame.skew;  // where the row's frame begins in the outputs
    float s[V][VE];
    float sq[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = first + v * lanes;
#pragma unroll
      for (int e = 0; e < VE; ++e) s[v][e] = 0.f;
      if (live && i < nvec) {
        if (RAGGED && !STAGED && !frame.readable(i, row >= p.edge && row < p.rows - p.edge)) {
          xv[STAGED ? 0 : v] = frame.fetch(static_cast<const Tx*>(p.x) + row * p.x_stride - frame.skew, i);
          if constexpr (RES) rv[STAGED ? 0 : v] = frame.fetch(static_cast<const Ts*>(p.residual) + row * p.r_stride - frame.skew, i);
        }
        if constexpr (STAGED)
          unpack<Tx, VE>(load_vec<Tx, VE>(reinterpret_cast<const Tx*>(here) + i * VE), s[v]);
        else
          unpack<Tx, VE>(xv[v], s[v]);
        if constexpr (RES) {
          float f[VE];
          if constexpr (STAGED)
            unpack<Ts, VE>(load_vec<Ts, VE>(reinterpret_cast<const Ts*>(here + r_at) + i * VE), f);
          else
            unpack<Ts, VE>(rv[v], f);
          add_each(s[v], f);
          frame.store(static_cast<Ts*>(p.sum) + out_at, i, s[v]);
        }
        frame.cut(s[v], i);
        if constexpr (RAGGED) frame.lay_out(at.line, i, s[v]);
      }
      if constexpr (!RAGGED) dot_each(sq, s[v], s[v]);
    }
    if constexpr (RAGGED) {
      at.meet();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (live) {
          float f[VE];
          frame.take(at.line, v, first, lanes, f);
          dot_each(sq, f, f);
        }
      }
      at.part();
    }
    ask();  // (a lane's own vectors: read, so free)
    const float all_sq = WARP ? lanes_sum(sq[0] + sq[1], lanes) : team_sum<false>(sq[0] + sq[1], slots, turn, lanes, 0);
    const float rstd = __frsqrt_rn(fmaf(all_sq, p.inv_c, p.eps));
    if (!is_four(OUT) && p.rstd && live && first == 0) p.rstd[row] = rstd;
    if constexpr (is_four(OUT) && RAGGED) {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int c = (first + v * lanes) * VE + e;
          s[v][e] = live && c < p.C ? at.line[frame.skew + c] : 0.f;
        }
      at.meet();  // (the next row's line is written behind these looks at it)
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // (4-bit codes: zeros behind the channels, which NaN would change; here a vector at a time, below element by element)
      scale_each(s[v], is_four(OUT) && !RAGGED && first + v * lanes >= nvec ? 0.f : rstd);
      mul_each(s[v], w[v]);
    }
    if constexpr (is_four(OUT) && RAGGED) {
      if (!(rstd < __uint_as_float(0x7f800000u))) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if ((first + v * lanes) * VE + e >= p.C) s[v][e] = 0.f;
      }
    }
    if constexpr (OUT == kPlain) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = first + v * lanes;
        if (live && i < nvec) frame.store(static_cast<Tx*>(p.y) + out_at, i, s[v]);
      }
    } else if constexpr (is_four(OUT)) {
      constexpr int BLOCK = OUT == kCodes4Of16 ? 16 : 32, share = BLOCK / VE;
      const TensorScale tensor(BLOCK == 16 ? p.rstd : nullptr);
      const int wide = (int)four_wide(p.C) / VE;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = first + v * lanes;
        const bool inside = live && i < wide;
        float y[8], most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = e < VE ? s[v][e] : 0.f;
#pragma unroll
        for (int e = 0; e < VE; e += 2) most = largest(most, y[e], y[e + 1]);
#pragma unroll
        for (int delta = 1; delta < share; delta *= 2) most = larger(most, __shfl_xor_sync(0xffffffffu, most, delta));
        const FourStep step = four_step<BLOCK>(most, tensor);
        const uint32_t word = codes8<BLOCK>(y, step);
        uint8_t* const to = static_cast<uint8_t*>(p.y) + (row * wide + i) * (VE / 2);
        if (inside) {
          if constexpr (VE == 8)
            *reinterpret_cast<uint32_t*>(to) = word;
          else
            *reinterpret_cast<uint16_t*>(to) = (uint16_t)word;
        }
        const int block = i / share;
        uint32_t four = i < wide ? step.byte << (8 * (block & 3)) : 0;
#pragma unroll
        for (int k = 1; k <= 2; ++k) {  // of four blocks, where the row has them in this group
          const uint32_t other = __shfl_xor_sync(0xffffffffu, four, k * share);
          if (k * share < lanes) four |= other;
        }
        if (inside && (i & (4 * share - 1)) == 0) put_scales(reinterpret_cast<uint8_t*>(p.scale), row, p.rows, block >> 2, p.blocks, four);
      }
    } else {
      uint8_t* const out = static_cast<uint8_t*>(p.y) + out_at;
      uint32_t m[V], before[RAGGED ? V : 1];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = first + v * lanes;
        m[v] = 0;
        if constexpr (RAGGED) before[v] = 0;
        if (i < nvec) {  // (beyond the row a NaN rstd would leave NaN in the zeros)
          frame.cut(s[v], i);
          float most_of = 0.f, most_before = 0.f;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float a = fabsf(s[v][e]);
            const bool early = RAGGED && e < frame.skew;
            most_of = larger(most_of, early ? 0.f : a);
            if constexpr (RAGGED) most_before = larger(most_before, early ? a : 0.f);
          }
          m[v] = magnitude(most_of);
          if constexpr (RAGGED) before[v] = magnitude(most_before);
        }
      }
      if (p.block == 0) {
        uint32_t all = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) all = RAGGED ? max(all, max(m[v], before[v])) : max(all, m[v]);
        all = WARP ? lanes_max(all, lanes) : cta_max(all, most);
        const Scale scale = scale_of(all, p.format);
        if (live && first == 0) p.scale[row] = scale.value;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int i = first + v * lanes;
          if (live && i < nvec) {
            over_each<VE>(s[v], scale);
            store_codes<VE, RAGGED>(out, frame, i, s[v], p.format);
          }
        }
      } else {
        // A block's vectors lie in neighbouring lanes: block / VE of them, at most a warp's.  In a frame the first of them begins with the
        // `skew` last channels of the block before: both parts of a block's maximum meet in shared memory, each written by one lane (the
        // row's sum has a barrier between two rows' use of it).  (4000 x 12345 fp16 over fp32 in blocks
        // of 128 takes 223 us.)
        const int share = p.block / VE, among = min(share, WARP ? lanes : 32), shift = 31 - __clz(share);
        uint2* const parts = blocks + (WARP ? (int)threadIdx.x / lanes * lanes : 0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int i = first + v * lanes;
          const bool leads = (i & (share - 1)) == 0;
          m[v] = lanes_max(RAGGED && !leads ? max(m[v], before[v]) : m[v], among);
          if (RAGGED && leads && i < nvec) parts[i >> shift] = make_uint2(m[v], before[v]);
        }
        if constexpr (RAGGED) at.meet();
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int i = first + v * lanes, block = i >> shift;
          if (live && i < nvec) {
            const bool leads = (i & (share - 1)) == 0;
            if (RAGGED && (block + 1) * share < nvec) m[v] = max(m[v], parts[block + 1].y);
            const Scale scale = scale_of(m[v], p.format);
            if (leads && (!RAGGED || block < p.blocks)) p.scale[row * p.blocks + block] = scale.value;  // (the last vector may hold the last block's end alone)
            if constexpr (RAGGED) {
              Scale early = scale;
              if (leads && block > 0) early = scale_of(max(parts[block - 1].x, before[v]), p.format);
#pragma unroll
              for (int e = 0; e < VE; ++e) s[v][e] = e < frame.skew ? over(s[v][e], early.inverse, early.back) : over(s[v][e], scale.inverse, scale.back);
            } else {
              over_each<VE>(s[v], scale);
            }
            store_codes<VE, RAGGED>(out, frame, i, s[v], p.format);
          }
        }
      }
    }
  }
  if constexpr (is_four(OUT)) clear_behind(reinterpret_cast<uint8_t*>(p.scale), p.rows, p.blocks, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
}

// Rows of any length: one CTA per row, element by element, read once for the sum and once more for each thing that needs it.  Outputs are
// stored in the last of these passes, by the thread that has just read the element: y and sum may be the inputs' own buffers.
template <typename Tx, typename Ts, bool Q>
__global__ void __launch_bounds__(kMostThreads, 4) rms_fwd_any_kernel(const RmsFwd p) {
  __shared__ TeamSlots slots;
  __shared__ uint32_t most[32];
  clear<false>(slots, blockDim.x, 0, threadIdx.x);
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
    }
    sq = team_sum<false>(sq, slots, turn, blockDim.x, 0);
    const float rstd = __frsqrt_rn(fmaf(sq, p.inv_c, p.eps));
    if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
    auto y_of = [&](int i, float s) { return s * rstd * (p.weight ? p.offset + param_at(p.weight, p.w_dtype, i, 1.f) : 1.f); };
    auto y_and_store_sum = [&](int i) {  // the last look at element i
      const float s = sum_at(i);
      if (r) static_cast<Ts*>(p.sum)[row * p.C + i] = store_param<Ts>(s);
      return y_of(i, s);
    };
    if constexpr (!Q) {
      for (int i = threadIdx.x; i < p.C; i += blockDim.x) static_cast<Tx*>(p.y)[row * p.C + i] = store_param<Tx>(y_and_store_sum(i));
    } else {
      uint8_t* out = static_cast<uint8_t*>(p.y) + row * p.C;
      if (p.block == 0) {
        uint32_t m = 0;
        for (int i = threadIdx.x; i < p.C; i += blockDim.x) m = max(m, magnitude(y_of(i, sum_at(i))));
        const Scale scale = scale_of(cta_max(m, most), p.format);
        if (threadIdx.x == 0) p.scale[row] = scale.value;
        for (int i = threadIdx.x; i < p.C; i += blockDim.x) out[i] = (uint8_t)code_of(over(y_and_store_sum(i), scale.inverse, scale.back), p.format);
      } else {  // one warp per block of at most 128 channels
        const int lane = threadIdx.x & 31, nwarps = blockDim.x >> 5;
        for (int b = threadIdx.x >> 5; b < p.blocks; b += nwarps) {
          float f[4];
          uint32_t m = 0;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int in = lane + 32 * v, i = b * p.block + in;
            f[v] = in < p.block && i < p.C ? y_and_store_sum(i) : 0.f;
            m = max(m, magnitude(f[v]));
          }
          const Scale scale = scale_of(lanes_max(m, 32), p.format);
          if (lane == 0) p.scale[row * p.blocks + b] = scale.value;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int in = lane + 32 * v, i = b * p.block + in;
            if (in < p.block && i < p.C) out[i] = (uint8_t)code_of(over(f[v], scale.inverse, scale.back), p.format);
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------------
// CTA sizes: the more rows a CTA takes at once, the fewer rows of partial sums there are to add up afterwards
constexpr int bwd_threads(int ve, int v) { return ve * v <= 8 ? 1024 : ve * v <= 16 ? 640 : 512; }

struct RmsBwd {
  const void *dy, *dsum, *sum, *addend, *weight;  // s = sum, or sum + addend (dy's type) where the stored sum was rounded to 16 bits
  const float* rstd;
  void *dx, *dsum_out;  // the same gradient in dy's type and, where sum has another type, in sum's
  float* part;          // one row of C floats per CTA, or NULL
  long long rows, dy_stride, ds_stride, s_stride, a_stride;
  int C, lanes, stages, stage_bytes, w_dtype;
  float offset, inv_c;
  int edge;  // as in RmsFwd
};

template <typename Tx, typename Ts, int VE, int V, int THREADS, bool RES, bool RAGGED>
__global__ void __launch_bounds__(bwd_threads(VE, V), 1) rms_bwd_kernel(const RmsBwd p) {
  constexpr bool WARP = THREADS == kWarpThreads, TEAMS = !WARP;
  extern __shared__ __align__(16) char smem[];
  __shared__ TeamSlots all_slots[TEAMS ? kMostTeams : 1];
  const Place<WARP, TEAMS> at(p.lanes, p.stage_bytes, p.stages, line_bytes(p.C, VE, RAGGED), smem);
  TeamSlots& slots = all_slots[TEAMS ? at.group : 0];
  const int lanes = at.lanes, first = at.first;
  grid_dep_launch_dependents();
  const Frame<VE, RAGGED> frame((uint32_t)(reinterpret_cast<uintptr_t>(static_cast<const Tx*>(p.dy) + at.row * p.dy_stride) / sizeof(Tx)), p.C);
  const int nvec = frame.nvec;
  const Tx *dy = static_cast<const Tx*>(p.dy) - frame.skew, *add = RES && p.addend ? static_cast<const Tx*>(p.addend) - frame.skew : nullptr;
  const Ts *ds = RES && p.dsum ? static_cast<const Ts*>(p.dsum) - frame.skew : nullptr, *sum = static_cast<const Ts*>(p.sum) - frame.skew;
  // a stage: sum, dy, then the addend and the sum's gradient where there are any
  const int narrow = segment_bytes(p.C, VE, sizeof(Tx), RAGGED), wide = segment_bytes(p.C, VE, sizeof(Ts), RAGGED);
  const int dy_at = wide, add_at = dy_at + narrow, ds_at = add_at + (add ? narrow : 0);
  long long asked = at.row;
  int ask_stage = 0, stage = 0;
  auto ask = [&]() {
    if (asked < p.rows) {
      const bool inner = asked >= p.edge && asked < p.rows - p.edge;
      char* s = at.stages + ask_stage * p.stage_bytes;
      ask_row<Ts, VE, V, RAGGED>(s, sum + asked * p.s_stride, frame, first, lanes, inner);
      ask_row<Tx, VE, V, RAGGED>(s + dy_at, dy + asked * p.dy_stride, frame, first, lanes, inner);
      if (add) ask_row<Tx, VE, V, RAGGED>(s + add_at, add + asked * p.a_stride, frame, first, lanes, inner);
      if (ds) ask_row<Ts, VE, V, RAGGED>(s + ds_at, ds + asked * p.ds_stride, frame, first, lanes, inner);
    }
    cp_async_commit();
    asked += at.step;
    ask_stage = ask_stage + 1 == p.stages ? 0 : ask_stage + 1;
  };
  for (int i = 0; i < p.stages; ++i) ask();
  float w[V][VE], dw[V][VE];
  fetch_weight<VE, V, RAGGED>(w, p.weight, p.w_dtype, p.offset, frame, first, lanes);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < VE; ++e) dw[v][e] = 0.f;
  if constexpr (!WARP) clear<TEAMS>(slots, at.lanes, at.group, first);
  int turn = 0;
  long long row = at.row;
  float rn = row < p.rows ? p.rstd[row] : 0.f;
  for (long long base = at.base; base < p.rows; base += at.step, row += at.step) {
    const bool live = !WARP || row < p.rows;
    const float rstd = rn;
    if (row + at.step < p.rows) rn = p.rstd[row + at.step];
    cp_async_wait_dyn8(p.stages - 1);
    const char* here = at.stages + stage * p.stage_bytes;
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    // s * rstd and dy of this thread's vector i
    auto terms = [&](int i, float (&n)[VE], float (&g)[VE]) {
      unpack<Ts, VE>(load_vec<Ts, VE>(reinterpret_cast<const Ts*>(here) + i * VE), n);
      unpack<Tx, VE>(load_vec<Tx, VE>(reinterpret_cast<const Tx*>(here + dy_at) + i * VE), g);
      if (add) {
        float f[VE];
        unpack<Tx, VE>(load_vec<Tx, VE>(reinterpret_cast<const Tx*>(here + add_at) + i * VE), f);
        add_each(n, f);
      }
      scale_each(n, rstd);
      frame.cut(n, i);
      frame.cut(g, i);
    };
    float dot[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (live && first + v * lanes < nvec) {
        float n[VE], g[VE];
        terms(first + v * lanes, n, g);
        mul_each(g, n);
        add_each(dw[v], g);
        if constexpr (RAGGED) {
          mul_each(g, w[v]);
          frame.lay_out(at.line, first + v * lanes, g);
        } else {
          dot_each(dot, g, w[v]);
        }
      }
    }
    if constexpr (RAGGED) {
      at.meet();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (live) {
          float f[VE];
          frame.take(at.line, v, first, lanes, f);
#pragma unroll
          for (int e = 0; e < VE; ++e) dot[e & 1] += f[e];
        }
      }
      at.part();
    }
    const float c = -(WARP ? lanes_sum(dot[0] + dot[1], lanes) : team_sum<TEAMS>(dot[0] + dot[1], slots, turn, at.lanes, at.group)) * p.inv_c;
    const long long out_at = row * p.C - frame.skew;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = first + v * lanes;
      if (live && i < nvec) {
        float n[VE], g[VE], d[VE];
        terms(i, n, g);
        mul_each(g, w[v]);
        axpy_each(g, n, c);
        scale_each(g, rstd);
        if (ds) {
          unpack<Ts, VE>(load_vec<Ts, VE>(reinterpret_cast<const Ts*>(here + ds_at) + i * VE), d);
          add_each(d, g);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) d[e] = g[e];
        }
        frame.store(static_cast<Tx*>(p.dx) + out_at, i, d);
        if constexpr (!std::is_same<Tx, Ts>::value)
          if (p.dsum_out) frame.store(static_cast<Ts*>(p.dsum_out) + out_at, i, d);
      }
    }
    ask();  // (a lane's own vectors: read, so free)
  }
  if (p.part == nullptr) return;
  // the groups hold the same channels: their sums are added in order.  They fit the stages, whose rows have two tensors of at least
  // two bytes an element.
  cp_async_wait<0>();
  __syncthreads();
  float* share = reinterpret_cast<float*>(smem);
  const int groups = (int)blockDim.x / lanes;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = first + v * lanes;
    if (i < nvec) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (frame.has(i, e)) share[at.group * p.C + frame.channel(i) + e] = dw[v][e];
    }
  }
  __syncthreads();
  float* part = p.part + (long long)blockIdx.x * p.C;
  for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
    float t = 0.f;
    for (int g = 0; g < groups; ++g) t += share[g * p.C + i];
    part[i] = t;
  }
}

// Rows of any length.  A thread fetches two elements before it uses the first, since no load may pass a store into what could be an input's own
// buffer (one at a time: 2000 x 33000 bf16 828 us, two 696, four 853).
constexpr int kAtOnce = 2;
template <typename Fetch, typename Use>
__device__ __forceinline__ void each_channel(int C, Fetch&& fetch, Use&& use) {
  for (int first = threadIdx.x; first < C; first += kAtOnce * (int)blockDim.x) {
    decltype(fetch(0)) v[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (first + k * (int)blockDim.x < C) v[k] = fetch(first + k * (int)blockDim.x);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (first + k * (int)blockDim.x < C) use(first + k * (int)blockDim.x, v[k]);
  }
}
template <typename Tx, typename Ts>
__global__ void __launch_bounds__(kMostThreads, 3) rms_bwd_any_kernel(const RmsBwd p) {
  __shared__ TeamSlots slots;
  clear<false>(slots, blockDim.x, 0, threadIdx.x);
  int turn = 0;
  grid_dep_launch_dependents();
  float* const part = p.part ? p.part + (long long)blockIdx.x * p.C : nullptr;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const Tx* dy = static_cast<const Tx*>(p.dy) + row * p.dy_stride;
    const Ts* sum = static_cast<const Ts*>(p.sum) + row * p.s_stride;
    const Ts* ds = p.dsum ? static_cast<const Ts*>(p.dsum) + row * p.ds_stride : nullptr;
    const Tx* add = p.addend ? static_cast<const Tx*>(p.addend) + row * p.a_stride : nullptr;
    const float rstd = p.rstd[row];
    struct Terms {
      float dy, g, n, ds, t;
    };
    auto terms_at = [&](int i) {
      Terms v;
      v.dy = load_param<Tx>(dy, i);
      v.g = v.dy * (p.weight ? p.offset + param_at(p.weight, p.w_dtype, i, 1.f) : 1.f);
      v.n = (load_param<Ts>(sum, i) + (add ? load_param<Tx>(add, i) : 0.f)) * rstd;
      return v;
    };
    auto all_at = [&](int i) {
      Terms v = terms_at(i);
      v.ds = ds ? load_param<Ts>(ds, i) : 0.f;
      v.t = part && row != blockIdx.x ? part[i] : 0.f;
      return v;
    };
    float dot = 0.f;
    each_channel(p.C, terms_at, [&](int, const Terms& v) { dot = fmaf(v.g, v.n, dot); });
    const float c = team_sum<false>(dot, slots, turn, blockDim.x, 0) * p.inv_c;
    each_channel(p.C, all_at, [&](int i, const Terms& v) {
      if (part) part[i] = fmaf(v.dy, v.n, v.t);
      const float d = fmaf(rstd, fmaf(-v.n, c, v.g), v.ds);
      static_cast<Tx*>(p.dx)[row * p.C + i] = store_param<Tx>(d);
      if constexpr (!std::is_same<Tx, Ts>::value)
        if (p.dsum_out) static_cast<Ts*>(p.dsum_out)[row * p.C + i] = store_param<Ts>(d);
    });
  }
}

// One warp-wide column block of 32 channels per CTA; the rows are dealt out to its warps, whose sums are added in order.
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps) column_sums_kernel(const ColumnSums p) {
  __shared__ float share[kSumWarps][32];
  const int per_set = (p.C + 31) / 32, set = (int)blockIdx.x / per_set;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = ((int)blockIdx.x - set * per_set) * 32 + lane;
  const float* part = p.part[set];
  const int rows = p.rows[set];
  grid_dep_wait();
  float t = 0.f;
  if (c < p.C) {
#pragma unroll 8
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
  int ve, v, lanes, threads;  // lanes: per row; threads: per CTA; v = 0: the kernels for rows of any length
  bool warp, ragged;          // warp: lanes of one warp; otherwise whole warps
  int most;                   // the kernel's limit of lanes
};

// How a call's rows lie: on vector boundaries, all in the same frame, or neither
enum Rows { kAligned, kRagged, kAny };

RmsGeom rms_geometry(int64_t C, int dtype, Rows rows, bool backward) {
  RmsGeom g = {};
  g.ve = dtype == GNB200_F32 ? 4 : 8;
  if (rows == kAny) return RmsGeom{1, 0, kMostThreads, kMostThreads, false, false, 0};
  g.ragged = rows == kRagged;
  const int64_t nvec = g.ragged ? (C + 2 * g.ve - 2) / g.ve : C / g.ve;  // (ragged: one more for rows that begin late in their frame)
  if (nvec <= 32 * 4) {  // four vectors a lane
    g.warp = true;
    g.lanes = 1;
    while (g.lanes < 32 && g.lanes < nvec) g.lanes *= 2;
    const int64_t each = (nvec + g.lanes - 1) / g.lanes;
    g.v = each <= 1 ? 1 : each <= 2 ? 2 : 4;
    g.most = kWarpThreads;
  } else {
    // two vectors a thread, and four of fp32 above 512 threads; the backward, with twice the registers, up to 640 threads, above them four
    // (eight of fp32) and 512.  (One vector a thread and more teams: the backward of 16384 x 4096 bf16 takes 131 us instead of 106.)
    const auto fits = [&](int v, int most) {
      if (nvec > (int64_t)v * most) return false;
      g.v = v;
      g.most = most;
      return true;
    };
    const int twice = g.ve == 4 ? 2 : 1;
    const bool any = backward ? fits(2, 512) || (g.ve == 4 && fits(4, 512)) || fits(2 * twice, 640) || fits(4 * twice, 512)
                              : fits(2, 512) || (g.ve == 4 && fits(4, 512)) || fits(2 * twice, 1024);
    if (!any) return rms_geometry(C, dtype, kAny, backward);
    g.lanes = (int)((nvec + g.v - 1) / g.v + 31) / 32 * 32;
  }
  g.threads = g.warp ? kWarpThreads : g.lanes;
  if (backward) {
    const int most = bwd_threads(g.ve, g.v);
    g.threads = g.warp ? most : std::max(1, std::min(kMostTeams, most / g.lanes)) * g.lanes;
  }
  return g;
}

constexpr int kMostStages = 4;  // of a row; two do as well where a row is 16 KB, eight are no faster anywhere

struct RmsLaunch {
  unsigned grid;
  int threads, smem, stages;
};
// CTA size, stages, shared memory and CTAs of a call whose rows take `row_bytes` in a stage (0: no stages) and `line` for their sums: no more CTAs than are resident at
// once nor than there are rows; where ragged rows take several turns, a number that
// keeps their frames.  cudaErrorInvalidValue: a row does not fit.
cudaError_t rms_launch(const void* kernel, const RmsGeom& g, int64_t rows, int64_t row_bytes, int64_t line, RmsLaunch* out) {
  Residency r = {};
  out->threads = g.threads;
  out->stages = 0;
  if (row_bytes + line > kMostDynamicSmem) return cudaErrorInvalidValue;
  out->smem = (int)(g.threads / g.lanes * line);
  if (row_bytes) {
    // fewer teams where two stages for each do not fit, or where there are no rows for them on every SM
    const auto halve = [&](int teams) { return g.warp ? teams / 2 : teams - 1; };
    int teams = g.threads / g.lanes;
    cudaError_t err = residency(kernel, g.threads, 0, &r);
    if (err != cudaSuccess) return err;
    const int least = g.warp ? 32 / g.lanes : 1;
    while (teams > least && (teams * (2 * row_bytes + line) > kMostDynamicSmem || (int64_t)teams * r.sms > rows)) teams = std::max(least, halve(teams));
    out->threads = teams * g.lanes;
    if ((err = residency(kernel, out->threads, 0, &r)) != cudaSuccess) return err;
    const int64_t bytes = row_bytes * teams, fixed = line * teams;
    if (bytes + fixed > kMostDynamicSmem) return cudaErrorInvalidValue;
    int64_t stages = std::max<int64_t>(1, (kMostDynamicSmem / r.per_sm - fixed) / bytes);
    stages = std::min<int64_t>(kMostStages, std::max<int64_t>(stages, std::min<int64_t>(2, (kMostDynamicSmem - fixed) / bytes)));
    const int64_t turns = (rows + (int64_t)teams * r.sms - 1) / ((int64_t)teams * r.sms);  // at most, of a team
    out->stages = (int)std::max<int64_t>(1, std::min(stages, turns));
    out->smem = (int)(bytes * out->stages + fixed);
  }
  const int cap = r.per_sm;
  const cudaError_t err = residency(kernel, out->threads, out->smem, &r);
  if (err != cudaSuccess) return err;
  if (row_bytes) r.per_sm = std::min(r.per_sm, cap);
  const int64_t per_cta = out->threads / g.lanes;
  const int64_t need = (rows + per_cta - 1) / per_cta, most = (int64_t)r.per_sm * r.sms;
  out->grid = (unsigned)(need < most ? need : most);
  if (g.ragged && need > most) {  // the step, per_cta * grid rows, becomes a multiple of VE
    int64_t grid = out->grid;
    while (grid > 1 && per_cta * grid % g.ve != 0) --grid;
    if (per_cta * grid % g.ve != 0) return cudaErrorInvalidValue;
    out->grid = (unsigned)grid;
  }
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
// ... and with the geometry's numbers: elements a vector, vectors a thread, the limit of threads, ragged?
template <int VE, bool BACK, typename F>
cudaError_t with_geometry(const RmsGeom& g, F&& f) {
  const auto ragged = [&](auto v, auto most) { return g.ragged ? f(Int<VE>(), v, most, std::true_type()) : f(Int<VE>(), v, most, std::false_type()); };
  if (g.warp) {
    if (g.v == 1) return ragged(Int<1>(), Int<kWarpThreads>());
    if (g.v == 2) return ragged(Int<2>(), Int<kWarpThreads>());
    return ragged(Int<4>(), Int<kWarpThreads>());
  }
  // (the backward's limit goes by its vectors)
  if constexpr (BACK) {
    if (g.v == 2) return ragged(Int<2>(), Int<512>());
    if (g.v == 4) return ragged(Int<4>(), Int<512>());
    if constexpr (VE == 4) return ragged(Int<8>(), Int<512>());
    return cudaErrorInvalidValue;
  } else {
    if constexpr (VE == 8) {
      return g.most == 512 ? ragged(Int<2>(), Int<512>()) : ragged(Int<2>(), Int<1024>());
    } else {
      if (g.v == 2) return ragged(Int<2>(), Int<512>());
      return g.most == 512 ? ragged(Int<4>(), Int<512>()) : ragged(Int<4>(), Int<1024>());
    }
  }
}

template <int OUT>
cudaError_t launch_rms_fwd(RmsFwd p, int dtype, int sum_dtype, Rows rows, cudaStream_t stream) {
  return with_types(dtype, sum_dtype, [&](auto tx, auto ts) {
    using Tx = decltype(tx);
    using Ts = decltype(ts);
    int64_t lanes_for = p.C;  // channels that a row's lanes have to do with
    if (is_four(OUT)) lanes_for = std::max<int64_t>(p.C, four_wide(p.C) - (rows == kRagged ? 2 * (16 / (int)sizeof(Tx)) - 2 : 0));
    RmsGeom g = rms_geometry(lanes_for, dtype, rows, false);
    bool staged = false;
    auto go = [&](void (*kernel)(const RmsFwd)) {
      RmsLaunch l = {};
      int row_bytes = 0;
      if (staged) row_bytes = segment_bytes(p.C, g.ve, sizeof(Tx), g.ragged) + (p.residual ? segment_bytes(p.C, g.ve, sizeof(Ts), g.ragged) : 0);
      const cudaError_t err = rms_launch((const void*)kernel, g, p.rows, row_bytes, g.v ? line_bytes(p.C, g.ve, g.ragged) : 0, &l);
      if (err != cudaSuccess) return err;
      p.lanes = g.lanes, p.stages = l.stages, p.stage_bytes = row_bytes;
      kernel<<<l.grid, l.threads, l.smem, stream>>>(p);
      return cudaGetLastError();
    };
    if (g.v) {
      const cudaError_t err = with_geometry<16 / (int)sizeof(Tx), false>(g, [&](auto ve, auto v, auto most, auto ragged) {
        constexpr int VE = decltype(ve)::value, V = decltype(v)::value, THREADS = decltype(most)::value;
        constexpr bool RAGGED = decltype(ragged)::value;
        staged = kStaged<Tx, Ts, VE, V, THREADS>;
        if constexpr (std::is_same<Tx, Ts>::value)
          if (!p.residual) return go(&rms_fwd_kernel<Tx, Ts, VE, V, THREADS, OUT, false, RAGGED>);
        return go(&rms_fwd_kernel<Tx, Ts, VE, V, THREADS, OUT, true, RAGGED>);
      });
      if (is_four(OUT) || err != cudaErrorInvalidValue) return err;
      g = RmsGeom{1, 0, kMostThreads, kMostThreads, false, false, 0};
      staged = false;
    }
    if constexpr (is_four(OUT))
      return cudaErrorInvalidValue;
    else
      return go(&rms_fwd_any_kernel<Tx, Ts, OUT == kCodes8>);
  });
}

// `grid`: the number of CTAs, that is of rows of partial sums.  With `room` (bytes of workspace) nothing is launched where they do not fit;
// kGridOnly: nothing at all.
constexpr size_t kGridOnly = ~(size_t)0;
cudaError_t launch_rms_bwd(RmsBwd p, int dtype, int sum_dtype, Rows rows, cudaStream_t stream, unsigned* grid, size_t room) {
  return with_types(dtype, sum_dtype, [&](auto tx, auto ts) {
    using Tx = decltype(tx);
    using Ts = decltype(ts);
    RmsGeom g = rms_geometry(p.C, dtype, rows, true);
    auto go = [&](void (*kernel)(const RmsBwd)) {
      RmsLaunch l = {};
      int row_bytes = 0;
      if (g.v)
        row_bytes = segment_bytes(p.C, g.ve, sizeof(Tx), g.ragged) * (p.addend ? 2 : 1) + segment_bytes(p.C, g.ve, sizeof(Ts), g.ragged) * (p.dsum ? 2 : 1);
      const cudaError_t err = rms_launch((const void*)kernel, g, p.rows, row_bytes, g.v ? line_bytes(p.C, g.ve, g.ragged) : 0, &l);
      if (err != cudaSuccess) return err;
      *grid = g.v ? l.grid : std::min(l.grid, (unsigned)std::max(1, (1 << 24) / p.C));  // 64 MB of partial sums at most, or one row
      if (room == kGridOnly || (p.part && (size_t)*grid * (size_t)p.C * sizeof(float) > room)) return cudaSuccess;
      p.lanes = g.lanes, p.stages = l.stages, p.stage_bytes = row_bytes;
      kernel<<<*grid, l.threads, l.smem, stream>>>(p);
      return cudaGetLastError();
    };
    if (g.v) {
      const cudaError_t err = with_geometry<16 / (int)sizeof(Tx), true>(g, [&](auto ve, auto v, auto most, auto ragged) {
        constexpr int VE = decltype(ve)::value, V = decltype(v)::value, THREADS = decltype(most)::value;
        constexpr bool RAGGED = decltype(ragged)::value;
        if constexpr (std::is_same<Tx, Ts>::value)
          if (!p.addend && !p.dsum) return go(&rms_bwd_kernel<Tx, Ts, VE, V, THREADS, false, RAGGED>);
        return go(&rms_bwd_kernel<Tx, Ts, VE, V, THREADS, true, RAGGED>);
      });
      if (err != cudaErrorInvalidValue) return err;
      g = RmsGeom{1, 0, kMostThreads, kMostThreads, false, false, 0};
    }
    return go(&rms_bwd_any_kernel<Tx, Ts>);
  });
}

// How the rows of a call's tensors lie together.  `width`: elements a vector.  Aligned: addresses and strides on vector boundaries, whole
// vectors a row.  In one frame: every tensor's first row begins as many elements behind a vector boundary, and its rows keep the distance of
// contiguous ones from such boundaries.
struct TensorRows {
  const void* p;  // NULL: not there
  int64_t stride;
  int size;
};
Rows rows_of(int width, int64_t C, int64_t rows, const void* weight, std::initializer_list<TensorRows> tensors) {
  bool aligned = C % width == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0, framed = true;
  int64_t skew = -1;
  for (const TensorRows& t : tensors) {
    if (!t.p) continue;
    const int64_t bytes = (int64_t)width * t.size, behind = (int64_t)(reinterpret_cast<uintptr_t>(t.p) % (uintptr_t)bytes);
    aligned = aligned && behind % std::min<int64_t>(bytes, 16) == 0 && (rows == 1 || t.stride % width == 0);
    framed = framed && behind % t.size == 0 && (skew < 0 || behind / t.size == skew) && (rows == 1 || (t.stride != 0 && (t.stride - C) % width == 0));
    if (skew < 0) skew = behind / t.size;
  }
  return aligned ? kAligned : framed ? kRagged : kAny;
}
int edge_of(int width, std::initializer_list<TensorRows> tensors) {
  int edge = 1;
  for (const TensorRows& t : tensors)
    if (t.p) edge = std::max(edge, edge_rows(width, t.stride));
  return edge;
}
int size_of(int dtype) { return dtype == GNB200_F32 ? 4 : 2; }
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

cudaError_t launch_rms_4bit(const FourNorm& n, cudaStream_t stream) {
  const int size = size_of(n.dtype), wide = size_of(n.residual_dtype), width = n.dtype == GNB200_F32 ? 4 : 8;
  const Rows how = rows_of(width, n.C, n.rows, n.weight, {{n.x, n.x_stride, size}, {n.residual, n.r_stride, wide}, {n.sum, n.C, wide}});
  if (how == kAny) return cudaErrorInvalidValue;
  RmsFwd p = {};
  p.x = n.x, p.residual = n.residual, p.weight = n.weight, p.y = n.codes, p.sum = n.sum;
  p.rstd = const_cast<float*>(n.tensor_scale), p.scale = reinterpret_cast<float*>(n.scales);
  p.rows = n.rows, p.x_stride = n.x_stride, p.r_stride = n.r_stride;
  p.C = n.C, p.w_dtype = n.weight_dtype, p.block = n.block, p.blocks = (int)four_tiles(n.C, n.block);
  p.eps = (float)n.eps, p.offset = (float)n.offset, p.inv_c = (float)(1.0 / (double)n.C);
  p.edge = edge_of(width, {{n.x, n.x_stride, size}, {n.residual, n.r_stride, wide}});
  return n.block == 16 ? launch_rms_fwd<kCodes4Of16>(p, n.dtype, n.residual_dtype, how, stream) : launch_rms_fwd<kCodes4Of32>(p, n.dtype, n.residual_dtype, how, stream);
}

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
  const int size = size_of(dtype), wide = size_of(residual_dtype);
  const int width = dtype == GNB200_F32 ? 4 : 8;
  const Rows how = rows_of(width, C, rows, weight,
                           {{x, x_stride, size}, {residual, residual_stride, wide}, {y, C, codes ? 1 : size}, {sum, C, wide}});
  p.edge = edge_of(width, {{x, x_stride, size}, {residual, residual_stride, wide}});
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launched(name, codes ? launch_rms_fwd<kCodes8>(p, dtype, residual_dtype, how, s)
                              : launch_rms_fwd<kPlain>(p, dtype, residual_dtype, how, s));
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
  static thread_local Remembered<4> known;  // the answer depends on nothing but these and the device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const Remembered<4>::Key key = {rows, C, dtype * 4 + sum_dtype, dev};
  if (const size_t* v = known.find(key)) return *v;
  RmsBwd p = {};
  p.rows = rows, p.C = (int)C;
  size_t most = 0;
  const int width = dtype == GNB200_F32 ? 4 : 8;
  for (int kind = 0; kind < 12; ++kind) {  // whichever kernel and stages the call's tensors will ask for (none of these is read)
    p.addend = kind & 1 ? &p : nullptr;
    p.dsum = kind & 2 ? &p : nullptr;
    const Rows how = kind < 4 ? kAligned : kind < 8 ? kRagged : kAny;
    if (how == kAligned && C % width != 0) continue;
    unsigned grid = 0;
    if (launch_rms_bwd(p, dtype, sum_dtype, how, nullptr, &grid, kGridOnly) != cudaSuccess) return 0;
    const size_t need = (size_t)grid * (size_t)C * sizeof(float);
    most = need > most ? need : most;
  }
  return known.keep(key, most);
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
  const int size = size_of(dtype), wide = size_of(sum_dtype);
  const int width = dtype == GNB200_F32 ? 4 : 8;
  p.edge = edge_of(width, {{dy, dy_stride, size}, {dsum, dsum_stride, wide}, {sum, sum_stride, wide}, {addend, addend_stride, size}});
  const Rows how = rows_of(width, C, rows, weight,
                           {{dy, dy_stride, size}, {dsum, dsum_stride, wide}, {sum, sum_stride, wide}, {addend, addend_stride, size},
                            {dx, C, size}, {dsum_out, C, wide}});
  unsigned grid = 0;
  if (dweight) {
    if (!workspace) return report_error(GNB200_ERR_WORKSPACE, "%s: a gradient of the weight without a workspace", name);
    p.part = static_cast<float*>(workspace);
  }
  cudaError_t err = launch_rms_bwd(p, dtype, sum_dtype, how, s, &grid, workspace_bytes);
  const size_t need = (size_t)grid * (size_t)C * sizeof(float);
  if (err == cudaSuccess && dweight && need > workspace_bytes)
    return report_error(GNB200_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu are needed", name, workspace_bytes, need);
  if (err == cudaSuccess && dweight) err = launch_column_sums(ColumnSums{{p.part}, {dweight}, {(int)grid}, (int)C, weight_dtype}, 1, s, true);
  return launched(name, err);
}

}  // extern "C"
