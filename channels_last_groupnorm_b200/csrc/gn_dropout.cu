// Dropout with the residual's addition, its mask made from a counter wherever it is needed and never stored:
//
//   s_i = r_i + (k_i ? x_i / (1 - p) : 0)       in fp32, rounded once;   backward  dx_i = k_i ? ds_i / (1 - p) : 0,  dr = ds
//   k_i: word i % 4 of Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011) is at least p 2^32; counter (i / 4, layer), 64 bits each, key the seed
//
// i counts the elements in order, so that the mask depends neither on layout nor on the grid.  A dropped element is zero whatever it was.
#include <algorithm>

#include "../../include/gnb200.h"
#include "gn_kernels.h"
#include "gn_tokens.cuh"

namespace gnb200 {
namespace {

constexpr long long kNear = 1ll << 33;  // elements up to which 32 bits count the counters, the grid's last steps included

struct DropoutArgs {
  const void *in, *residual;
  void* out;
  const unsigned long long* seed_at;  // on the device, or NULL: `seed`
  unsigned long long seed, layer;
  long long n;
  uint32_t least;  // kept from this word on
  float scale;
};

// Four words of Philox 4x32-10.  The keys of the rounds are in registers: what is left of a round is two products of 64 bits and two xors.
struct Philox {
  uint32_t k0[10], k1[10], l0, l1;
  __device__ __forceinline__ Philox(unsigned long long seed, unsigned long long layer) {
    l0 = (uint32_t)layer, l1 = (uint32_t)(layer >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) k0[round] = (uint32_t)seed + round * 0x9E3779B9u, k1[round] = (uint32_t)(seed >> 32) + round * 0xBB67AE85u;
  }
  template <typename I>  // (of 32 bits: the counter's high word is zero, and with it the first two rounds have half their products from the layer alone)
  __device__ __forceinline__ void words(I at, uint32_t (&w)[4]) const {
    uint32_t a = (uint32_t)at, b = sizeof(I) == 8 ? (uint32_t)((unsigned long long)at >> 32) : 0u, c = l0, d = l1;
#pragma unroll
    for (int round = 0; round < 10; ++round) {
      const unsigned long long left = (unsigned long long)a * 0xD2511F53u, right = (unsigned long long)c * 0xCD9E8D57u;
      a = (uint32_t)(right >> 32) ^ b ^ k0[round], b = (uint32_t)right;
      c = (uint32_t)(left >> 32) ^ d ^ k1[round], d = (uint32_t)left;
    }
    w[0] = a, w[1] = b, w[2] = c, w[3] = d;
  }
};

// acc + x * scale where the word is large enough, else acc; x * scale or zero
__device__ __forceinline__ float add_kept(float acc, float x, float scale, uint32_t word, uint32_t least) {
  asm("{\n\t.reg .pred p;\n\tsetp.hs.u32 p, %3, %4;\n\t@p fma.rn.f32 %0, %1, %2, %0;\n\t}" : "+f"(acc) : "f"(x), "f"(scale), "r"(word), "r"(least));
  return acc;
}

// Vectors of 16 bytes of the wider type, 8 elements or 4, and 16 elements that a thread has under way: four chains of products hide their latency.
template <typename Ti, typename To>
constexpr int kVector = sizeof(Ti) == 4 || sizeof(To) == 4 ? 4 : 8;
// Threads of a CTA at most: 16384 x 4096 bf16 with and without a residual 69.5 and 65 us with 256, 65 and 62 with 512, 64.5 and 60 with 1024; fp32 127, 124.5, 141.
// Small calls take 256, to reach more SMs.
template <typename Ti, typename To>
constexpr int kMostThreads = kVector<Ti, To> == 8 ? 1024 : 512;
constexpr int kFewThreads = 256;

// VEC: tensors begin on vector boundaries and are taken a vector at a time, but for their end; otherwise element by element.  I: an index of counters.
// What a thread needs from memory is asked for in front of its words and unpacked behind them (unpacked in front: bf16 with a residual 83 us, so 66).
// Bound by HBM with a residual (16384 x 4096 bf16 61 us of 61, fp32 123 of 123); without one, in 16 bits, by the products: 56 us of 41.
template <typename Ti, typename To, bool RES, bool VEC, typename I>
__global__ void __launch_bounds__(kMostThreads<Ti, To>) dropout_kernel(const DropoutArgs p) {
  constexpr int VE = kVector<Ti, To>, AT_ONCE = VEC ? 16 / VE : 1;
  const Ti* in = static_cast<const Ti*>(p.in);
  const To* res = static_cast<const To*>(p.residual);
  To* out = static_cast<To*>(p.out);
  const Philox philox(p.seed_at ? *p.seed_at : p.seed, p.layer);
  const I vectors = (I)((p.n + VE - 1) / VE), step = gridDim.x * blockDim.x;
  const float scale = p.scale;
  const uint32_t least = p.least;
  for (I v = blockIdx.x * blockDim.x + threadIdx.x; v < vectors; v += AT_ONCE * step) {
    Pack<Ti, VE> x[AT_ONCE];
    Pack<To, VE> r[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const long long first = (long long)(v + k * step) * VE;
      if (VEC && first + VE <= p.n) {
        x[k] = load_vec<Ti, VE>(in + first);
        if constexpr (RES) r[k] = load_vec<To, VE>(res + first);
      }
    }
    uint32_t w[AT_ONCE][VE / 4][4];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
      for (int c = 0; c < VE / 4; ++c) philox.words<I>(VE / 4 * (v + k * step) + c, w[k][c]);
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const long long first = (long long)(v + k * step) * VE;
      if (VEC && first + VE <= p.n) {
        float f[VE], sum[VE];
        unpack<Ti, VE>(x[k], f);
        if constexpr (RES) unpack<To, VE>(r[k], sum);
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] = add_kept(RES ? sum[e] : 0.f, f[e], scale, w[k][e / 4][e % 4], least);
        store_vec<To, VE>(out + first, pack<To, VE>(sum));
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e)
          if (first + e < p.n)
            out[first + e] = store_param<To>(add_kept(RES ? load_param<To>(res + first, e) : 0.f, load_param<Ti>(in + first, e), scale, w[k][e / 4][e % 4], least));
      }
    }
  }
}

template <typename F>
cudaError_t with_type(int dtype, F&& f) {
  if (dtype == GNB200_F32) return f(float());
  if (dtype == GNB200_F16) return f(__half());
  return f(__nv_bfloat16());
}
bool dtype_ok(int d) { return d == GNB200_F32 || d == GNB200_F16 || d == GNB200_BF16; }
bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename Ti, typename To, bool RES>
cudaError_t launch_dropout(const DropoutArgs& p, cudaStream_t stream) {
  const auto go = [&](void (*kernel)(const DropoutArgs)) {
    constexpr int VE = kVector<Ti, To>, most = kMostThreads<Ti, To>;
    Residency r = {};
    cudaError_t err = residency((const void*)kernel, most, 0, &r);
    if (err != cudaSuccess) return err;
    const long long vectors = (p.n + VE - 1) / VE;
    const int threads = vectors >= (long long)r.per_sm * r.sms * most ? most : kFewThreads;
    if (threads != most && (err = residency((const void*)kernel, threads, 0, &r)) != cudaSuccess) return err;
    kernel<<<(unsigned)std::min<long long>((vectors + threads - 1) / threads, (long long)r.per_sm * r.sms), threads, 0, stream>>>(p);
    return cudaGetLastError();
  };
  const bool vec = on16(p.in) && on16(p.residual) && on16(p.out);  // (8 bytes do for the narrow side of two types)
  if (p.n < kNear) return vec ? go(&dropout_kernel<Ti, To, RES, true, uint32_t>) : go(&dropout_kernel<Ti, To, RES, false, uint32_t>);
  return vec ? go(&dropout_kernel<Ti, To, RES, true, unsigned long long>) : go(&dropout_kernel<Ti, To, RES, false, unsigned long long>);
}

}  // namespace
}  // namespace gnb200

using namespace gnb200;

extern "C" int gnb200_dropout_add(const void* x, const void* residual, int64_t n, double p, const int64_t* seed_at, uint64_t seed, uint64_t layer, int dtype,
                                  int out_dtype, void* out, void* stream) {
  const char* name = "gnb200_dropout_add";
  if (!dtype_ok(dtype) || !dtype_ok(out_dtype)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if (dtype != out_dtype && dtype != GNB200_F32 && out_dtype != GNB200_F32)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: the types of the input and the output are the same, or one is float32", name);
  if (residual && dtype == GNB200_F32 && out_dtype != GNB200_F32)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: a residual has the type of x or float32", name);
  if (n < 0) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: the number of elements must not be negative (got %lld)", name, (long long)n);
  const double word = p * 4294967296.0;
  if (!(p >= 0.0) || !(word < 4294967295.5)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: p is at least 0 and less than 1 (got %g)", name, p);
  if (n == 0) return GNB200_OK;
  if (!x || !out) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  DropoutArgs a = {};
  a.in = x, a.residual = residual, a.out = out, a.seed_at = reinterpret_cast<const unsigned long long*>(seed_at), a.seed = seed, a.layer = layer, a.n = n;
  a.least = (uint32_t)(word + 0.5), a.scale = (float)(1.0 / (1.0 - p));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = with_type(dtype, [&](auto ti) {
    return with_type(out_dtype, [&](auto to) {
      using Ti = decltype(ti);
      using To = decltype(to);
      if constexpr (std::is_same<Ti, To>::value || std::is_same<To, float>::value) {
        return residual ? launch_dropout<Ti, To, true>(a, s) : launch_dropout<Ti, To, false>(a, s);
      } else if constexpr (std::is_same<Ti, float>::value) {
        return launch_dropout<Ti, To, false>(a, s);
      } else {
        return cudaErrorInvalidValue;
      }
    });
  });
  if (err != cudaSuccess) return report_error(GNB200_ERR_CUDA, "%s: CUDA error: %s", name, cudaGetErrorString(err));
  return GNB200_OK;
}
