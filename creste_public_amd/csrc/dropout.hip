// Dropout whose mask is a function of (seed, offset, element) and never stored:
//   word_i = Philox4x32-10(counter = (i div 4, offset), key = seed)[i mod 4]   (Salmon et al., SC 2011)
//   y_i = word_i >= round(p 2^32) ? x_i / (1 - p) : 0   (+ residual_i);  the backward is the same call on the cotangent.
// A dropped element is SELECTED away, so an infinity or NaN there does not reach the output.  fp32 arithmetic, one rounding.
// Bound: HBM.  40 M fp32 elements: 53 us, 6.0 TB/s; 34 M bf16 with a residual: 31 us, 6.5 TB/s (part of it from the cache; a large
// copy: 5.1).  The generator's 20 wide multiplies per four elements stay below that.
#include "common.h"

namespace creste {

typedef _Float16 drh;
typedef __bf16 drb;

struct DropArgs {
  const void *x, *res;
  void* y;
  int64_t n;
  unsigned threshold;
  float scale;
  uint64_t seed, offset;
  const int64_t* state;
};

// four words for counter block `i`
__device__ __forceinline__ void philox4(uint64_t i, uint64_t offset, uint64_t seed, unsigned (&w)[4]) {
  unsigned c0 = (unsigned)i, c1 = (unsigned)(i >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
    c1 = (unsigned)p1;
    c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
    c3 = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// VE elements per thread and step; VE > 1 needs pointers aligned to VE elements
template <typename T, int VE>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs p) {
  typedef T vec __attribute__((ext_vector_type(VE)));
  const uint64_t seed = p.state ? (uint64_t)p.state[0] : p.seed, off = p.offset + (p.state ? (uint64_t)p.state[1] : 0);
  const T *x = (const T*)p.x, *res = (const T*)p.res;
  T* y = (T*)p.y;
  const int64_t nv = (p.n + VE - 1) / VE;
  for (int64_t v = blockIdx.x * 256LL + threadIdx.x; v < nv; v += gridDim.x * 256LL) {
    const int64_t i0 = v * VE;
    const bool full = i0 + VE <= p.n;
    float a[VE], r[VE];
    if (full) {
      const vec xv = *reinterpret_cast<const vec*>(x + i0);
#pragma unroll
      for (int e = 0; e < VE; ++e) a[e] = (float)xv[e];
      if (res) {
        const vec rv = *reinterpret_cast<const vec*>(res + i0);
#pragma unroll
        for (int e = 0; e < VE; ++e) r[e] = (float)rv[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        a[e] = i0 + e < p.n ? (float)x[i0 + e] : 0.f;
        r[e] = res && i0 + e < p.n ? (float)res[i0 + e] : 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < (VE + 3) / 4; ++q) {
      unsigned w[4];
      philox4((uint64_t)(i0 >> 2) + q, off, seed, w);
#pragma unroll
      for (int e = 4 * q; e < 4 * q + 4 && e < VE; ++e) {
        const unsigned word = VE >= 4 ? w[e & 3] : (i0 & 3) == 0 ? w[0] : (i0 & 3) == 1 ? w[1] : (i0 & 3) == 2 ? w[2] : w[3];
        const float d = word >= p.threshold ? a[e] * p.scale : 0.f;
        a[e] = res ? d + r[e] : d;
      }
    }
    if (full) {
      vec yv;
#pragma unroll
      for (int e = 0; e < VE; ++e) yv[e] = (T)a[e];
      // past the caches: 160 MB fp32 57 -> 53 us, 67 MB bf16 with a residual 34 -> 31 us
      __builtin_nontemporal_store(yv, reinterpret_cast<vec*>(y + i0));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (i0 + e < p.n) y[i0 + e] = (T)a[e];
    }
  }
}

// p = 0: every element is kept (threshold 0); p rounding to 2^32: none is, which no 32-bit threshold says
template <typename T>
__global__ __launch_bounds__(256) void dropout_all_kernel(DropArgs p) {
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < p.n; i += gridDim.x * 256LL)
    ((T*)p.y)[i] = p.res ? ((const T*)p.res)[i] : (T)0;
}

template <typename T, int VE>
int dropout_launch(const DropArgs& a, bool all, hipStream_t s) {
  const bool vec = (((uintptr_t)a.x | (uintptr_t)a.res | (uintptr_t)a.y) & (VE * sizeof(T) - 1)) == 0;
  auto grid = [](int64_t items) { const int64_t b = (items + 255) / 256; return (int)(b > 8192 ? 8192 : b); };
  if (all) dropout_all_kernel<T><<<grid(a.n), 256, 0, s>>>(a);
  else if (vec) dropout_kernel<T, VE><<<grid((a.n + VE - 1) / VE), 256, 0, s>>>(a);
  else dropout_kernel<T, 1><<<grid(a.n), 256, 0, s>>>(a);
  CRESTE_CHECK_LAUNCH("dropout");
  return CRESTE_OK;
}

}  // namespace creste

using namespace creste;

extern "C" int creste_dropout(const void* x, const void* residual, void* y, int64_t n, int dtype, double p, int64_t seed,
                              int64_t offset, const int64_t* state, void* stream) {
  CRESTE_REQUIRE(x && y && n > 0, "dropout: bad args");
  CRESTE_REQUIRE(p >= 0. && p <= 1., "dropout: p = %g outside [0, 1]", p);
  const double t = nearbyint(p * 4294967296.);
  DropArgs a{x, residual, y, n, (unsigned)(t > 4294967295. ? 4294967295. : t), (float)(p < 1. ? 1. / (1. - p) : 0.),
             (uint64_t)seed, (uint64_t)offset, state};
  const bool all = t > 4294967295.;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == CRESTE_DT_F32) return dropout_launch<float, 4>(a, all, s);
  if (dtype == CRESTE_DT_BF16) return dropout_launch<drb, 8>(a, all, s);
  if (dtype == CRESTE_DT_F16) return dropout_launch<drh, 8>(a, all, s);
  set_error("dropout: dtype %d", dtype);
  return CRESTE_ERR_ARG;
}
