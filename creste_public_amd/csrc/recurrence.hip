// Gated linear recurrence over time, per sequence b and channel c, f = sigmoid(gate), u = 1 - f, state in fp32:
//   h_t = f_t h_(t-1) + u_t x_t
// and its reverse:  e_t = f_t (dh_t + e_(t+1))  with e_T = dh_last;  delta_t = dh_t + e_(t+1);  dx_t = u_t delta_t;
//   dgate_t = delta_t (h_(t-1) - x_t) f_t u_t;  dh0 = e_0.
// Both are first-order linear maps of the carried value, so a run of steps is one pair (A, B): out = A in + B.
// Layout.  Lanes = channels (VEC neighbours each, (b, c) flattened), the 8 waves of a workgroup = consecutive runs of LR steps held in
// registers and joined through LDS: a workgroup takes one chunk of 8 * LR steps of 64 * VEC columns with ONE pass over its data.
// Chunks of one column group meet by look-back: a workgroup publishes its chunk's (A, B), fetches those of the chunks in front of
// it in its window of 16 and the value carried into the window (published by the window in front), the 8 waves two each at once.
// Always the same pairs in the same order, whoever is ready first: results do not depend on timing.
// Chunks are handed out by tickets, so one only ever waits for chunks that started earlier: every wait ends.  Each published word
// is 8 bytes written at once, valid when not zero -- (-A, B): A >= 0, so the sign bit marks it -- hence no fences.  (The spin is
// bounded all the same: past the bound the columns become NaN.)
// The backward recomputes h inside a chunk from the chunk's starting state, which the forward saves (4 bytes per 64 steps).
// Steps behind a sequence's length have f = 1, u = 0, dh = 0: states and cotangents pass through unchanged.
// Bound: HBM (forward 3 elements, backward 5 per step and channel), a single step: launch latency.  Measured, 4 x 16384 x 1024
// bf16: forward 93 us (4.3 TB/s), backward 179 us (3.7 TB/s; a large copy: 5.1); two passes over the data with a launch between
// them took 176 and 280.  Flags that a single lane polls, or windows of windows to shorten the chain, were slower (more round trips).
#include "common.h"

namespace creste {

// steps a wave holds: 16 in the forward (4 x 16384 x 1024 bf16: 100 us against 121 with 8: half as many workgroups to meet), 8 in the
// backward, whose 16 would leave one workgroup per CU (191 us against 183)
constexpr int kRecWaves = 8, kRecRunF = 16, kRecRunB = 8;
constexpr int kRecChunkB = kRecRunB * kRecWaves;                     // the backward's chunk: one saved state each

struct RecArgs {
  const void *gate, *x, *gh;
  int64_t g_sb, g_st, x_sb, x_st, h_sb, h_st;
  const float *h0, *gh_last;
  const int64_t* lengths;
  int64_t T, C, BC;
  int chunks, groups;
  void *h, *ggate, *gx;
  float *h_last, *starts, *gh0;
  unsigned* ticket;                             // [groups][16]; zeroed, as the words below
  uint64_t *pair, *known;                       // [chunks][BC] (-A, B) of a chunk; [chunks / 16][BC] (carried value behind a window, 1)
};

constexpr int kRecSpin = 1 << 22, kRecWindow = 16, kRecTicket = 16;

__device__ __forceinline__ uint64_t rec_word(unsigned lo, float hi) { return (uint64_t)__float_as_uint(hi) << 32 | lo; }
__device__ __forceinline__ uint64_t rec_get(const uint64_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void rec_put(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// f = sigmoid(g), u = 1 - f; the exponential's rounded argument leaves the smaller of the two (2 + 1.5 |g|) 2^-24 off, relatively, the
// larger a few 2^-24 (hardware exponential and reciprocal: a full division would cost as much as the rest of a step)
__device__ __forceinline__ void rec_gate(float g, float& f, float& u) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * fabsf(g)), r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
  f = g >= 0.f ? r : s;
  u = g >= 0.f ? s : r;
}

// outputs are written past the caches and leave their room to the inputs (4 x 16384 x 1024 bf16: forward 103 -> 93 us, backward
// 184 -> 179 us)
template <typename V>
__device__ __forceinline__ void rec_store(V* p, V v) { __builtin_nontemporal_store(v, p); }

template <typename T, int VEC>
struct RecVec { typedef T type __attribute__((ext_vector_type(VEC))); };

// column -> (b, c); columns of a lane are VEC neighbours of one sequence
template <int VEC>
struct RecCol {
  int64_t col, b, c, len;
  bool on;
  __device__ __forceinline__ RecCol(const RecArgs& p, int group) {
    col = ((int64_t)group * 64 + threadIdx.x) * VEC;
    on = col < p.BC;
    if (!on) col = p.BC - VEC;                  // a copy of the last column; it stores nothing
    b = col / p.C;
    c = col - b * p.C;
    len = p.T;
    if (p.lengths) {
      len = p.lengths[b];
      len = len < 0 ? 0 : len > p.T ? p.T : len;
    }
  }
};

// steps of the run t0 .. t0 + LR - 1 in front of `len`
template <int LR>
__device__ __forceinline__ int rec_live(int64_t t0, int64_t len) {
  const int64_t n = len - t0;
  return n < 0 ? 0 : n > LR ? LR : (int)n;
}

// which (column group, chunk in the order of the recurrence) this workgroup takes.  One counter per group, a cache line each: chunks
// wait within their group only
__device__ __forceinline__ void rec_ticket(const RecArgs& p, int& group, int& turn) {
  group = blockIdx.x % p.groups;
  turn = 0;
  if (p.chunks == 1) return;
  __shared__ unsigned t;
  if (threadIdx.x == 0 && threadIdx.y == 0) t = atomicAdd(p.ticket + (int64_t)group * kRecTicket, 1u);
  __syncthreads();
  turn = __builtin_amdgcn_readfirstlane((int)t);
}

// s (on entry the value in front of the first chunk) <- the value carried into this chunk.  (A, B): this chunk's pair.  turn = the
// chunk's place in the order of the recurrence.  All threads of the workgroup call and get the result
template <int VEC>
__device__ __forceinline__ void rec_lookback(const RecArgs& p, const RecCol<VEC>& k, int turn, const float (&A)[VEC],
                                             const float (&B)[VEC], float (&s)[VEC]) {
  __shared__ float2 sh[kRecWindow][64 * VEC];
  __shared__ float carried[64 * VEC];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.y), at_w = turn % kRecWindow, base = turn - at_w;
  const bool last = at_w == kRecWindow - 1;
  if (w == 0 && k.on && !last)                  // (nobody asks for the pair of a window's last chunk)
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      rec_put(p.pair + (int64_t)turn * p.BC + k.col + e, rec_word(__float_as_uint(A[e]) | 0x80000000u, B[e]));
  // wave w fetches the pairs number w, w + 8, .. of the window, the last wave the value carried into the window
  constexpr int PQ = kRecWindow / kRecWaves;
  const uint64_t* src[PQ + 1];
#pragma unroll
  for (int q = 0; q <= PQ; ++q) src[q] = nullptr;
#pragma unroll
  for (int q = 0; q < PQ; ++q)
    if (w + kRecWaves * q < at_w) src[q] = p.pair + (int64_t)(base + w + kRecWaves * q) * p.BC + k.col;
  if (w == kRecWaves - 1 && base > 0) src[PQ] = p.known + (int64_t)(base / kRecWindow - 1) * p.BC + k.col;
  uint64_t v[PQ + 1][VEC];
  for (int spin = 0;; ++spin) {
    bool all = true;
#pragma unroll
    for (int q = 0; q <= PQ; ++q)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[q][e] = src[q] ? rec_get(src[q] + e) : 1;
#pragma unroll
    for (int q = 0; q <= PQ; ++q)
#pragma unroll
      for (int e = 0; e < VEC; ++e) all &= v[q][e] != 0;
    if (__all(all)) break;
    if (spin == kRecSpin) {
#pragma unroll
      for (int q = 0; q <= PQ; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[q][e] = rec_word(0x7fc00000u, __builtin_nanf(""));
      break;
    }
    __builtin_amdgcn_s_sleep(1);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
#pragma unroll
    for (int q = 0; q < PQ; ++q)
      if (src[q])
        sh[w + kRecWaves * q][threadIdx.x * VEC + e] =
            make_float2(__uint_as_float((unsigned)v[q][e] & 0x7fffffffu), __uint_as_float((unsigned)(v[q][e] >> 32)));
    if (src[PQ]) carried[threadIdx.x * VEC + e] = __uint_as_float((unsigned)(v[PQ][e] >> 32));
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (base > 0) s[e] = carried[threadIdx.x * VEC + e];
    for (int j = 0; j < at_w; ++j) {
      const float2 q = sh[j][threadIdx.x * VEC + e];
      s[e] = fmaf(q.x, s[e], q.y);
    }
    if (last && w == 0 && k.on) rec_put(p.known + (int64_t)(turn / kRecWindow) * p.BC + k.col + e, rec_word(1u, fmaf(A[e], s[e], B[e])));
  }
}

template <typename T, int VEC, int LR>
__global__ __launch_bounds__(512, 4) void rec_forward_kernel(RecArgs p) {
  typedef typename RecVec<T, VEC>::type vec;
  __shared__ float2 sh[kRecWaves][64 * VEC];
  int group, ch;
  rec_ticket(p, group, ch);
  const RecCol<VEC> k(p, group);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.y), nw = blockDim.y;
  const int64_t t0 = ((int64_t)ch * nw + w) * LR;
  const T *gp = (const T*)p.gate + k.b * p.g_sb + k.c, *xp = (const T*)p.x + k.b * p.x_sb + k.c;
  vec gv[LR], xv[LR];
#pragma unroll
  for (int i = 0; i < LR; ++i) {
    const int64_t t = t0 + i < p.T ? t0 + i : p.T - 1;
    gv[i] = *reinterpret_cast<const vec*>(gp + t * p.g_st);
    xv[i] = *reinterpret_cast<const vec*>(xp + t * p.x_st);
  }
  float s[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = p.h0 ? p.h0[k.col + e] : 0.f;
  const int live = rec_live<LR>(t0, k.len);     // steps of this run in front of the sequence's end
  const bool whole = __all(live == LR);
  float f[LR][VEC], b[LR][VEC], A[VEC], B[VEC];
#pragma unroll
  for (int i = 0; i < LR; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float u;
      rec_gate((float)gv[i][e], f[i][e], u);
      b[i][e] = u * (float)xv[i][e];
    }
  if (!whole)
#pragma unroll
    for (int i = 0; i < LR; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[i][e] = i < live ? f[i][e] : 1.f;
        b[i][e] = i < live ? b[i][e] : 0.f;
      }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    A[e] = 1.f;
    B[e] = 0.f;
#pragma unroll
    for (int i = 0; i < LR; ++i) {
      A[e] *= f[i][e];
      B[e] = fmaf(f[i][e], B[e], b[i][e]);
    }
  }
  float wa[VEC], wb[VEC];                       // pair of the runs in front of this wave's
#pragma unroll
  for (int e = 0; e < VEC; ++e) { wa[e] = 1.f; wb[e] = 0.f; }
  if (nw > 1) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) sh[w][threadIdx.x * VEC + e] = make_float2(A[e], B[e]);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float ca = 1.f, cb = 0.f;
      for (int j = 0; j < nw; ++j) {
        const float2 v = sh[j][threadIdx.x * VEC + e];
        if (j == w) { wa[e] = ca; wb[e] = cb; }
        cb = fmaf(v.x, cb, v.y);
        ca *= v.x;
      }
      A[e] = ca;
      B[e] = cb;
    }
  }
  if constexpr (LR > 1)
    if (p.chunks > 1) rec_lookback<VEC>(p, k, ch, A, B, s);
  if (w == 0 && k.on && ch == p.chunks - 1)
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.h_last[k.col + e] = fmaf(A[e], s[e], B[e]);
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = fmaf(wa[e], s[e], wb[e]);
  if (p.starts && k.on && (LR == 1 || t0 % kRecChunkB == 0) && t0 < p.T)
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.starts[t0 / kRecChunkB * p.BC + k.col + e] = s[e];
  T* hp = (T*)p.h + (k.b * p.T) * p.C + k.c;
#pragma unroll
  for (int i = 0; i < LR; ++i) {
    vec o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      s[e] = fmaf(f[i][e], s[e], b[i][e]);
      o[e] = (T)(i < live ? s[e] : 0.f);
    }
    if (k.on && t0 + i < p.T) rec_store(reinterpret_cast<vec*>(hp + (t0 + i) * p.C), o);
  }
}

template <typename T, int VEC, int LR>
__global__ __launch_bounds__(512, 4) void rec_backward_kernel(RecArgs p) {
  typedef typename RecVec<T, VEC>::type vec;
  __shared__ float2 sh[kRecWaves][64 * VEC], fw[kRecWaves][64 * VEC];
  int group, turn;
  rec_ticket(p, group, turn);
  const int ch = p.chunks - 1 - turn;
  const RecCol<VEC> k(p, group);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.y), nw = blockDim.y;
  const int64_t t0 = ((int64_t)ch * nw + w) * LR;
  const T *gp = (const T*)p.gate + k.b * p.g_sb + k.c, *xp = (const T*)p.x + k.b * p.x_sb + k.c;
  const T* dp = (const T*)p.gh + k.b * p.h_sb + k.c;
  vec gv[LR], xv[LR], dv[LR];
#pragma unroll
  for (int i = 0; i < LR; ++i) {
    const int64_t t = t0 + i < p.T ? t0 + i : p.T - 1;
    gv[i] = *reinterpret_cast<const vec*>(gp + t * p.g_st);
    dv[i] = *reinterpret_cast<const vec*>(dp + t * p.h_st);
    xv[i] = *reinterpret_cast<const vec*>(xp + t * p.x_st);
  }
  float st[VEC], s[VEC];                        // h in front of the chunk; e behind it
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    st[e] = p.starts[(int64_t)ch * p.BC + k.col + e];
    s[e] = p.gh_last ? p.gh_last[k.col + e] : 0.f;
  }
  const int live = rec_live<LR>(t0, k.len);
  const bool whole = __all(live == LR);
  float f[LR][VEC], u[LR][VEC], x[LR][VEC], d[LR][VEC], A[VEC], B[VEC], wa[VEC], wb[VEC];
#pragma unroll
  for (int i = 0; i < LR; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      rec_gate((float)gv[i][e], f[i][e], u[i][e]);
      x[i][e] = (float)xv[i][e];
      d[i][e] = (float)dv[i][e];
    }
  if (!whole)
#pragma unroll
    for (int i = 0; i < LR; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[i][e] = i < live ? f[i][e] : 1.f;
        u[i][e] = i < live ? u[i][e] : 0.f;
        x[i][e] = i < live ? x[i][e] : 0.f;
        d[i][e] = i < live ? d[i][e] : 0.f;
      }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float a = 1.f, b = 0.f, h = 0.f;            // (a, b): e through the run, (a, h): the state
#pragma unroll
    for (int i = LR - 1; i >= 0; --i) {
      b = f[i][e] * (d[i][e] + b);
      a *= f[i][e];
    }
#pragma unroll
    for (int i = 0; i < LR; ++i) h = fmaf(f[i][e], h, u[i][e] * x[i][e]);
    A[e] = a; B[e] = b;
    wa[e] = 1.f; wb[e] = 0.f;
    if (nw > 1) {
      sh[w][threadIdx.x * VEC + e] = make_float2(a, b);
      fw[w][threadIdx.x * VEC + e] = make_float2(a, h);
    }
  }
  if (nw > 1) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float ca = 1.f, cb = 0.f;
      for (int j = nw - 1; j >= 0; --j) {
        const float2 v = sh[j][threadIdx.x * VEC + e];
        if (j == w) { wa[e] = ca; wb[e] = cb; }
        cb = fmaf(v.x, cb, v.y);
        ca *= v.x;
      }
      A[e] = ca;
      B[e] = cb;
      for (int j = 0; j < w; ++j) {
        const float2 v = fw[j][threadIdx.x * VEC + e];
        st[e] = fmaf(v.x, st[e], v.y);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {               // x <- (h_(t-1) - x_t) f_t u_t, all that dgate needs besides delta
#pragma unroll
    for (int i = 0; i < LR; ++i) {
      const float h = st[e];
      st[e] = fmaf(f[i][e], h, u[i][e] * x[i][e]);
      x[i][e] = (h - x[i][e]) * (f[i][e] * u[i][e]);
    }
  }
  if constexpr (LR > 1)
    if (p.chunks > 1) rec_lookback<VEC>(p, k, turn, A, B, s);
  if (w == 0 && k.on && ch == 0 && p.gh0)
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.gh0[k.col + e] = fmaf(A[e], s[e], B[e]);
#pragma unroll
  for (int e = 0; e < VEC; ++e) s[e] = fmaf(wa[e], s[e], wb[e]);
  T* ggp = (T*)p.ggate + (k.b * p.T) * p.C + k.c;
  T* gxp = (T*)p.gx + (k.b * p.T) * p.C + k.c;
#pragma unroll
  for (int i = LR - 1; i >= 0; --i) {
    vec og, ox;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {             // (behind the end: u = 0 and d = 0, so both are 0 and e passes)
      const float delta = d[i][e] + s[e];
      og[e] = (T)(i < live ? delta * x[i][e] : 0.f);
      ox[e] = (T)(i < live ? delta * u[i][e] : 0.f);
      s[e] = f[i][e] * delta;
    }
    if (k.on && t0 + i < p.T) {
      rec_store(reinterpret_cast<vec*>(ggp + (t0 + i) * p.C), og);
      rec_store(reinterpret_cast<vec*>(gxp + (t0 + i) * p.C), ox);
    }
  }
}

__global__ __launch_bounds__(256) void rec_zero_kernel(uint4* __restrict__ p, int64_t n) {
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) p[i] = make_uint4(0, 0, 0, 0);
}

namespace {

int64_t rec_chunks(int64_t T) { return (T + kRecChunkB - 1) / kRecChunkB; }     // the smaller of the two chunks

// The workspace, all zero at the start: a ticket line per column group (sized as if a lane took one column), the published pairs
// and values; a multiple of 16 bytes in all, none for a single chunk
int64_t rec_tickets(int64_t BC) { return (BC + 63) / 64 * kRecTicket * 4; }
int64_t rec_work(int64_t BC, int64_t chunks) {
  return chunks == 1 ? 0 : rec_tickets(BC) + ((chunks + chunks / kRecWindow) * BC + 1) / 2 * 16;
}

template <typename T, int VEC, int LF, int LB>
int rec_launch(RecArgs& p, bool bwd, char* work, hipStream_t s) {
  const int LR = bwd ? LB : LF;
  const int64_t groups = (p.BC / VEC + 63) / 64;
  int64_t nw = (p.T + LR - 1) / LR;
  nw = nw > kRecWaves ? kRecWaves : nw;
  const int64_t chunks = (p.T + nw * LR - 1) / (nw * LR);
  CRESTE_REQUIRE(groups * chunks * 64 < (1ll << 32), "gated_recurrence: too many columns and chunks of steps for a launch (2^26 workgroups)");
  p.chunks = (int)chunks;
  p.groups = (int)groups;
  if (chunks > 1) {
    const int64_t n = rec_work(p.BC, chunks) / 16, nb = (n + 255) / 256;
    p.ticket = (unsigned*)work;
    p.pair = (uint64_t*)(work + rec_tickets(p.BC));
    p.known = p.pair + chunks * p.BC;
    rec_zero_kernel<<<(int)(nb > 2048 ? 2048 : nb), 256, 0, s>>>((uint4*)work, n);
    CRESTE_CHECK_LAUNCH("gated_recurrence zero");
  }
  const dim3 grid((unsigned)(groups * chunks)), block(64, (unsigned)nw);
  if (bwd) rec_backward_kernel<T, VEC, LB><<<grid, block, 0, s>>>(p);
  else rec_forward_kernel<T, VEC, LF><<<grid, block, 0, s>>>(p);
  CRESTE_CHECK_LAUNCH("gated_recurrence");
  return CRESTE_OK;
}

template <typename T>
int rec_typed(RecArgs& p, bool bwd, char* work, hipStream_t s) {
  // two channels per lane where every row starts on a boundary of two elements
  const uintptr_t ptrs = (uintptr_t)p.gate | (uintptr_t)p.x | (uintptr_t)p.gh | (uintptr_t)p.h | (uintptr_t)p.ggate | (uintptr_t)p.gx;
  const int64_t strides = p.C | p.g_sb | p.g_st | p.x_sb | p.x_st | p.h_sb | p.h_st;
  const bool two = (ptrs & (2 * sizeof(T) - 1)) == 0 && (strides & 1) == 0;
  if (p.T == 1) return two ? rec_launch<T, 2, 1, 1>(p, bwd, work, s) : rec_launch<T, 1, 1, 1>(p, bwd, work, s);
  return two ? rec_launch<T, 2, kRecRunF, kRecRunB>(p, bwd, work, s) : rec_launch<T, 1, kRecRunF, kRecRunB>(p, bwd, work, s);
}

int rec_run(RecArgs& p, int dtype, bool bwd, char* work, hipStream_t s) {
  if (dtype == CRESTE_DT_F32) return rec_typed<float>(p, bwd, work, s);
  if (dtype == CRESTE_DT_BF16) return rec_typed<__bf16>(p, bwd, work, s);
  if (dtype == CRESTE_DT_F16) return rec_typed<_Float16>(p, bwd, work, s);
  set_error("gated_recurrence: dtype %d", dtype);
  return CRESTE_ERR_ARG;
}

bool rec_work_ok(const void* work, int64_t bytes, int64_t B, int64_t T, int64_t C) {
  const int64_t need = rec_work(B * C, rec_chunks(T));
  return need == 0 || (work && ((uintptr_t)work & 15) == 0 && bytes >= need);
}

int rec_check(int64_t B, int64_t T, int64_t C) {
  CRESTE_REQUIRE(B > 0 && T > 0 && C > 0 && B < (1ll << 31) && C < (1ll << 31) && B * C < (1ll << 40) && T < (1ll << 36),
                 "gated_recurrence: B %lld T %lld C %lld", (long long)B, (long long)T, (long long)C);
  return CRESTE_OK;
}

}  // namespace
}  // namespace creste

using namespace creste;

extern "C" int creste_gated_recurrence_chunk_steps(void) { return kRecChunkB; }

extern "C" int64_t creste_gated_recurrence_workspace_bytes(int64_t B, int64_t T, int64_t C) {
  if (B <= 0 || T <= 0 || C <= 0 || B >= (1ll << 31) || C >= (1ll << 31) || B * C >= (1ll << 40) || T >= (1ll << 36)) return -1;
  return rec_work(B * C, rec_chunks(T));
}

extern "C" int creste_gated_recurrence_forward(const void* gate, int64_t gate_sb, int64_t gate_st, const void* x, int64_t x_sb,
                                               int64_t x_st, const float* h0, const int64_t* lengths, int64_t B, int64_t T,
                                               int64_t C, int dtype, void* h, float* h_last, float* starts, void* work,
                                               int64_t work_bytes, void* stream) {
  const int rc = rec_check(B, T, C);
  if (rc) return rc;
  CRESTE_REQUIRE(gate && x && h && h_last && rec_work_ok(work, work_bytes, B, T, C),
                 "gated_recurrence_forward: null pointer or workspace of %lld bytes", (long long)work_bytes);
  RecArgs p{};
  p.gate = gate; p.g_sb = gate_sb; p.g_st = gate_st;
  p.x = x; p.x_sb = x_sb; p.x_st = x_st;
  p.h0 = h0; p.lengths = lengths;
  p.T = T; p.C = C; p.BC = B * C;
  p.h = h; p.h_last = h_last; p.starts = starts;
  return rec_run(p, dtype, false, (char*)work, (hipStream_t)stream);
}

extern "C" int creste_gated_recurrence_backward(const void* gate, int64_t gate_sb, int64_t gate_st, const void* x, int64_t x_sb,
                                                int64_t x_st, const void* gh, int64_t gh_sb, int64_t gh_st,
                                                const float* gh_last, const int64_t* lengths, const float* starts, int64_t B,
                                                int64_t T, int64_t C, int dtype, void* ggate, void* gx, float* gh0, void* work,
                                                int64_t work_bytes, void* stream) {
  const int rc = rec_check(B, T, C);
  if (rc) return rc;
  CRESTE_REQUIRE(gate && x && gh && starts && ggate && gx && rec_work_ok(work, work_bytes, B, T, C),
                 "gated_recurrence_backward: null pointer or workspace of %lld bytes", (long long)work_bytes);
  RecArgs p{};
  p.gate = gate; p.g_sb = gate_sb; p.g_st = gate_st;
  p.x = x; p.x_sb = x_sb; p.x_st = x_st;
  p.gh = gh; p.h_sb = gh_sb; p.h_st = gh_st;
  p.gh_last = gh_last; p.lengths = lengths; p.starts = const_cast<float*>(starts);
  p.T = T; p.C = C; p.BC = B * C;
  p.ggate = ggate; p.gx = gx; p.gh0 = gh0;
  return rec_run(p, dtype, true, (char*)work, (hipStream_t)stream);
}
