// Gated linear recurrence over time, per sequence b and channel c, f = sigmoid(gate), u = 1 - f, state in fp32:
//   h_t = f_t h_(t-1) + u_t x_t
// and its reverse:  e_t = f_t (dh_t + e_(t+1))  with e_T = dh_last;  delta_t = dh_t + e_(t+1);  dx_t = u_t delta_t;
//   dgate_t = delta_t (h_(t-1) - x_t) f_t u_t;  dh0 = e_0.
// Both are first-order linear maps of the carried value, so a run of steps is one pair (A, B): out = A in + B.
// Layout.  Lanes = channels (VEC neighbours each, (b, c) flattened), waves of a workgroup = consecutive runs of LR steps held in
// registers, joined through LDS: a workgroup takes a chunk of 8 * LR steps with one pass over its data, and walks its segment of the
// time axis chunk by chunk, carrying the state.  With enough (b, c) columns one segment covers all of T and everything is read once.
// With few, the time axis is split into segments: a first launch leaves each segment's (A, B) (forward: gate and x read twice;
// backward: gate and dh), the second joins the segments in front of its own.
// The backward recomputes h inside a chunk from the chunk's starting state, which the forward saves (4 bytes per 8 * LR steps).
// Steps behind a sequence's length have f = 1, u = 0, dh = 0: states and cotangents pass through unchanged.
// Bound: HBM (forward 3 elements, backward 5 per step and channel), a single step: launch latency.
#include "common.h"

namespace creste {

constexpr int kRecRun = 8, kRecWaves = 8, kRecChunk = kRecRun * kRecWaves;

struct RecArgs {
  const void *gate, *x, *gh;
  int64_t g_sb, g_st, x_sb, x_st, h_sb, h_st;
  const float *h0, *gh_last;
  const int64_t* lengths;
  int64_t T, C, BC;
  int chunks, seg_chunks, segs;
  void *h, *ggate, *gx;
  float *h_last, *starts, *gh0;
  float2* agg;                                  // [segs][BC] (A, B) of a segment
};

// f = sigmoid(g), u = 1 - f, both to full relative accuracy
__device__ __forceinline__ void rec_gate(float g, float& f, float& u) {
  const float e = __expf(-fabsf(g)), r = 1.f / (1.f + e), s = e * r;
  f = g >= 0.f ? r : s;
  u = g >= 0.f ? s : r;
}

template <typename T, int VEC>
struct RecVec { typedef T type __attribute__((ext_vector_type(VEC))); };

// column -> (b, c); columns of a lane are VEC neighbours of one sequence
template <int VEC>
struct RecCol {
  int64_t col, b, c, len;
  bool on;
  __device__ __forceinline__ RecCol(const RecArgs& p) {
    col = ((int64_t)blockIdx.x * 64 + threadIdx.x) * VEC;
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

// AGG: leave the segment's (A, B) only
template <typename T, int VEC, int LR, bool AGG>
__global__ __launch_bounds__(512) void rec_forward_kernel(RecArgs p) {
  typedef typename RecVec<T, VEC>::type vec;
  __shared__ float2 sh[kRecWaves][64 * VEC];
  const RecCol<VEC> k(p);
  const int w = threadIdx.y, nw = blockDim.y, seg = blockIdx.y;
  const T* gp = (const T*)p.gate + k.b * p.g_sb + k.c;
  const T* xp = (const T*)p.x + k.b * p.x_sb + k.c;
  float s[VEC], sa[VEC];                        // carried state; AGG: carried (A, B)
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    s[e] = !AGG && p.h0 ? p.h0[k.col + e] : 0.f;
    sa[e] = 1.f;
  }
  if constexpr (!AGG)
    for (int j = 0; j < seg; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 v = p.agg[(int64_t)j * p.BC + k.col + e];
        s[e] = fmaf(v.x, s[e], v.y);
      }
  const int c0 = seg * p.seg_chunks, c1 = min(p.chunks, c0 + p.seg_chunks);
  for (int ch = c0; ch < c1; ++ch) {
    const int64_t t0 = ((int64_t)ch * nw + w) * LR;
    vec gv[LR], xv[LR];
#pragma unroll
    for (int i = 0; i < LR; ++i) {
      const int64_t t = t0 + i < p.T ? t0 + i : p.T - 1;
      gv[i] = *reinterpret_cast<const vec*>(gp + t * p.g_st);
      xv[i] = *reinterpret_cast<const vec*>(xp + t * p.x_st);
    }
    float f[LR][VEC], b[LR][VEC], A[VEC], B[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 1.f; B[e] = 0.f; }
#pragma unroll
    for (int i = 0; i < LR; ++i) {
      const bool live = t0 + i < k.len;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float u;
        rec_gate((float)gv[i][e], f[i][e], u);
        f[i][e] = live ? f[i][e] : 1.f;
        b[i][e] = live ? u * (float)xv[i][e] : 0.f;
        A[e] *= f[i][e];
        B[e] = fmaf(f[i][e], B[e], b[i][e]);
      }
    }
    if (nw > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) sh[w][threadIdx.x * VEC + e] = make_float2(A[e], B[e]);
      __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (!AGG)
        if (w == 0 && p.starts && k.on) p.starts[(int64_t)ch * p.BC + k.col + e] = s[e];
      float mine = s[e];                        // state in front of this wave's run
      for (int j = 0; j < nw; ++j) {
        const float2 v = nw > 1 ? sh[j][threadIdx.x * VEC + e] : make_float2(A[e], B[e]);
        if (j == w) mine = s[e];
        s[e] = fmaf(v.x, s[e], v.y);
        if constexpr (AGG) sa[e] *= v.x;
      }
      if constexpr (!AGG) {
#pragma unroll
        for (int i = 0; i < LR; ++i) {
          mine = fmaf(f[i][e], mine, b[i][e]);
          b[i][e] = mine;
        }
      }
    }
    if constexpr (!AGG) {
      T* hp = (T*)p.h + (k.b * p.T) * p.C + k.c;
#pragma unroll
      for (int i = 0; i < LR; ++i) {
        vec o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = (T)(t0 + i < k.len ? b[i][e] : 0.f);
        if (k.on && t0 + i < p.T) *reinterpret_cast<vec*>(hp + (t0 + i) * p.C) = o;
      }
    }
    if (nw > 1) __syncthreads();
  }
  if (w == 0 && k.on) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (AGG) p.agg[(int64_t)seg * p.BC + k.col + e] = make_float2(sa[e], s[e]);
      else if (seg == p.segs - 1) p.h_last[k.col + e] = s[e];
    }
  }
}

template <typename T, int VEC, int LR, bool AGG>
__global__ __launch_bounds__(512) void rec_backward_kernel(RecArgs p) {
  typedef typename RecVec<T, VEC>::type vec;
  __shared__ float2 sh[kRecWaves][64 * VEC], fw[AGG ? 1 : kRecWaves][64 * VEC];
  const RecCol<VEC> k(p);
  const int w = threadIdx.y, nw = blockDim.y, seg = blockIdx.y;
  const T* gp = (const T*)p.gate + k.b * p.g_sb + k.c;
  const T* xp = (const T*)p.x + k.b * p.x_sb + k.c;
  const T* dp = (const T*)p.gh + k.b * p.h_sb + k.c;
  float s[VEC], sa[VEC];                        // e carried from the later steps
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    s[e] = !AGG && p.gh_last ? p.gh_last[k.col + e] : 0.f;
    sa[e] = 1.f;
  }
  if constexpr (!AGG)
    for (int j = p.segs - 1; j > seg; --j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 v = p.agg[(int64_t)j * p.BC + k.col + e];
        s[e] = fmaf(v.x, s[e], v.y);
      }
  const int c0 = seg * p.seg_chunks, c1 = min(p.chunks, c0 + p.seg_chunks);
  for (int ch = c1 - 1; ch >= c0; --ch) {
    const int64_t t0 = ((int64_t)ch * nw + w) * LR;
    vec gv[LR], xv[LR], dv[LR];
    float st[VEC];
#pragma unroll
    for (int i = 0; i < LR; ++i) {
      const int64_t t = t0 + i < p.T ? t0 + i : p.T - 1;
      gv[i] = *reinterpret_cast<const vec*>(gp + t * p.g_st);
      if constexpr (!AGG) xv[i] = *reinterpret_cast<const vec*>(xp + t * p.x_st);
      dv[i] = *reinterpret_cast<const vec*>(dp + t * p.h_st);
    }
    if constexpr (!AGG)
#pragma unroll
      for (int e = 0; e < VEC; ++e) st[e] = p.starts[(int64_t)ch * p.BC + k.col + e];
    float f[LR][VEC], u[LR][VEC];
#pragma unroll
    for (int i = 0; i < LR; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        rec_gate((float)gv[i][e], f[i][e], u[i][e]);
        if (t0 + i >= k.len) { f[i][e] = 1.f; u[i][e] = 0.f; }
      }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float A = 1.f, B = 0.f;
#pragma unroll
      for (int i = LR - 1; i >= 0; --i) {
        const float d = t0 + i < k.len ? (float)dv[i][e] : 0.f;
        B = f[i][e] * (d + B);
        A *= f[i][e];
      }
      sh[w][threadIdx.x * VEC + e] = make_float2(A, B);
      if constexpr (!AGG) {
        float H = 0.f;                          // the forward pair of the run: (A, H)
#pragma unroll
        for (int i = 0; i < LR; ++i) H = fmaf(f[i][e], H, u[i][e] != 0.f ? u[i][e] * (float)xv[i][e] : 0.f);
        fw[w][threadIdx.x * VEC + e] = make_float2(A, H);
      }
    }
    if (nw > 1) __syncthreads();
    float mine[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      for (int j = nw - 1; j >= 0; --j) {
        const float2 v = sh[j][threadIdx.x * VEC + e];
        if (j == w) mine[e] = s[e];
        s[e] = fmaf(v.x, s[e], v.y);
        if constexpr (AGG) sa[e] *= v.x;
      }
      if constexpr (!AGG)
        for (int j = 0; j < w; ++j) {
          const float2 v = fw[j][threadIdx.x * VEC + e];
          st[e] = fmaf(v.x, st[e], v.y);
        }
    }
    if constexpr (!AGG) {
      float hp[LR][VEC];                        // h_(t-1)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
#pragma unroll
        for (int i = 0; i < LR; ++i) {
          hp[i][e] = st[e];
          st[e] = fmaf(f[i][e], st[e], u[i][e] != 0.f ? u[i][e] * (float)xv[i][e] : 0.f);
        }
      T* ggp = (T*)p.ggate + (k.b * p.T) * p.C + k.c;
      T* gxp = (T*)p.gx + (k.b * p.T) * p.C + k.c;
#pragma unroll
      for (int i = LR - 1; i >= 0; --i) {
        vec og, ox;
        const bool live = t0 + i < k.len;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = (live ? (float)dv[i][e] : 0.f) + mine[e];
          og[e] = (T)(live ? d * (hp[i][e] - (float)xv[i][e]) * (f[i][e] * u[i][e]) : 0.f);
          ox[e] = (T)(live ? d * u[i][e] : 0.f);
          mine[e] = f[i][e] * d;
        }
        if (k.on && t0 + i < p.T) {
          *reinterpret_cast<vec*>(ggp + (t0 + i) * p.C) = og;
          *reinterpret_cast<vec*>(gxp + (t0 + i) * p.C) = ox;
        }
      }
    }
    if (nw > 1) __syncthreads();
  }
  if (w == 0 && k.on) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (AGG) p.agg[(int64_t)seg * p.BC + k.col + e] = make_float2(sa[e], s[e]);
      else if (seg == 0 && p.gh0) p.gh0[k.col + e] = s[e];
    }
  }
}

namespace {

// segments: one while the columns alone give >= 512 workgroups, else enough for ~1024, at most one per chunk and at most 64 (every
// workgroup reads the pairs of the segments in front of it)
int rec_segments(int64_t BC, int64_t chunks) {
  const int64_t groups = (BC + 63) / 64;
  if (groups >= 512 || chunks < 2) return 1;
  int64_t s = 1024 / groups;
  s = s > chunks ? chunks : s;
  return (int)(s > 64 ? 64 : s < 1 ? 1 : s);
}

template <typename T, int VEC, int LR>
int rec_launch(RecArgs& p, bool bwd, hipStream_t s) {
  const int64_t groups = (p.BC / VEC + 63) / 64;
  CRESTE_REQUIRE(groups < (1ll << 31), "gated_recurrence: too many columns");
  int64_t nw = (p.T + LR - 1) / LR;
  nw = nw > kRecWaves ? kRecWaves : nw;
  p.chunks = (int)((p.T + nw * LR - 1) / (nw * LR));
  int segs = LR == 1 ? 1 : rec_segments(p.BC, p.chunks);
  p.seg_chunks = (p.chunks + segs - 1) / segs;
  p.segs = (p.chunks + p.seg_chunks - 1) / p.seg_chunks;
  const dim3 grid((unsigned)groups, p.segs), block(64, (unsigned)nw);
  if (p.segs > 1) {
    if (bwd) rec_backward_kernel<T, VEC, LR, true><<<grid, block, 0, s>>>(p);
    else rec_forward_kernel<T, VEC, LR, true><<<grid, block, 0, s>>>(p);
    CRESTE_CHECK_LAUNCH("gated_recurrence segments");
  }
  if (bwd) rec_backward_kernel<T, VEC, LR, false><<<grid, block, 0, s>>>(p);
  else rec_forward_kernel<T, VEC, LR, false><<<grid, block, 0, s>>>(p);
  CRESTE_CHECK_LAUNCH("gated_recurrence");
  return CRESTE_OK;
}

template <typename T>
int rec_typed(RecArgs& p, bool bwd, hipStream_t s) {
  // two channels per lane where every row starts on a boundary of two elements
  const uintptr_t ptrs = (uintptr_t)p.gate | (uintptr_t)p.x | (uintptr_t)p.gh | (uintptr_t)p.h | (uintptr_t)p.ggate | (uintptr_t)p.gx;
  const int64_t strides = p.C | p.g_sb | p.g_st | p.x_sb | p.x_st | p.h_sb | p.h_st;
  const bool two = (ptrs & (2 * sizeof(T) - 1)) == 0 && (strides & 1) == 0;
  if (p.T == 1) return two ? rec_launch<T, 2, 1>(p, bwd, s) : rec_launch<T, 1, 1>(p, bwd, s);
  return two ? rec_launch<T, 2, kRecRun>(p, bwd, s) : rec_launch<T, 1, kRecRun>(p, bwd, s);
}

int rec_run(RecArgs& p, int dtype, bool bwd, hipStream_t s) {
  if (dtype == CRESTE_DT_F32) return rec_typed<float>(p, bwd, s);
  if (dtype == CRESTE_DT_BF16) return rec_typed<__bf16>(p, bwd, s);
  if (dtype == CRESTE_DT_F16) return rec_typed<_Float16>(p, bwd, s);
  set_error("gated_recurrence: dtype %d", dtype);
  return CRESTE_ERR_ARG;
}

int rec_check(int64_t B, int64_t T, int64_t C) {
  CRESTE_REQUIRE(B > 0 && T > 0 && C > 0 && B < (1ll << 31) && C < (1ll << 31) && B * C < (1ll << 40) && T < (1ll << 36),
                 "gated_recurrence: B %lld T %lld C %lld", (long long)B, (long long)T, (long long)C);
  return CRESTE_OK;
}

}  // namespace
}  // namespace creste

using namespace creste;

extern "C" int creste_gated_recurrence_chunk_steps(void) { return kRecChunk; }

extern "C" int64_t creste_gated_recurrence_workspace_bytes(int64_t B, int64_t T, int64_t C) {
  if (B <= 0 || T <= 0 || C <= 0 || B >= (1ll << 31) || C >= (1ll << 31) || B * C >= (1ll << 40) || T >= (1ll << 36)) return -1;
  return rec_segments(B * C, (T + kRecChunk - 1) / kRecChunk) * B * C * (int64_t)sizeof(float2) + 16;
}

extern "C" int creste_gated_recurrence_forward(const void* gate, int64_t gate_sb, int64_t gate_st, const void* x, int64_t x_sb,
                                               int64_t x_st, const float* h0, const int64_t* lengths, int64_t B, int64_t T,
                                               int64_t C, int dtype, void* h, float* h_last, float* starts, void* work,
                                               int64_t work_bytes, void* stream) {
  const int rc = rec_check(B, T, C);
  if (rc) return rc;
  CRESTE_REQUIRE(gate && x && h && h_last && work && work_bytes >= creste_gated_recurrence_workspace_bytes(B, T, C),
                 "gated_recurrence_forward: null pointer or workspace of %lld bytes", (long long)work_bytes);
  RecArgs p{};
  p.gate = gate; p.g_sb = gate_sb; p.g_st = gate_st;
  p.x = x; p.x_sb = x_sb; p.x_st = x_st;
  p.h0 = h0; p.lengths = lengths;
  p.T = T; p.C = C; p.BC = B * C;
  p.h = h; p.h_last = h_last; p.starts = starts; p.agg = (float2*)work;
  return rec_run(p, dtype, false, (hipStream_t)stream);
}

extern "C" int creste_gated_recurrence_backward(const void* gate, int64_t gate_sb, int64_t gate_st, const void* x, int64_t x_sb,
                                                int64_t x_st, const void* gh, int64_t gh_sb, int64_t gh_st,
                                                const float* gh_last, const int64_t* lengths, const float* starts, int64_t B,
                                                int64_t T, int64_t C, int dtype, void* ggate, void* gx, float* gh0, void* work,
                                                int64_t work_bytes, void* stream) {
  const int rc = rec_check(B, T, C);
  if (rc) return rc;
  CRESTE_REQUIRE(gate && x && gh && starts && ggate && gx && work &&
                     work_bytes >= creste_gated_recurrence_workspace_bytes(B, T, C),
                 "gated_recurrence_backward: null pointer or workspace of %lld bytes", (long long)work_bytes);
  RecArgs p{};
  p.gate = gate; p.g_sb = gate_sb; p.g_st = gate_st;
  p.x = x; p.x_sb = x_sb; p.x_st = x_st;
  p.gh = gh; p.h_sb = gh_sb; p.h_st = gh_st;
  p.gh_last = gh_last; p.lengths = lengths; p.starts = const_cast<float*>(starts);
  p.T = T; p.C = C; p.BC = B * C;
  p.ggate = ggate; p.gx = gx; p.gh0 = gh0; p.agg = (float2*)work;
  return rec_run(p, dtype, true, (hipStream_t)stream);
}
