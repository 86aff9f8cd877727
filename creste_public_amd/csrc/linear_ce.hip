// Softmax cross entropy over a large set of classes, straight from the features, without the logits in memory:
//   z_ij = (x_i . w_j) / tau,  lse_i = log sum_j exp z_ij,  nll_i = lse_i - z_i,y_i   (rows with y_i = ignore_index: 0)
//   G_ij = exp(z_ij - lse_i) - [j = y_i],  dx = s G w,  dw = s G^T x,  s = dloss / (tau * count)
// One tiled matrix product (kernel ce_gemm) serves all four products:
//   LOSS   z = w x^T; its epilogue leaves (max, sum exp) of the tile's 256 classes per row, and the label's logit
//   GRAD   z again, its epilogue turns the tile into G (16 bit) for a PIECE of the classes; a piece is bounded in bytes
//   DX     dx += w^T G over the piece, DW  dw = x^T G over the rows
// Layout.  Every product has the operand whose index lands in the accumulator REGISTERS first (classes for LOSS / GRAD, feature
// columns for DX / DW) and the other one in the lanes: a lane then owns one row of the softmax (reductions over classes are
// in-lane loops plus one half-wave exchange) and four consecutive registers are four consecutive columns of the output.
// LDS.  Operands arrive by 16-byte LDS-DMA in the order they have in memory.  Where the contraction runs along memory, fragments
// are plain 16-byte reads; where it runs across (w in DX, both in DW) they are transposing 8-byte reads, so no operand is ever
// stored transposed.  Both layouts are swizzled in 16-byte chunks (on the global address of the DMA, whose LDS side is fixed).
// Precision.  16-bit features enter as they are, fp32 features as two fp16 pieces under one power-of-two scale per tensor
// (22 significand bits; three products hi*hi + hi*lo + lo*hi, error <= 2^-21 of |x||w|).  Accumulation, the softmax statistics and
// the sums over splits are fp32.  G is rounded once to the operand type (bf16: 2^-8; fp16: 2^-11 relative, scaled by 2^14 so that
// probabilities down to 2^-28 keep it; fp32 features: two fp16 pieces, 2^-22): the matrix cores take 16-bit operands.
#include "common.h"

namespace creste {

typedef float cef4 __attribute__((ext_vector_type(4)));
typedef float cef16 __attribute__((ext_vector_type(16)));
typedef short ces4 __attribute__((ext_vector_type(4)));
typedef short ces8 __attribute__((ext_vector_type(8)));
typedef _Float16 ceh8 __attribute__((ext_vector_type(8)));
typedef __bf16 ceb8 __attribute__((ext_vector_type(8)));

constexpr float kCeLog2e = 1.44269504088896341f, kCeLn2 = 0.693147180559945309f;
constexpr int kCeTile = 256;                 // classes per LOSS / GRAD tile, rows (LOSS, GRAD, DX) or classes (DW) per tile
constexpr float kCeF16Scale = 16384.f;       // G enters as G * 2^14 where it is stored in fp16

enum { CE_LOSS, CE_GRAD, CE_DX, CE_DW };

struct CeArgs {
  const char *a, *b;                // first operand (accumulator rows), second (accumulator columns), 16-bit elements
  int64_t lda, ldb;                 // bytes between their memory rows
  int64_t pa, pb;                   // bytes between the two pieces
  int64_t ra, rb;                   // memory rows that exist (loads clamp to the last one)
  int ca, cb;                       // bytes of a memory row that exist (transposed operands: loads clamp to the last 16)
  int m, n;                         // extents of the output
  int mt, nt;                       // tiles along m, n
  int k0, k1, ksplit;               // contraction range; ksplit > 0: split s works [k0 + s * ksplit, + ksplit)
  // LOSS / GRAD
  const int64_t* labels;
  int64_t ignore;
  int class0;                       // first class of the piece
  int classes;                      // all classes
  float inv_tau;
  const float* amax;                // [2] max|x|, max|w| (two-piece operands) or null
  float2* part;                     // LOSS: [class tile][n] (max, sum) in log2 units
  float* zlab;                      // LOSS: [n] label logit, log2 units
  const float* lse2;                // GRAD: [n]
  char* g;                          // GRAD: [n64][ldg] elements, pieces pg bytes apart
  int64_t ldg, pg;
  int n64;
  // DX / DW
  float* partial;                   // [split][n][ldp] or null: direct
  int64_t ldp, psplit;
  int accumulate;
  void* out;
  int64_t ldo;
  int out_dt;
  const float *gl, *stat;           // dloss, {sum nll, count}
  int mean;
  float gscale;                     // the power of two G was stored with
  int which;                        // 0: operand a is x, 1: it is w (picks the operand scale)
};

__device__ __forceinline__ float ce_operand_inv(const float* amax, int which) {
  if (!amax) return 1.f;
  float inv;
  f16_operand_scale(amax[which], &inv);
  return inv;
}

// dloss / (tau * count) and the powers of two of the stored operands
__device__ __forceinline__ float ce_out_scale(const CeArgs& p) {
  float s = p.gl[0] * p.inv_tau;
  if (p.mean) s = s / fmaxf(p.stat[1], 1.f);
  return s * (ce_operand_inv(p.amax, p.which) / p.gscale);
}

template <int DT>
__device__ __forceinline__ cef16 ce_mfma(ces8 a, ces8 b, cef16 c) {
  if constexpr (DT == CRESTE_DT_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ceb8, a), __builtin_bit_cast(ceb8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ceh8, a), __builtin_bit_cast(ceh8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ short ce_cvt(float v) {
  if constexpr (DT == CRESTE_DT_BF16) return __builtin_bit_cast(short, (__bf16)v);
  else return __builtin_bit_cast(short, (_Float16)v);
}

// ---- tile of one operand in LDS.  BX = extent across the contraction, BK = along it, KM: memory rows run along the contraction
// ("transposed").  Plain rows hold BK elements; 256 bytes = 64 banks = 16 chunks, so chunk c of row r sits at
// c ^ (r / rows-per-256-bytes): 16 lanes reading one chunk column of 16 rows touch 16 different chunk positions.
// Transposed rows hold BX elements; a transposing read takes 64 bytes of each of 4 rows, which (k & 3) << 2 spreads over the banks.
template <int BX, int BK, bool KM>
struct CeTile {
  static constexpr int ROWB = KM ? BX * 2 : BK * 2;
  static constexpr int CPR = ROWB / 16;
  static constexpr int BYTES = BX * BK * 2;
  static constexpr int INSTR = BYTES / 1024;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (KM) return (r & 3) << 2;
    else return (r / (16 / CPR)) & (CPR - 1);
  }
};

template <int BX, int BK, bool KM>
__device__ __forceinline__ void ce_dma(char* lds, const char* base, int64_t ld, int64_t rows, int colbytes, int64_t row0, int x0,
                                       int k, int wave, int lane) {
  using L = CeTile<BX, BK, KM>;
#pragma unroll
  for (int i0 = 0; i0 < L::INSTR; i0 += 8) {
    const int i = i0 + wave;
    const int pos = i * 64 + lane, r = pos / L::CPR, c = (pos % L::CPR) ^ L::swz(r);
    int64_t row = (KM ? (int64_t)k : row0) + r;
    row = row < rows ? row : rows - 1;
    int64_t off = (KM ? (int64_t)x0 : (int64_t)k) * 2 + c * 16;
    if constexpr (KM) off = off <= colbytes - 16 ? off : colbytes - 16;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + row * ld + off),
                                     (__attribute__((address_space(3))) void*)(lds + i * 1024), 16, 0, 0);
  }
}

// 8 consecutive contraction elements of index x0 + li: lanes lh = 0 / 1 take elements kk * 16 + 8 * lh ..
template <int BX, int BK, bool KM>
__device__ __forceinline__ ces8 ce_frag(const char* lds, int x0, int kk, int lane) {
  using L = CeTile<BX, BK, KM>;
  if constexpr (!KM) {
    const int row = x0 + (lane & 31), c = kk * 2 + (lane >> 5);
    return *reinterpret_cast<const ces8*>(lds + row * L::ROWB + ((c ^ L::swz(row)) << 4));
  } else {
    const int l = lane & 15, g = lane >> 4;
    const int col = x0 + 16 * (g & 1) + 4 * (l & 3);
    ces8 v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = kk * 16 + 8 * (g >> 1) + 4 * j + (l >> 2);
      const char* p = lds + k * L::ROWB + (((col >> 3) ^ L::swz(k)) << 4) + (col & 7) * 2;
      const ces4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ces4*)p);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * j + e] = t[e];
    }
    return v;
  }
}

// DT: 16-bit operand type (fp16 for two-piece fp32), P: pieces, BM: tile extent along the accumulator rows
template <int MODE, int DT, int P, int BM>
__global__ __launch_bounds__(512, 2) void ce_gemm_kernel(CeArgs p) {
  constexpr bool AKM = MODE == CE_DX || MODE == CE_DW, BKM = MODE == CE_DW;
  constexpr int BN = kCeTile, BK = 64 / P, MT = BM / 64, NT = 2;
  using LA = CeTile<BM, BK, AKM>;
  using LB = CeTile<BN, BK, BKM>;
  constexpr int STAGE = P * (LA::BYTES + LB::BYTES);
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, lh = lane >> 5;
  const int wm = wave >> 2, wn = wave & 3;
  int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tm = t % p.mt;
  t /= p.mt;
  const int tn = t % p.nt, split = t / p.nt;
  const int m0 = tm * BM, n0 = tn * BN;
  const int kb = p.k0 + split * p.ksplit;
  const int ke = p.ksplit ? min(p.k1, kb + p.ksplit) : p.k1;

  cef16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  auto dma = [&](int k, int s) __attribute__((always_inline)) {
    char* st = smem + s * STAGE;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      ce_dma<BM, BK, AKM>(st + q * LA::BYTES, p.a + q * p.pa, p.lda, p.ra, p.ca, m0, m0, k, wave, lane);
      ce_dma<BN, BK, BKM>(st + P * LA::BYTES + q * LB::BYTES, p.b + q * p.pb, p.ldb, p.rb, p.cb, n0, n0, k, wave, lane);
    }
  };

  if (kb < ke) {
    dma(kb, 0);
    for (int k = kb, c = 0; k < ke; k += BK, ++c) {
      __syncthreads();                                  // stage c has landed, everybody has left the other one
      if (k + BK < ke) dma(k + BK, (c + 1) & 1);
      const char* A = smem + (c & 1) * STAGE;
      const char* B = A + P * LA::BYTES;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) {
        ces8 af[P][MT], bf[P][NT];
#pragma unroll
        for (int q = 0; q < P; ++q) {
#pragma unroll
          for (int i = 0; i < MT; ++i) af[q][i] = ce_frag<BM, BK, AKM>(A + q * LA::BYTES, wm * (BM / 2) + i * 32, kk, lane);
#pragma unroll
          for (int j = 0; j < NT; ++j) bf[q][j] = ce_frag<BN, BK, BKM>(B + q * LB::BYTES, wn * 64 + j * 32, kk, lane);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if constexpr (P == 2) {                     // small products first
              acc[i][j] = ce_mfma<DT>(af[1][i], bf[0][j], acc[i][j]);
              acc[i][j] = ce_mfma<DT>(af[0][i], bf[1][j], acc[i][j]);
            }
            acc[i][j] = ce_mfma<DT>(af[0][i], bf[0][j], acc[i][j]);
          }
      }
    }
  }

  if constexpr (MODE == CE_LOSS || MODE == CE_GRAD) {
    const float c2 = ce_operand_inv(p.amax, 0) * ce_operand_inv(p.amax, 1) * p.inv_tau * kCeLog2e;
    const int mw = m0 + wm * (BM / 2);                  // first class of this wave, within the piece
    if constexpr (MODE == CE_LOSS) {
      float2* sh = reinterpret_cast<float2*>(smem);     // [wm][256 rows]
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = n0 + wn * 64 + j * 32 + li;
        // the label's class relative to this wave's first one (a label outside [0, classes) matches nothing)
        const int64_t y = row < p.n ? p.labels[row] : -1;
        const int64_t yr = y - mw;
        const int lab = y >= 0 && y < p.classes && yr >= 0 && yr < BM / 2 ? (int)yr : -1;
        float mx = -INFINITY, sum = 0.f, z = 0.f;
        if (mw + BM / 2 > p.m) {                        // classes behind the last one: exp2 gives 0
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (mw + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh >= p.m) acc[i][j][r] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[i][j][r]);
        if (__any(lab >= 0)) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh == lab ? acc[i][j][r] : z;
        }
        mx = fmaxf(mx * c2, -3.0e38f);                  // (a half tile without classes has no maximum)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], c2, -mx));
        const float mo = __shfl_xor(mx, 32, 64), so = __shfl_xor(sum, 32, 64);
        const float mm = fmaxf(mx, mo);
        sum = sum * __builtin_amdgcn_exp2f(mx - mm) + so * __builtin_amdgcn_exp2f(mo - mm);
        if (lh == 0) sh[wm * 256 + wn * 64 + j * 32 + li] = make_float2(mm, sum);
        if (lab >= 0 && ((lab >> 2) & 1) == lh) p.zlab[row] = z * c2;
      }
      __syncthreads();
      const int i = threadIdx.x;
      if (i < 256 && n0 + i < p.n) {
        const float2 u = sh[i], v = sh[256 + i];
        const float mm = fmaxf(u.x, v.x);
        p.part[(int64_t)tm * p.n + n0 + i] =
            make_float2(mm, u.y * __builtin_amdgcn_exp2f(u.x - mm) + v.y * __builtin_amdgcn_exp2f(v.x - mm));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = n0 + wn * 64 + j * 32 + li;
        if (row >= p.n64) continue;
        int64_t y = row < p.n ? p.labels[row] : p.ignore;
        const bool on = row < p.n && y != p.ignore;
        // a label that names no class: nll is NaN, and so is its row of G
        const float scale = !on ? 0.f : (y < 0 || y >= p.classes) ? __builtin_nanf("") : p.gscale;
        const float l2 = on ? p.lse2[row] : 0.f;
        const int64_t yr = y - p.class0 - mw;
        const int lab = on && yr >= 0 && yr < BM / 2 ? (int)yr : -1;
        char* grow = p.g + row * p.ldg;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int cl = i * 32 + 8 * q + 4 * lh;
            ces4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = __builtin_amdgcn_exp2f(fmaf(acc[i][j][4 * q + e], c2, -l2));
              v = cl + e == lab ? v - 1.f : v;
              v = on && mw + cl + e < p.m ? v * scale : 0.f;
              const short h = ce_cvt<DT>(v);
              hi[e] = h;
              if constexpr (P == 2) lo[e] = ce_cvt<DT>(v - (float)__builtin_bit_cast(_Float16, h));
            }
            *reinterpret_cast<ces4*>(grow + (int64_t)(mw + cl) * 2) = hi;
            if constexpr (P == 2) *reinterpret_cast<ces4*>(grow + p.pg + (int64_t)(mw + cl) * 2) = lo;
          }
      }
    }
  } else {
    const float fs = p.partial ? 1.f : ce_out_scale(p);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int row = n0 + wn * 64 + j * 32 + li;
      if (row >= p.n) continue;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d = m0 + wm * (BM / 2) + i * 32 + 8 * q + 4 * lh;
          if (d >= p.m) continue;
          cef4 v{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          if (p.partial) {                              // rows of partials are padded to 4
            cef4* dst = reinterpret_cast<cef4*>(p.partial + split * p.psplit + row * p.ldp + d);
            *dst = p.accumulate ? *dst + v : v;
            continue;
          }
          v *= fs;
          const int64_t o = row * p.ldo + d;
          if ((p.m & 3) == 0) {
            if (p.out_dt == CRESTE_DT_F32) {
              *reinterpret_cast<cef4*>((float*)p.out + o) = v;
            } else {
              ces4 s;
#pragma unroll
              for (int e = 0; e < 4; ++e) s[e] = ce_cvt<DT>(v[e]);
              *reinterpret_cast<ces4*>((short*)p.out + o) = s;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (d + e >= p.m) continue;
              if (p.out_dt == CRESTE_DT_F32) ((float*)p.out)[o + e] = v[e];
              else ((short*)p.out)[o + e] = ce_cvt<DT>(v[e]);
            }
          }
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------------- few rows
// LOSS for at most 32 rows: bound by reading w once, so no LDS and no copy of the operands -- a wave streams 64 classes from
// memory straight into the matrix instructions, one group of loads (128 bytes of each class row) ahead.  fp32 goes through
// the fp32 matrix instruction (32 x 32 x 2, 157 TF: 32 rows need 16 products a loaded element, well below it).  The lane
// halves take alternate 16-byte pieces of the contraction in both operands, which for fp32 makes a 16-byte load feed four instructions.
template <int DT>
__global__ __launch_bounds__(256) void ce_few_kernel(CeArgs p, int D) {
  constexpr int EB = DT == CRESTE_DT_F32 ? 4 : 2, STEP = 32 / EB;      // elements both halves take per load
  typedef int iv4 __attribute__((ext_vector_type(4)));
  __shared__ float2 sh[4][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, lh = lane >> 5;
  const int m0 = blockIdx.x * kCeTile + wave * 64;
  const int row = li < p.n ? li : p.n - 1;
  const char* xr = p.b + row * p.ldb + lh * 16;
  const char* wr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t c = m0 + i * 32 + li;
    wr[i] = p.a + (c < p.m ? c : p.m - 1) * p.lda + lh * 16;
  }
  cef16 acc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  const int steps = D / STEP;
  iv4 xa[2][4], wa[2][2][4];
  auto load = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t o = (int64_t)(s + q < steps ? s + q : steps - 1) * 32;
      xa[buf][q] = *reinterpret_cast<const iv4*>(xr + o);
#pragma unroll
      for (int i = 0; i < 2; ++i) wa[buf][i][q] = *reinterpret_cast<const iv4*>(wr[i] + o);
    }
  };
  auto mul = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (s + q >= steps) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (DT == CRESTE_DT_F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(cef4, wa[buf][i][q])[e], __builtin_bit_cast(cef4, xa[buf][q])[e],
                                                          acc[i], 0, 0, 0);
        } else {
          acc[i] = ce_mfma<DT>(__builtin_bit_cast(ces8, wa[buf][i][q]), __builtin_bit_cast(ces8, xa[buf][q]), acc[i]);
        }
      }
    }
  };
  load(0, 0);
  for (int s = 0; s < steps; s += 8) {
    load(s + 4, 1);
    mul(s, 0);
    load(s + 8, 0);
    mul(s + 4, 1);
  }
  const float c2 = p.inv_tau * kCeLog2e;
  const int64_t y = li < p.n ? p.labels[li] : -1;
  const int64_t yr = y - m0;
  const int lab = y >= 0 && y < p.classes && yr >= 0 && yr < 64 ? (int)yr : -1;
  float mx = -INFINITY, sum = 0.f, z = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int cl = i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh;
      if (m0 + cl >= p.m) acc[i][r] = -INFINITY;
      z = cl == lab ? acc[i][r] : z;
      mx = fmaxf(mx, acc[i][r]);
    }
  mx = fmaxf(mx * c2, -3.0e38f);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][r], c2, -mx));
  const float mo = __shfl_xor(mx, 32, 64), so = __shfl_xor(sum, 32, 64);
  float mm = fmaxf(mx, mo);
  sum = sum * __builtin_amdgcn_exp2f(mx - mm) + so * __builtin_amdgcn_exp2f(mo - mm);
  if (lh == 0) sh[wave][li] = make_float2(mm, sum);
  if (lab >= 0 && ((lab >> 2) & 1) == lh) p.zlab[li] = z * c2;
  __syncthreads();
  if (threadIdx.x < 32 && (int)threadIdx.x < p.n) {
    for (int j = 1; j < 4; ++j) {
      const float2 v = sh[j][li];
      const float m = fmaxf(mm, v.x);
      sum = sum * __builtin_amdgcn_exp2f(mm - m) + v.y * __builtin_amdgcn_exp2f(v.x - m);
      mm = m;
    }
    p.part[(int64_t)blockIdx.x * p.n + li] = make_float2(mm, sum);
  }
}

// ---------------------------------------------------------------------------------------------------- small kernels
__global__ void ce_zero_kernel(float* p, int n) {
  if ((int)threadIdx.x < n) p[threadIdx.x] = 0.f;
}

// max |x| of a [rows][cols] fp32 matrix with row stride ld
__global__ __launch_bounds__(256) void ce_amax_kernel(const float* __restrict__ x, int64_t rows, int cols, int64_t ld,
                                                      float* __restrict__ amax) {
  __shared__ float scratch[4];
  float m = 0.f;
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int64_t r = i / cols;
    m = fmaxf(m, fabsf(x[r * ld + (i - r * cols)]));
  }
  block_amax_update(m, amax, scratch);
}

// 16-bit copy of the features with rows of cp (a multiple of 64) elements, zero behind the last column.  fp32: two pieces
template <typename T>
__global__ __launch_bounds__(256) void ce_pack_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ld, int cp,
                                                      const float* __restrict__ amax, short* __restrict__ out, int64_t piece) {
  float inv = 1.f, s = 1.f;
  if constexpr (sizeof(T) == 4) s = f16_operand_scale(*amax, &inv);
  const int64_t total = rows * (cp / 4);
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int64_t r = i / (cp / 4);
    const int c = (int)(i - r * (cp / 4)) * 4;
    ces4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const T v = c + e < cols ? x[r * ld + c + e] : (T)0;
      if constexpr (sizeof(T) == 4) {
        const float a = v * s;
        const short h = ce_cvt<CRESTE_DT_F16>(a);
        hi[e] = h;
        lo[e] = ce_cvt<CRESTE_DT_F16>(a - (float)__builtin_bit_cast(_Float16, h));
      } else {
        hi[e] = (short)v;
      }
    }
    *reinterpret_cast<ces4*>(out + r * cp + c) = hi;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<ces4*>(out + piece + r * cp + c) = lo;
  }
}

// per row: join the class tiles' (max, sum).  64 rows x 16 slices of the tiles per block; per block the sums of nll and count, or
// the loss itself when there is one block
__global__ __launch_bounds__(1024) void ce_join_kernel(const float2* __restrict__ part, int tiles, int n, const float* __restrict__ zlab,
                                                       const int64_t* __restrict__ labels, int64_t ignore, int classes,
                                                       float* __restrict__ nll, float* __restrict__ lse2, float2* __restrict__ bsum,
                                                       int mean, float* __restrict__ loss, float* __restrict__ stat) {
  __shared__ float2 sh[16][64];
  const int li = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const int row = blockIdx.x * 64 + li;
  float mx = -3.0e38f, sum = 0.f;
  if (row < n)
#pragma unroll 4
    for (int t = sl; t < tiles; t += 16) {
      const float2 v = part[(int64_t)t * n + row];
      const float m = fmaxf(mx, v.x);
      sum = sum * __builtin_amdgcn_exp2f(mx - m) + v.y * __builtin_amdgcn_exp2f(v.x - m);
      mx = m;
    }
  sh[sl][li] = make_float2(mx, sum);
  __syncthreads();
  if (sl) return;
  for (int s = 1; s < 16; ++s) {
    const float2 v = sh[s][li];
    const float m = fmaxf(mx, v.x);
    sum = sum * __builtin_amdgcn_exp2f(mx - m) + v.y * __builtin_amdgcn_exp2f(v.x - m);
    mx = m;
  }
  float l = 0.f, c = 0.f;
  if (row < n) {
    const float z = mx + __builtin_amdgcn_logf(sum);
    const int64_t y = labels[row];
    const bool on = y != ignore;
    lse2[row] = z;
    if (on) {
      l = y >= 0 && y < classes ? (z - zlab[row]) * kCeLn2 : __builtin_nanf("");
      c = 1.f;
    }
    nll[row] = l;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    l += __shfl_xor(l, o, 64);
    c += __shfl_xor(c, o, 64);
  }
  if (li) return;
  if (gridDim.x > 1) {
    bsum[blockIdx.x] = make_float2(l, c);
  } else {
    stat[0] = l;
    stat[1] = c;
    *loss = mean ? l / fmaxf(c, 1.f) : l;
  }
}

// loss from the blocks' sums (fixed order), stat = {sum nll, count}
__global__ __launch_bounds__(256) void ce_final_kernel(const float2* __restrict__ bsum, int nb, int mean, float* __restrict__ loss,
                                                       float* __restrict__ stat) {
  __shared__ double sl[256], sc[256];
  double l = 0., c = 0.;
  for (int i = threadIdx.x; i < nb; i += 256) {
    l += bsum[i].x;
    c += bsum[i].y;
  }
  sl[threadIdx.x] = l;
  sc[threadIdx.x] = c;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) {
      sl[threadIdx.x] += sl[threadIdx.x + o];
      sc[threadIdx.x] += sc[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    stat[0] = (float)sl[0];
    stat[1] = (float)sc[0];
    *loss = (float)(mean ? sl[0] / fmax(sc[0], 1.) : sl[0]);
  }
}

// out[n][m] = scale * sum over splits of partial[split][n][ldp]
__global__ __launch_bounds__(256) void ce_reduce_kernel(CeArgs p, int splits) {
  const float fs = ce_out_scale(p);
  const int64_t total = (int64_t)p.n * p.ldp;
  for (int64_t i = (blockIdx.x * 256LL + threadIdx.x) * 4; i < total; i += gridDim.x * 1024LL) {
    cef4 v = *reinterpret_cast<const cef4*>(p.partial + i);
    for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const cef4*>(p.partial + s * p.psplit + i);
    v *= fs;
    const int64_t row = i / p.ldp;
    const int d = (int)(i - row * p.ldp);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (d + e >= p.m) continue;
      const int64_t o = row * p.ldo + d + e;
      if (p.out_dt == CRESTE_DT_F32) ((float*)p.out)[o] = v[e];
      else if (p.out_dt == CRESTE_DT_BF16) ((short*)p.out)[o] = ce_cvt<CRESTE_DT_BF16>(v[e]);
      else ((short*)p.out)[o] = ce_cvt<CRESTE_DT_F16>(v[e]);
    }
  }
}

// --------------------------------------------------------------------------------------------------------- host side
namespace {

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Where everything sits in the caller's workspace.  The operands are used in place when a row is a multiple of 64 elements on
// 16-byte boundaries, else copied once (padded; fp32 always: into its two pieces).
struct CePlan {
  int P, dt16, es, Dp, ldq, bm;
  bool packx, packw;
  int64_t amax, xp, wp, part, zlab, bsum, g, dxp, dwp, total;
  int64_t vc, n64;                 // classes per piece, rows of G
  int pieces, tiles, sx, sw;       // class tiles of the loss, splits of DX / DW
};

constexpr int64_t kCePieceBytes = 512ll << 20;     // bound on G

bool ce_direct(const void* x, int64_t ld, int D, int dtype) {
  return dtype != CRESTE_DT_F32 && D % 64 == 0 && ld % 8 == 0 && ((uintptr_t)x & 15) == 0;
}

constexpr int kCeFewRows = 32;

// rows that the few-rows kernel can read in place: whole 32-byte steps on 16-byte boundaries
bool ce_few(const void* x, int64_t ld, int D, int dtype) {
  const int es = dtype == CRESTE_DT_F32 ? 4 : 2;
  return D * es % 32 == 0 && ld * es % 16 == 0 && ((uintptr_t)x & 15) == 0;
}

CePlan ce_plan(int64_t N, int64_t V, int D, int dtype, bool packx, bool packw, bool train) {
  CePlan q{};
  q.P = dtype == CRESTE_DT_F32 ? 2 : 1;
  q.dt16 = dtype == CRESTE_DT_BF16 ? CRESTE_DT_BF16 : CRESTE_DT_F16;
  q.es = dtype == CRESTE_DT_F32 ? 4 : 2;
  q.Dp = (int)up(D, 64);
  q.ldq = (int)up(D, 4);
  q.packx = packx;
  q.packw = packw;
  q.bm = D <= 128 ? 128 : 256;
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o = up(o + bytes, 1024); return at; };
  q.amax = take(64);
  q.xp = packx ? take(N * q.Dp * 2 * q.P) : 0;
  q.wp = packw ? take(V * q.Dp * 2 * q.P) : 0;
  q.tiles = (int)((V + kCeTile - 1) / kCeTile);
  if (!train) {
    q.part = take((int64_t)q.tiles * N * 8);
    q.zlab = take(N * 4);
    q.bsum = take((N + 63) / 64 * 8);
  } else {
    q.n64 = up(N, 64);
    const int64_t vall = up(V, kCeTile);
    int64_t vc = kCePieceBytes / (q.n64 * 2 * q.P) / kCeTile * kCeTile;
    vc = vc < kCeTile ? kCeTile : vc > vall ? vall : vc;
    q.pieces = (int)((vall + vc - 1) / vc);
    q.vc = up((vall + q.pieces - 1) / q.pieces, kCeTile);        // pieces of one size
    q.pieces = (int)((vall + q.vc - 1) / q.vc);
    q.g = take(q.n64 * q.vc * 2 * q.P);
    // splits of the contraction: enough workgroups for the 256 CUs, chunks of at least 512
    const int64_t mt = (D + q.bm - 1) / q.bm;
    auto splits = [&](int64_t tiles, int64_t k) {
      int64_t s = (256 + tiles - 1) / tiles;
      const int64_t most = (k + 511) / 512;
      s = s > most ? most : s;
      return (int)(s < 1 ? 1 : s);
    };
    q.sx = splits(mt * ((N + kCeTile - 1) / kCeTile), q.vc);
    q.sw = splits(mt * (q.vc / kCeTile), q.n64);
    if (q.sx > 1 || q.pieces > 1) q.dxp = take((int64_t)q.sx * N * q.ldq * 4);
    if (q.sw > 1) q.dwp = take((int64_t)q.sw * q.vc * q.ldq * 4);
  }
  q.total = o;
  return q;
}

template <int MODE, int DT, int P, int BM>
int ce_launch(const CeArgs& a, int blocks, hipStream_t s) {
  constexpr int bytes = 2 * (BM + kCeTile) * 64 * 2;
  static std::atomic<uint64_t> mask{0};
  CRESTE_HIP(ensure_dyn_smem((const void*)ce_gemm_kernel<MODE, DT, P, BM>, bytes, mask));
  ce_gemm_kernel<MODE, DT, P, BM><<<blocks, 512, bytes, s>>>(a);
  CRESTE_CHECK_LAUNCH("linear_ce gemm");
  return CRESTE_OK;
}

template <int MODE>
int ce_dispatch(const CePlan& q, const CeArgs& a, int blocks, hipStream_t s) {
  const bool narrow = MODE >= CE_DX && q.bm == 128;
  if (q.P == 2) {
    if constexpr (MODE >= CE_DX)
      if (narrow) return ce_launch<MODE, CRESTE_DT_F16, 2, 128>(a, blocks, s);
    return ce_launch<MODE, CRESTE_DT_F16, 2, 256>(a, blocks, s);
  }
  if (q.dt16 == CRESTE_DT_BF16) {
    if constexpr (MODE >= CE_DX)
      if (narrow) return ce_launch<MODE, CRESTE_DT_BF16, 1, 128>(a, blocks, s);
    return ce_launch<MODE, CRESTE_DT_BF16, 1, 256>(a, blocks, s);
  }
  if constexpr (MODE >= CE_DX)
    if (narrow) return ce_launch<MODE, CRESTE_DT_F16, 1, 128>(a, blocks, s);
  return ce_launch<MODE, CRESTE_DT_F16, 1, 256>(a, blocks, s);
}

int ce_grid(int64_t items) { return (int)(items < 1 ? 1 : items > 2048 ? 2048 : items); }

int ce_pack(const void* src, int64_t ld, int64_t rows, int D, int dtype, const CePlan& q, float* amax, char* dst, hipStream_t s) {
  const int nb = ce_grid(rows * (q.Dp / 4) / 256 + 1);
  const int64_t piece = rows * q.Dp;
  if (dtype == CRESTE_DT_F32) {
    ce_amax_kernel<<<ce_grid(rows * D / 1024 + 1), 256, 0, s>>>((const float*)src, rows, D, ld, amax);
    ce_pack_kernel<float><<<nb, 256, 0, s>>>((const float*)src, rows, D, ld, q.Dp, amax, (short*)dst, piece);
  } else {
    ce_pack_kernel<short><<<nb, 256, 0, s>>>((const short*)src, rows, D, ld, q.Dp, nullptr, (short*)dst, piece);
  }
  CRESTE_CHECK_LAUNCH("linear_ce pack");
  return CRESTE_OK;
}

struct CeOperand { const char* p; int64_t ld, piece; };

int ce_operands(const CePlan& q, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int64_t V, int D, int dtype,
                char* work, CeOperand* X, CeOperand* W, hipStream_t s) {
  float* amax = (float*)(work + q.amax);
  if (q.P == 2) {
    ce_zero_kernel<<<1, 64, 0, s>>>(amax, 2);
    CRESTE_CHECK_LAUNCH("linear_ce zero");
  }
  *X = {(const char*)x, ldx * 2, 0};
  *W = {(const char*)w, ldw * 2, 0};
  if (q.packx) {
    const int rc = ce_pack(x, ldx, N, D, dtype, q, amax, work + q.xp, s);
    if (rc) return rc;
    *X = {work + q.xp, (int64_t)q.Dp * 2, N * q.Dp * 2};
  }
  if (q.packw) {
    const int rc = ce_pack(w, ldw, V, D, dtype, q, amax + 1, work + q.wp, s);
    if (rc) return rc;
    *W = {work + q.wp, (int64_t)q.Dp * 2, V * q.Dp * 2};
  }
  return CRESTE_OK;
}

int ce_check(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* labels, int64_t N, int64_t V, int D, int dtype,
             float tau) {
  CRESTE_REQUIRE(x && w && labels, "linear_ce: null pointer");
  CRESTE_REQUIRE(dtype >= CRESTE_DT_F32 && dtype <= CRESTE_DT_F16, "linear_ce: dtype %d", dtype);
  CRESTE_REQUIRE(N > 0 && V > 0 && D > 0 && N < (1ll << 30) && V < (1ll << 30) && D <= 65536, "linear_ce: N %lld V %lld D %d",
                 (long long)N, (long long)V, D);
  CRESTE_REQUIRE((ldx >= D || (ldx == 0 || N == 1)) && ldx >= 0 && (ldw >= D || V == 1 || ldw == 0) && ldw >= 0,
                 "linear_ce: row strides %lld %lld", (long long)ldx, (long long)ldw);
  CRESTE_REQUIRE(tau > 0.f && tau < INFINITY, "linear_ce: temperature must be positive and finite");
  return CRESTE_OK;
}

}  // namespace
}  // namespace creste

using namespace creste;

extern "C" int64_t creste_linear_ce_workspace_bytes(int64_t N, int64_t V, int D, int dtype, int train) {
  if (N <= 0 || V <= 0 || D <= 0 || N >= (1ll << 30) || V >= (1ll << 30) || D > 65536 || dtype < CRESTE_DT_F32 || dtype > CRESTE_DT_F16)
    return -1;
  return ce_plan(N, V, D, dtype, true, true, train != 0).total;      // as if both operands had to be copied
}

extern "C" int creste_linear_ce_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* labels, int64_t N,
                                        int64_t V, int D, int dtype, int64_t ignore_index, float temperature, int mean,
                                        float* loss, float* nll, float* lse2, float* stat, void* work, int64_t work_bytes,
                                        void* stream) {
  const int bad = ce_check(x, ldx, w, ldw, labels, N, V, D, dtype, temperature);
  if (bad) return bad;
  const bool few = N <= kCeFewRows && ce_few(x, ldx, D, dtype) && ce_few(w, ldw, D, dtype);
  const CePlan q = ce_plan(N, V, D, dtype, !few && !ce_direct(x, ldx, D, dtype), !few && !ce_direct(w, ldw, D, dtype), false);
  CRESTE_REQUIRE(loss && nll && lse2 && stat && work && work_bytes >= q.total, "linear_ce_forward: outputs / workspace (%lld of %lld bytes)",
                 (long long)work_bytes, (long long)q.total);
  hipStream_t s = (hipStream_t)stream;
  char* wk = (char*)work;
  CeOperand X{(const char*)x, ldx * q.es, 0}, W{(const char*)w, ldw * q.es, 0};
  if (!few) {
    const int rc = ce_operands(q, x, ldx, w, ldw, N, V, D, dtype, wk, &X, &W, s);
    if (rc) return rc;
  }
  CeArgs a{};
  a.a = W.p; a.lda = W.ld; a.pa = W.piece; a.ra = V;
  a.b = X.p; a.ldb = X.ld; a.pb = X.piece; a.rb = N;
  a.m = (int)V; a.n = (int)N;
  a.mt = q.tiles; a.nt = cdiv(N, kCeTile);
  a.k1 = q.Dp;
  a.labels = labels; a.ignore = ignore_index; a.classes = (int)V;
  a.inv_tau = 1.f / temperature;
  a.amax = q.P == 2 ? (const float*)(wk + q.amax) : nullptr;
  a.part = (float2*)(wk + q.part); a.zlab = (float*)(wk + q.zlab);
  CRESTE_REQUIRE((int64_t)a.mt * a.nt < (1ll << 31), "linear_ce: too many tiles");
  if (few) {
    if (dtype == CRESTE_DT_F32) ce_few_kernel<CRESTE_DT_F32><<<q.tiles, 256, 0, s>>>(a, D);
    else if (dtype == CRESTE_DT_BF16) ce_few_kernel<CRESTE_DT_BF16><<<q.tiles, 256, 0, s>>>(a, D);
    else ce_few_kernel<CRESTE_DT_F16><<<q.tiles, 256, 0, s>>>(a, D);
    CRESTE_CHECK_LAUNCH("linear_ce few rows");
  } else {
    const int rg = ce_dispatch<CE_LOSS>(q, a, a.mt * a.nt, s);
    if (rg) return rg;
  }
  const int nb = cdiv(N, 64);
  ce_join_kernel<<<nb, 1024, 0, s>>>(a.part, q.tiles, (int)N, a.zlab, labels, ignore_index, (int)V, nll, lse2, (float2*)(wk + q.bsum),
                                       mean, loss, stat);
  if (nb > 1) ce_final_kernel<<<1, 256, 0, s>>>((const float2*)(wk + q.bsum), nb, mean, loss, stat);
  CRESTE_CHECK_LAUNCH("linear_ce join");
  return CRESTE_OK;
}

extern "C" int creste_linear_ce_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* labels, int64_t N,
                                         int64_t V, int D, int dtype, int64_t ignore_index, float temperature, int mean,
                                         const float* lse2, const float* stat, const float* g_loss, void* gx, void* gw, void* work,
                                         int64_t work_bytes, void* stream) {
  const int bad = ce_check(x, ldx, w, ldw, labels, N, V, D, dtype, temperature);
  if (bad) return bad;
  const CePlan q = ce_plan(N, V, D, dtype, !ce_direct(x, ldx, D, dtype), !ce_direct(w, ldw, D, dtype), true);
  CRESTE_REQUIRE(lse2 && stat && g_loss && (gx || gw) && work && work_bytes >= q.total,
                 "linear_ce_backward: inputs / workspace (%lld of %lld bytes)", (long long)work_bytes, (long long)q.total);
  hipStream_t s = (hipStream_t)stream;
  char* wk = (char*)work;
  CeOperand X, W;
  const int rc = ce_operands(q, x, ldx, w, ldw, N, V, D, dtype, wk, &X, &W, s);
  if (rc) return rc;
  CeArgs c{};                                       // what every product shares
  c.labels = labels; c.ignore = ignore_index; c.classes = (int)V;
  c.inv_tau = 1.f / temperature;
  c.amax = q.P == 2 ? (const float*)(wk + q.amax) : nullptr;
  c.lse2 = lse2; c.stat = stat; c.gl = g_loss; c.mean = mean;
  c.g = wk + q.g; c.ldg = q.vc * 2; c.pg = q.n64 * q.vc * 2; c.n64 = (int)q.n64;
  c.gscale = q.dt16 == CRESTE_DT_F16 ? kCeF16Scale : 1.f;
  c.out_dt = dtype;
  CeArgs dx = c;
  for (int piece = 0; piece < q.pieces; ++piece) {
    const int64_t v0 = piece * q.vc, nv = V - v0 < q.vc ? V - v0 : q.vc;
    CeArgs a = c;                                   // G of the piece
    a.a = W.p + v0 * W.ld; a.lda = W.ld; a.pa = W.piece; a.ra = nv;
    a.b = X.p; a.ldb = X.ld; a.pb = X.piece; a.rb = N;
    a.m = (int)nv; a.n = (int)N; a.class0 = (int)v0;
    a.mt = (int)(q.vc / kCeTile); a.nt = cdiv(N, kCeTile);
    a.k1 = q.Dp;
    int rg = ce_dispatch<CE_GRAD>(q, a, a.mt * a.nt, s);
    if (rg) return rg;
    if (gx) {
      dx = c;
      dx.a = W.p + v0 * W.ld; dx.lda = W.ld; dx.pa = W.piece; dx.ra = nv; dx.ca = q.Dp * 2;
      dx.b = c.g; dx.ldb = c.ldg; dx.pb = c.pg; dx.rb = q.n64;
      dx.m = D; dx.n = (int)N;
      dx.mt = cdiv(D, q.bm); dx.nt = cdiv(N, kCeTile);
      dx.k1 = (int)up(nv, 64);
      dx.ksplit = q.sx > 1 ? (int)up(cdiv(q.vc, q.sx), 64) : 0;
      if (q.sx > 1 || q.pieces > 1) dx.partial = (float*)(wk + q.dxp);
      dx.ldp = q.ldq; dx.psplit = N * q.ldq; dx.accumulate = piece > 0;
      dx.out = gx; dx.ldo = D; dx.which = 1;
      rg = ce_dispatch<CE_DX>(q, dx, dx.mt * dx.nt * q.sx, s);
      if (rg) return rg;
    }
    if (gw) {
      CeArgs b = c;
      b.a = X.p; b.lda = X.ld; b.pa = X.piece; b.ra = N; b.ca = q.Dp * 2;
      b.b = c.g; b.ldb = c.ldg; b.pb = c.pg; b.rb = q.n64; b.cb = (int)(q.vc * 2);
      b.m = D; b.n = (int)nv;
      b.mt = cdiv(D, q.bm); b.nt = cdiv(nv, kCeTile);
      b.k1 = (int)q.n64;
      b.ksplit = q.sw > 1 ? (int)up(cdiv(q.n64, q.sw), 64) : 0;
      if (q.sw > 1) b.partial = (float*)(wk + q.dwp);
      b.ldp = q.ldq; b.psplit = q.vc * q.ldq;
      b.out = (char*)gw + v0 * D * q.es; b.ldo = D; b.which = 0;
      rg = ce_dispatch<CE_DW>(q, b, b.mt * b.nt * q.sw, s);
      if (rg) return rg;
      if (b.partial) {
        ce_reduce_kernel<<<ce_grid((int64_t)b.n * q.ldq / 1024 + 1), 256, 0, s>>>(b, q.sw);
        CRESTE_CHECK_LAUNCH("linear_ce reduce");
      }
    }
  }
  if (gx && dx.partial) {
    ce_reduce_kernel<<<ce_grid(N * q.ldq / 1024 + 1), 256, 0, s>>>(dx, q.sx);
    CRESTE_CHECK_LAUNCH("linear_ce reduce");
  }
  return CRESTE_OK;
}
