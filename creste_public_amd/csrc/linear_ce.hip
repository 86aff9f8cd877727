// Softmax cross entropy over a large set of classes, straight from the features, without the logits in memory:
//   z_ij = (x_i . w_j) / tau,  lse_i = log sum_j exp z_ij,  nll_i = lse_i - z_i,y_i   (rows with y_i = ignore_index: 0)
//   G_ij = exp(z_ij - lse_i) - [j = y_i],  dx = s G w,  dw = s G^T x,  s = dloss / (tau * count)
// Up to 256 feature columns (fp32: 128) one kernel per direction streams past features held in registers (ce_stream_body, below).  Beyond,
// one tiled matrix product (ce_gemm_kernel) serves all four products:
//   LOSS   z = w x^T; its epilogue leaves (max, sum exp) of the tile's 256 classes per row, and the label's logit
//   GRAD   z again, its epilogue turns the tile into G (16 bit) for a PIECE of the classes; a piece is bounded in bytes
// Every kernel forms a logit in the same order of additions, so the largest of a row comes out of the gradients' products with the bits
// it had in the loss and G is taken against it, not against a rounded log-sum-exp: at logits of 10^6 that would be off by tens of percent.
// (Up to 32 rows fp32 features therefore stay fp32 in both directions, as the few-rows kernel takes them.)
//   DX     dx += w^T G over the piece, DW  dw = x^T G over the rows
// Layout.  Every product has the operand whose index lands in the accumulator REGISTERS first (classes for LOSS / GRAD, feature
// columns for DX / DW) and the other one in the lanes: a lane then owns one row of the softmax (reductions over classes are
// in-lane loops plus one half-wave exchange) and four consecutive registers are four consecutive columns of the output.
// LDS.  Operands arrive by 16-byte LDS-DMA in the order they have in memory.  Where the contraction runs along memory, fragments
// are plain 16-byte reads; where it runs across (w in DX, both in DW) they are transposing 8-byte reads, so no operand is ever
// stored transposed.  Both layouts are swizzled in 16-byte chunks (on the global address of the DMA, whose LDS side is fixed).
// A row's softmax is kept as (maximum, rest): sum of exponentials = exp(maximum) (1 + rest).  The maximum's own term never meets the
// others in one sum (CeTop), so that a confident row (rest << 1) keeps its loss to a few 2^-24 instead of 2^-24 / rest, and no loss is
// negative; the label's entry of G is expm1(-nll), so its gradient does too.  Against plain sums that is 1.5 % of a
// training step of 8192 x 65536 x 256 bf16 (1217 -> 1236 us), 0.5 % at 4096 x 131072 x 1024.
// Precision.  16-bit features enter as they are, fp32 features as two fp16 pieces under one power-of-two scale per tensor: an element
// is off by 2^-22 of itself or 2^-39 of the tensor's largest, whichever is more, and the three products hi*hi + hi*lo + lo*hi leave out
// 2^-22 of |x||w|.  Where some row's largest magnitude lies more than 17 binades below the tensor's (so that the 2^-39 would reach its 22
// bits), or anything is infinite or NaN, the operands stay fp32 and go through the fp32 matrix instruction (NATIVE; decided on the
// device, call by call: ce_pack_kernel).  Accumulation, the softmax statistics and
// the sums over splits are fp32.  G is rounded once to the operand type (bf16: 2^-8; fp16: 2^-11 relative, scaled by 2^14 so that
// probabilities down to 2^-28 keep it; fp32 features: two fp16 pieces, 2^-22 or 2^-39 of 1, NATIVE: none): the matrix cores take 16-bit operands.
#include "common.h"

namespace creste {

typedef float cef4 __attribute__((ext_vector_type(4)));
typedef float cef16 __attribute__((ext_vector_type(16)));
typedef int cei4 __attribute__((ext_vector_type(4)));
typedef short ces4 __attribute__((ext_vector_type(4)));
typedef short ces8 __attribute__((ext_vector_type(8)));
typedef _Float16 ceh8 __attribute__((ext_vector_type(8)));
typedef __bf16 ceb8 __attribute__((ext_vector_type(8)));

constexpr float kCeLog2e = 1.44269504088896341f, kCeLn2 = 0.693147180559945309f;
constexpr int kCeTile = 256;                 // classes per LOSS / GRAD tile, rows (LOSS, GRAD, DX) or classes (DW) per tile
constexpr float kCeF16Log2 = 14.f;           // G enters as G * 2^14 where it is fp16

enum { CE_LOSS, CE_GRAD, CE_DX, CE_DW };

struct CeArgs {
  const char *a, *b;                // first operand (accumulator rows), second (accumulator columns), 16-bit elements
  int64_t lda, ldb;                 // bytes between their memory rows
  int64_t pa, pb;                   // bytes between the two pieces
  int64_t ra, rb;                   // memory rows that exist (loads clamp to the last one)
  int ca, cb;                       // bytes of a memory row that exist (transposed operands: loads clamp to the last 16)
  int m, n;                         // extents of the output
  int mt, nt;                       // tiles along m, n
  int k1, ksplit;                   // contraction length; ksplit > 0: split s works [s * ksplit, + ksplit)
  // LOSS / GRAD
  const int64_t* labels;
  int class0;                       // GRAD, DX: first class of the piece
  int classes;                      // all classes
  float inv_tau;
  const float* amax;                // fp32: max|x|, max|w| (0 and 0 where `native`), native; else null
  float2* part;                     // LOSS: [class tile][n] (maximum, rest)
  float* zlab;                      // LOSS: [n] label logit, as maxima in the units of the products
  unsigned* done;                   // LOSS: the joining kernel's counter, cleared here
  // GRAD, DX, DW, per row (padded to 64): the largest product z, log2 of the sum relative to its term minus log2 of G's scale -- infinity
  // where a row does not count --, and the label's entry of G
  const float *row_max, *row_rest, *row_g;
  const int* row_lab;               // label, -1 where none applies
  char* g;                          // GRAD: [n64][ldg] elements, pieces pg bytes apart
  int64_t ldg, pg;
  int n64;
  // DX / DW
  float* partial;                   // [split][n][ldp] or null: direct
  int64_t ldp, psplit;
  int accumulate;
  void* out;
  int64_t ldo;
  int m_out;                        // feature columns of the output
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

// fp32 features whose magnitudes two fp16 pieces do not hold: the copies are plain fp32 (ce_pack_kernel decides)
template <int P>
__device__ __forceinline__ bool ce_native(const CeArgs& p) {
  if constexpr (P == 2) return p.amax[2] != 0.f;
  return false;
}

// exp2 argument of a softmax gradient: the logit against its row's largest, exactly (the kernels form both in the same order), then the rest.
// unit: power of two of the operands' products, kappa = log2(e) / tau
template <int P>
__device__ __forceinline__ float ce_exponent(float z, float unit, float mx, float kappa, float rest) {
  return fmaf(P == 2 ? fmaf(z, unit, -mx) : z - mx, kappa, -rest);
}

// dloss / (tau * count) and the powers of two of the stored operands
__device__ __forceinline__ float ce_out_scale(const CeArgs& p) {
  float s = p.gl[0] * p.inv_tau;
  if (p.mean) s = s / fmaxf(p.stat[1], 1.f);
  return s * (ce_operand_inv(p.amax, p.which) / p.gscale);
}

// join two (maximum, rest); c2: log2 units per unit of the maximum.  (-3e38, -1) is the empty sum
__device__ __forceinline__ float2 ce_merge(float2 a, float2 b, float c2) {
  const bool first = a.x >= b.x;
  const float2 u = first ? a : b, v = first ? b : a;
  return make_float2(u.x, u.y + (1.f + v.y) * __builtin_amdgcn_exp2f((v.x - u.x) * c2));
}

// A sum of exponentials as its largest term and the rest: what a row is surer of than 2^-24 is not lost beside that term.  2.5
// operations a term, where leaving out the terms that equal the maximum takes five; terms are positive (a NaN shows in the maximum)
struct CeTop {
  float t, rest;
  __device__ __forceinline__ void add(float a, float b) {
    const float lows = __builtin_amdgcn_fmed3f(t, a, b) + fminf(fminf(t, a), b);
    t = fmaxf(fmaxf(t, a), b);
    rest += lows;
  }
  __device__ __forceinline__ void add(const CeTop& v) {
    rest += v.rest + fminf(t, v.t);
    t = fmaxf(t, v.t);
  }
  // (maximum, rest) of the sum; a maximum without a term (infinite, NaN): NaN
  __device__ __forceinline__ float2 stat(float mx) const {
    return make_float2(mx, t > 0.f ? rest / t : mx == -3.0e38f ? -1.f : __builtin_nanf(""));
  }
};

// of two, NaN if one is (a NaN logit has to reach the loss)
__device__ __forceinline__ float ce_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <int DT>
__device__ __forceinline__ cef16 ce_mfma(ces8 a, ces8 b, cef16 c) {
  if constexpr (DT == CRESTE_DT_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ceb8, a), __builtin_bit_cast(ceb8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ceh8, a), __builtin_bit_cast(ceh8, b), c, 0, 0, 0);
}

// the same tile of fp32 operands, 4 floats a lane in alternate 16-byte pieces of the contraction: 8 elements of it
__device__ __forceinline__ cef16 ce_mfma_native(cef4 a, cef4 b, cef16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
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

template <int BX, int BK, bool KM, int NW>
__device__ __forceinline__ void ce_dma(char* lds, const char* base, int64_t ld, int64_t rows, int colbytes, int64_t row0, int x0,
                                       int k, int wave, int lane) {
  using L = CeTile<BX, BK, KM>;
#pragma unroll
  for (int i0 = 0; i0 < L::INSTR; i0 += NW) {
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

// a wave's own staging of 32 output rows of RB bytes (a multiple of 256): lanes write 8 or 16 bytes of "their" row, the rows leave in
// whole 256-byte runs.  16-byte chunks are swizzled by the row so that neither side meets bank conflicts
template <int RB>
__device__ __forceinline__ char* ce_stage(char* st, int row, int byte) {
  return st + row * RB + ((((byte >> 4) ^ (row & 15)) << 4) | (byte & 15));
}

// the wave's MT x NT accumulator tiles (registers = feature columns from d0, lanes = output rows from row0) to the output or the
// split's partial sums, 128 columns of 32 rows at a time through the wave's 16 KB of LDS at st
template <int DT, int MT, int NT>
__device__ __forceinline__ void ce_store(const CeArgs& p, const cef16 (&acc)[MT][NT], char* st, int row0, int d0, int split, int lane) {
  constexpr int TP = MT < 4 ? MT : 4, RB = TP * 128, LPR = RB / 16;      // tiles a pass, bytes and lanes of a row
  static_assert(MT % TP == 0 && (LPR == 32 || LPR == 16), "");
  const int li = lane & 31, lh = lane >> 5;
  const float fs = p.partial ? 1.f : ce_out_scale(p);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int h = 0; h < MT / TP; ++h) {
#pragma unroll
      for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const cef16& a = acc[h * TP + i][j];
          *reinterpret_cast<cef4*>(ce_stage<RB>(st, li, (i * 32 + 8 * q + 4 * lh) * 4)) =
              cef4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
        }
      __builtin_amdgcn_wave_barrier();                  // (a wave's LDS operations stay in order)
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 64 / LPR) {       // whole rows
        const int r = r0 + lane / LPR, row = row0 + j * 32 + r, c = lane % LPR, d = d0 + h * (TP * 32) + c * 4;
        cef4 v = *reinterpret_cast<const cef4*>(ce_stage<RB>(st, r, c * 16));
        if (row >= p.n || d >= p.m_out) continue;
        if (p.partial) {                                // rows of partials are padded to 4
          cef4* dst = reinterpret_cast<cef4*>(p.partial + split * p.psplit + row * p.ldp + d);
          *dst = p.accumulate ? *dst + v : v;
          continue;
        }
        v *= fs;
        const int64_t o = row * p.ldo + d;
        if ((p.m_out & 3) == 0) {
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
            if (d + e >= p.m_out) continue;
            if (p.out_dt == CRESTE_DT_F32) ((float*)p.out)[o + e] = v[e];
            else ((short*)p.out)[o + e] = ce_cvt<DT>(v[e]);
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
}

// The shape of a workgroup: tile BM x BN by WM x WN waves, BK / P contraction elements a stage, NS stages in LDS
template <int BM_, int BN_, int WM_, int WN_, int BK_, int NS_>
struct CeShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, NS = NS_, NW = WM * WN;
};

// DT: 16-bit operand type (fp16 for two-piece fp32), P: pieces.  Bound: matrix rate, and for DX / DW reading G.  4096 x 131072 x 1024 bf16:
// LOSS 1050-1140 us (1000 TF/s), and for each of eight pieces of 16384 classes GRAD 160, DX 155-175, DW 140-150 us (780-980 TF/s)
template <int MODE, int DT, int P, typename S, bool NATIVE>
__device__ __forceinline__ void ce_gemm_body(const CeArgs& p) {
  constexpr bool AKM = MODE == CE_DX || MODE == CE_DW, BKM = MODE == CE_DW;
  constexpr int BM = S::BM, BN = S::BN, BK = S::BK / P, NS = S::NS, NW = S::NW, WTM = BM / S::WM, WTN = BN / S::WN;
  constexpr int MT = WTM / 32, NT = WTN / 32;
  using LA = CeTile<BM, BK, AKM>;
  using LB = CeTile<BN, BK, BKM>;
  constexpr int STAGE = P * (LA::BYTES + LB::BYTES), kDma = STAGE / 1024 / NW;
  static_assert(LA::INSTR % NW == 0 && LB::INSTR % NW == 0, "every wave issues as many loads");
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, lh = lane >> 5;
  const int wm = wave / S::WN, wn = wave % S::WN;
  if constexpr (MODE == CE_LOSS)
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;
  int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tm = t % p.mt;
  t /= p.mt;
  const int tn = t % p.nt, split = t / p.nt;
  const int m0 = tm * BM, n0 = tn * BN;
  const int kb = split * p.ksplit;
  const int ke = p.ksplit ? min(p.k1, kb + p.ksplit) : p.k1;

  cef16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  if constexpr (NATIVE) {
    // 8 elements of the contraction a step, half a wave 4 of them: one 16-byte load where it runs along memory, four rows where across
    auto load = [&](const char* base, int64_t ld, int64_t rows, int cols, bool across, int x, int k) __attribute__((always_inline)) {
      cef4 v;
      if (!across) return *reinterpret_cast<const cef4*>(base + (x < rows ? x : rows - 1) * 2 * ld + (k + 4 * lh) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t r = k + 4 * lh + e;
        v[e] = *reinterpret_cast<const float*>(base + (r < rows ? r : rows - 1) * 2 * ld + (x < cols ? x : cols - 1) * 4);
      }
      return v;
    };
    // (columns of the output that are not there, most of them where there are few rows, stay 0)
    const int nw = n0 + wn * WTN, cols = nw >= p.n ? 0 : p.n - nw;
    const char* const first = p.a + (MODE == CE_GRAD || MODE == CE_DX ? p.class0 * p.lda : 0);      // (the piece's: rows are twice as long)
    // steps in flight (a step's loads take longer than its products): a training step of 16 x 65536 x 512 394 us with one, 353 with two, 363
    // with four, whose registers also cost a large uneven one (4096 x 65536 x 256: 6565 -> 7384)
    constexpr int AHEAD = 2;
    cef4 a[AHEAD][MT], b[AHEAD][NT];
    auto fetch = [&](int k, int at) __attribute__((always_inline)) {
      k = k < ke ? k : ke - 8;
#pragma unroll
      for (int i = 0; i < MT; ++i) a[at][i] = load(first, p.lda, p.ra, p.ca / 2, AKM, m0 + wm * WTM + i * 32 + li, k);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (cols > j * 32) b[at][j] = load(p.b, p.ldb, p.rb, p.cb / 2, BKM, nw + j * 32 + li, k);
    };
    if (cols > 0 && kb < ke) {                          // (whole 64 elements, hence whole rounds of AHEAD steps)
#pragma unroll
      for (int h = 0; h < AHEAD; ++h) fetch(kb + h * 8, h);
      for (int k = kb; k < ke; k += AHEAD * 8)
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (cols <= j * 32) break;
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j] = ce_mfma_native(a[h][i], b[h][j], acc[i][j]);
          }
          fetch(k + (h + AHEAD) * 8, h);
        }
    }
  }
  auto dma = [&](int k, int s) __attribute__((always_inline)) {
    char* st = smem + s * STAGE;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      ce_dma<BM, BK, AKM, NW>(st + q * LA::BYTES, p.a + q * p.pa, p.lda, p.ra, p.ca, m0, m0, k, wave, lane);
      ce_dma<BN, BK, BKM, NW>(st + P * LA::BYTES + q * LB::BYTES, p.b + q * p.pb, p.ldb, p.rb, p.cb, n0, n0, k, wave, lane);
    }
  };
  const int n = !NATIVE && ke > kb ? (ke - kb) / BK : 0;
#pragma unroll
  for (int s = 0; s < NS - 1; ++s)
    if (s < n) dma(kb + s * BK, s);
  int cur = 0, nxt = NS - 1;                            // stage in use, stage to fill
  for (int c = 0; c < n; ++c) {
    // this wave's loads of stage c have landed (younger ones: the NS - 2 stages behind it) -- and, past the barrier, everybody's;
    // everybody has also left stage c - 1, which is the one to fill
    if (NS > 2 && c + NS - 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * kDma) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (c + NS - 1 < n) dma(kb + (c + NS - 1) * BK, nxt);
    const char* A = smem + cur * STAGE;
    const char* B = A + P * LA::BYTES;
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      ces8 af[P][MT], bf[P][NT];
#pragma unroll
      for (int q = 0; q < P; ++q) {
#pragma unroll
        for (int i = 0; i < MT; ++i) af[q][i] = ce_frag<BM, BK, AKM>(A + q * LA::BYTES, wm * WTM + i * 32, kk, lane);
#pragma unroll
        for (int j = 0; j < NT; ++j) bf[q][j] = ce_frag<BN, BK, BKM>(B + q * LB::BYTES, wn * WTN + j * 32, kk, lane);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (P == 2) {                       // small products first
            acc[i][j] = ce_mfma<DT>(af[1][i], bf[0][j], acc[i][j]);
            acc[i][j] = ce_mfma<DT>(af[0][i], bf[1][j], acc[i][j]);
          }
          acc[i][j] = ce_mfma<DT>(af[0][i], bf[0][j], acc[i][j]);
        }
    }
    cur = cur + 1 == NS ? 0 : cur + 1;
    nxt = nxt + 1 == NS ? 0 : nxt + 1;
  }
  __syncthreads();                                      // the stages are free

  if constexpr (MODE == CE_LOSS || MODE == CE_GRAD) {
    const float unit = ce_operand_inv(p.amax, 0) * ce_operand_inv(p.amax, 1), c2 = unit * p.inv_tau * kCeLog2e, kappa = p.inv_tau * kCeLog2e;
    const int mw = m0 + wm * WTM;                       // first class of this wave, within the piece
    if constexpr (MODE == CE_LOSS) {
      float2* sh = reinterpret_cast<float2*>(smem);     // [wm][BN rows]
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = n0 + wn * WTN + j * 32 + li;
        // the label's class relative to this wave's first one (a label outside [0, classes) matches nothing)
        const int64_t y = row < p.n ? p.labels[row] : -1;
        const int64_t yr = y - mw;
        const int lab = y >= 0 && y < p.classes && yr >= 0 && yr < WTM ? (int)yr : -1;
        float mx = -3.0e38f, z = 0.f;                   // (a half tile without classes: the empty sum)
        if (mw + WTM > p.m) {                        // classes behind the last one: exp2 gives 0
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (mw + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh >= p.m) acc[i][j][r] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = ce_max(mx, acc[i][j][r]);
        if (__any(lab >= 0)) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = i * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh == lab ? acc[i][j][r] : z;
        }
        CeTop top[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 16; r += 2)
            top[(r >> 1) & 1].add(__builtin_amdgcn_exp2f((acc[i][j][r] - mx) * c2), __builtin_amdgcn_exp2f((acc[i][j][r + 1] - mx) * c2));
        top[0].add(top[1]);
        float2 st = top[0].stat(mx);
        st = ce_merge(st, make_float2(__shfl_xor(st.x, 32, 64), __shfl_xor(st.y, 32, 64)), c2);
        if (lh == 0) sh[wm * BN + wn * WTN + j * 32 + li] = st;
        if (lab >= 0 && ((lab >> 2) & 1) == lh) p.zlab[row] = z;
      }
      __syncthreads();
      const int i = threadIdx.x;
      static_assert(S::WM == 2, "");
      if (i < BN && n0 + i < p.n) p.part[(int64_t)tm * p.n + n0 + i] = ce_merge(sh[i], sh[BN + i], c2);
    } else {
      constexpr int RB = WTM * 2;
      static_assert(RB == 256 && NW * P * 32 * RB <= NS * STAGE, "");
      char* st = smem + wave * (P * 32 * RB);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = n0 + wn * WTN + j * 32 + li;
        const float mx = row < p.n64 ? p.row_max[row] : 0.f, rest = row < p.n64 ? p.row_rest[row] : INFINITY,
                    gl = row < p.n64 ? p.row_g[row] : 0.f;
        const int yr = (row < p.n64 ? p.row_lab[row] : -1) - p.class0 - mw;
        const bool any = __any(yr >= 0 && yr < WTM);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int cl = i * 32 + 8 * q + 4 * lh;
            ces4 hi, lo;
            cef4 whole;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = __builtin_amdgcn_exp2f(ce_exponent<P>(acc[i][j][4 * q + e], unit, mx, kappa, rest));
              if (any) v = cl + e == yr ? gl : v;
              if (mw + WTM > p.m) v = mw + cl + e < p.m ? v : 0.f;
              whole[e] = v;
              const short h = ce_cvt<DT>(v);
              hi[e] = h;
              if constexpr (P == 2) lo[e] = ce_cvt<DT>(v - (float)__builtin_bit_cast(_Float16, h));
            }
            if constexpr (NATIVE) {
              if (row < p.n64) *reinterpret_cast<cef4*>(p.g + row * 2 * p.ldg + (mw + cl) * 4ll) = whole;
              continue;
            }
            *reinterpret_cast<ces4*>(ce_stage<RB>(st, li, cl * 2)) = hi;
            if constexpr (P == 2) *reinterpret_cast<ces4*>(ce_stage<RB>(st + 32 * RB, li, cl * 2)) = lo;
          }
        if constexpr (NATIVE) continue;
        __builtin_amdgcn_wave_barrier();                // (a wave's LDS operations stay in order)
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 4) {          // 4 rows of 256 bytes per instruction
            const int r = r0 + (lane >> 4), c = (lane & 15) * 16;
            const int orow = n0 + wn * WTN + j * 32 + r;
            const cef4 v = *reinterpret_cast<const cef4*>(ce_stage<RB>(st + q * 32 * RB, r, c));
            if (orow < p.n64) *reinterpret_cast<cef4*>(p.g + q * p.pg + orow * p.ldg + (int64_t)mw * 2 + c) = v;
          }
        __builtin_amdgcn_wave_barrier();
      }
    }
  } else {
    static_assert(NW * 32 * 512 <= NS * STAGE, "");
    ce_store<DT, MT, NT>(p, acc, smem + wave * (32 * 512), n0 + wn * WTN, m0 + wm * WTM, split, lane);
  }
}

template <int MODE, int DT, int P, typename S>
__global__ __launch_bounds__(S::NW * 64, 2) void ce_gemm_kernel(CeArgs p) {
  if (ce_native<P>(p)) {
    if constexpr (P == 2) ce_gemm_body<MODE, DT, P, S, true>(p);
  } else {
    ce_gemm_body<MODE, DT, P, S, false>(p);
  }
}

// -------------------------------------------------------------------------------------------- up to 256 feature columns
// The features of a workgroup's OWN items (rows for LOSS and DX, classes for DW) fit in registers, so the other side is streamed past
// them once: per 32 others a wave forms z (others in the accumulator registers, its own items in the lanes), turns it into G in
// place and feeds G, still in registers, to the second product -- no G in memory at all, no second kernel.  What makes that free
// of exchanges: the contraction of the second product may run over the others in any order, so the transposing reads of the
// streamed tile take them in the order in which the accumulator holds them.  One tile in LDS serves both products (rows for z,
// transposed for the second), its 16-byte chunks swizzled by the row: a bijection over 16 rows for the row reads, different 64-byte
// windows for the 4 rows of a transposing read.
// Bound: matrix rate, then the exponentials beside it.  8192 x 65536 x 256 bf16: loss 270-290 us (980 TF/s), both gradients 1060-1170 us
// (8NVD, 940-1040 TF/s; a large library product: 1216).  19584 x 4096 x 128 fp32: 75 and 257 us (820 and 960 TF/s of fp16 products).
// Against the tiled product with G in memory: 1845 -> 1236 us and 596 -> 341 us for the whole step.
template <int DP, int OTS, int P>
struct CeStream {
  static constexpr int ROWB = DP * 2, CPR = ROWB / 16, PIECE = OTS * ROWB, INFO = P * PIECE, BYTES = INFO + 1024, INSTR = PIECE / 1024;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (CPR >= 16) return (r & 3) << 2 | ((r >> 2) & 3);
    else return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);   // two rows per 256 bytes
  }
  static constexpr int RPI = 64 / CPR;       // rows an instruction covers; instruction i + 8 covers the rows 8 * RPI further, whose
                                             // swizzle is the same: one lane offset serves all of a wave's instructions
  static __device__ __forceinline__ void dma(char* lds, const CeArgs& p, int64_t o0, int wave, int lane) {
    const int r0 = wave * RPI + lane / CPR, c = (lane % CPR) ^ swz(r0);
    const unsigned off = (unsigned)r0 * (unsigned)p.lda + c * 16;
    const bool inside = o0 + OTS <= p.ra;
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int i0 = 0; i0 < INSTR; i0 += 8) {
        const char* base = p.a + q * p.pa + (o0 + i0 * RPI) * p.lda;
        const char* src = base + off;
        if (!inside) {                       // rows behind the last one: the last one again
          const int64_t row = o0 + i0 * RPI + r0 < p.ra ? o0 + i0 * RPI + r0 : p.ra - 1;
          src = p.a + q * p.pa + row * p.lda + c * 16;
        }
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                         (__attribute__((address_space(3))) void*)(lds + q * PIECE + (i0 + wave) * 1024), 16, 0, 0);
      }
  }
  // Fragment addresses: what depends on the lane alone, then exclusive-or with what the step selects (the selecting bits are those
  // of the chunk, above them every term is a multiple of the row size)
  static __device__ __forceinline__ unsigned row_base(int lane) {
    const int r = lane & 31;
    return r * ROWB + (((lane >> 5) ^ swz(r)) << 4);
  }
  static __device__ __forceinline__ ces8 row(const char* smem, unsigned base, int kk) {
    return *reinterpret_cast<const ces8*>(smem + ((base ^ ((kk & 7) << 5)) + (kk >> 3) * 256));
  }
  // 16 others in the accumulator's order: of a half wave the 4 * lh .. and the 8 + 4 * lh .., feature columns d * 32 ..
  static __device__ __forceinline__ unsigned across_base(int lane) {
    const int l = lane & 15, g = lane >> 4, r = 4 * (g >> 1) + (l >> 2);
    return r * ROWB + (((2 * (g & 1) + ((l & 3) >> 1)) ^ swz(r)) << 4) + (l & 1) * 8;
  }
  static __device__ __forceinline__ ces8 across(const char* smem, unsigned base, int d) {
    ces8 v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* at = smem + (((base + j * 8 * ROWB) ^ (((d & 3) << 6) | j << 5)) + (d >> 2) * 256);
      const ces4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ces4*)at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * j + e] = t[e];
    }
    return v;
  }
  // DW: what a row brings along, behind the features (every wave issues as many loads: some twice)
  static __device__ __forceinline__ void dma_info(char* lds, const CeArgs& p, int64_t o0, int wave, int lane) {
    static_assert(OTS == 64, "one 4-byte load per lane");
    const int which = wave & 3;
    const char* src = which == 3 ? (const char*)p.row_g : which == 2 ? (const char*)p.row_rest : which ? (const char*)p.row_lab : (const char*)p.row_max;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + (o0 + lane) * 4),
                                     (__attribute__((address_space(3))) void*)(lds + INFO + which * 256), 4, 0, 0);
  }
};

constexpr int kCeStage = 64;                 // others per stage
constexpr int kAhead = 4;                    // (8192 x 65536 x 256 bf16 training step: 1206 us with the compiler's own order, 1189 with 4)

// order of the region in front: kAhead LDS reads, then matrix instructions with the remaining reads spread between them
template <int READS, int MFMAS>
__device__ __forceinline__ void ce_interleave() {
  constexpr int A = kAhead < READS ? kAhead : READS, REST = READS - A;
  __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
    for (int r = i * REST / MFMAS; r < (i + 1) * REST / MFMAS; ++r) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
}

// a = the streamed side (p.m items), b = the own side (p.n items), NT x 32 own items per wave
template <int MODE, int DT, int P, int DP, int NT, bool NATIVE>
__device__ __forceinline__ void ce_stream_body(const CeArgs& p, int block, int blocks) {
  using L = CeStream<DP, kCeStage, P>;
  constexpr int NS = 3, KS = DP / 16, kDma = P * L::INSTR / 8 + (MODE == CE_DW);
  extern __shared__ __align__(1024) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, lh = lane >> 5;
  if constexpr (MODE == CE_LOSS)
    if (block == 0 && threadIdx.x == 0) *p.done = 0;
  const int t = xcd_remap(block, blocks);
  const int tn = t % p.nt, split = t / p.nt;
  const int own0 = tn * (256 * NT) + wave * (32 * NT);
  const int kb = split * p.ksplit, ke = min(p.k1, kb + p.ksplit);
  const int n = ke > kb ? (ke - kb + kCeStage - 1) / kCeStage : 0;

  ces8 x[P][NT][KS];
  cef4 xn[NT][DP / 8];                       // native: 4 floats of every 8
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t o = own0 + j * 32 + li, row = o < p.n ? o : p.n - 1;
    if constexpr (NATIVE) {
#pragma unroll
      for (int kk = 0; kk < DP / 8; ++kk) xn[j][kk] = *reinterpret_cast<const cef4*>(p.b + row * 2 * p.ldb + kk * 32 + lh * 16);
      continue;
    }
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) x[q][j][kk] = *reinterpret_cast<const ces8*>(p.b + q * p.pb + row * p.ldb + kk * 32 + lh * 16);
  }
  const float unit = ce_operand_inv(p.amax, 0) * ce_operand_inv(p.amax, 1), c2 = unit * p.inv_tau * kCeLog2e, kappa = p.inv_tau * kCeLog2e;
  // LOSS: the maximum mx so far, the sum of exp2((z - near) c2) as two tops; near follows the maximum in steps, when a logit passes `lim`
  // (8 above: such an exponent is off by 2^-22)
  float rest[NT], gl[NT], mx[NT], zl[NT], near[NT], lim[NT];
  CeTop top[NT][2];
  int lab[NT];                               // LOSS / DX: the row's label; DW: the own class
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int o = own0 + j * 32 + li;
    mx[j] = -3.0e38f;
    lim[j] = -INFINITY;
    near[j] = -3.0e38f;
    top[j][0] = top[j][1] = CeTop{0.f, 0.f};
    zl[j] = rest[j] = gl[j] = 0.f;
    lab[j] = o;
    if constexpr (MODE == CE_LOSS) {
      const int64_t y = o < p.n ? p.labels[o] : -1;
      lab[j] = y >= 0 && y < p.classes ? (int)y : -1;
    }
    if constexpr (MODE == CE_DX) {
      mx[j] = o < p.n ? p.row_max[o] : 0.f;
      rest[j] = o < p.n ? p.row_rest[o] : INFINITY;
      gl[j] = o < p.n ? p.row_g[o] : 0.f;
      lab[j] = o < p.n ? p.row_lab[o] : -1;
    }
  }
  constexpr int AT = MODE == CE_LOSS ? 1 : DP / 32, AN = MODE == CE_LOSS ? 1 : NT;
  cef16 acc[AT][AN];
#pragma unroll
  for (int d = 0; d < AT; ++d)
#pragma unroll
    for (int j = 0; j < AN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][j][r] = 0.f;

  auto fill = [&](int c, int s) __attribute__((always_inline)) {
    L::dma(smem + s * L::BYTES, p, kb + c * kCeStage, wave, lane);
    if constexpr (MODE == CE_DW) L::dma_info(smem + s * L::BYTES, p, kb + c * kCeStage, wave, lane);
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (the counted waits below count stages only)
  if constexpr (!NATIVE) {
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
      if (s < n) fill(s, s);
  }
  const unsigned rbase = L::row_base(lane), abase = L::across_base(lane);
  int cur = 0, nxt = NS - 1;
  for (int c = 0; c < n; ++c) {
    if constexpr (!NATIVE) {
      if (c + NS - 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * kDma) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (c + NS - 1 < n) fill(c + NS - 1, nxt);
    }
    const char* st = smem + cur * L::BYTES;             // (the rows' values behind the features)
#pragma unroll 1
    for (int sub = 0; sub < kCeStage / 32; ++sub) {
      const int o0 = kb + c * kCeStage + sub * 32;      // first other of this half stage
      const unsigned stage = cur * L::BYTES + sub * 32 * L::ROWB;
      cef16 z[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) z[j][r] = 0.f;
      if constexpr (NATIVE) {
        const int64_t other = o0 + li < p.ra ? o0 + li : p.ra - 1;
#pragma unroll
        for (int kk = 0; kk < DP / 8; ++kk) {
          const cef4 a = *reinterpret_cast<const cef4*>(p.a + other * 2 * p.lda + kk * 32 + lh * 16);
#pragma unroll
          for (int j = 0; j < NT; ++j) z[j] = ce_mfma_native(a, xn[j][kk], z[j]);
        }
      } else {
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        ces8 a[P];
#pragma unroll
        for (int q = 0; q < P; ++q) a[q] = L::row(smem, stage + q * L::PIECE + rbase, kk);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (P == 2) {                       // w's low piece first on either side: the same sums
            z[j] = MODE == CE_DW ? ce_mfma<DT>(a[0], x[1][j][kk], z[j]) : ce_mfma<DT>(a[1], x[0][j][kk], z[j]);
            z[j] = MODE == CE_DW ? ce_mfma<DT>(a[1], x[0][j][kk], z[j]) : ce_mfma<DT>(a[0], x[1][j][kk], z[j]);
          }
          z[j] = ce_mfma<DT>(a[0], x[0][j][kk], z[j]);
        }
      }
      ce_interleave<KS * P, NT * (P == 2 ? 3 : 1) * KS>();
      }
      __builtin_amdgcn_sched_barrier(0);                // (the phases' operands do not fit the registers side by side)
      const bool edge = o0 + 32 > p.m;                  // others behind the last one
      ces8 g[P][NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (edge && MODE != CE_DW)                      // (DW: such rows have rest = infinity)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (o0 + (r & 3) + 8 * (r >> 2) + 4 * lh >= p.m) z[j][r] = -INFINITY;
        if constexpr (MODE == CE_LOSS) {
          const int rel = lab[j] - o0;
          if (__any(rel >= 0 && rel < 32))
#pragma unroll
            for (int r = 0; r < 16; ++r) zl[j] = (r & 3) + 8 * (r >> 2) + 4 * lh == rel ? z[j][r] : zl[j];
          float m = z[j][0];
#pragma unroll
          for (int r = 1; r < 16; ++r) m = ce_max(m, z[j][r]);
          if (__any(m > lim[j])) {
            if (m > lim[j]) {
              const float by = __builtin_amdgcn_exp2f((near[j] - m) * c2);      // (nothing summed yet: 0 or 1 times 0)
#pragma unroll
              for (int h = 0; h < 2; ++h) top[j][h] = CeTop{top[j][h].t * by, top[j][h].rest * by};
              near[j] = m;
              lim[j] = m + 8.f / c2;
            }
          }
#pragma unroll
          for (int r = 0; r < 16; r += 2)
            top[j][(r >> 1) & 1].add(__builtin_amdgcn_exp2f((z[j][r] - near[j]) * c2), __builtin_amdgcn_exp2f((z[j][r + 1] - near[j]) * c2));
          mx[j] = ce_max(mx[j], m);
        } else {
          float v[16];
          // DW: what the others, rows here (padded to whole stages), brought along: 4 of word `which`
          auto info = [&](int which, int q) __attribute__((always_inline)) {
            const int at = sub * 32 + 8 * q + 4 * lh;
            cei4 w4;
            if constexpr (NATIVE) {
              const int* src = which == 3 ? (const int*)p.row_g : which == 2 ? (const int*)p.row_rest : which ? p.row_lab : (const int*)p.row_max;
#pragma unroll
              for (int e = 0; e < 4; ++e) w4[e] = src[kb + c * kCeStage + at + e];
            } else {
              w4 = *reinterpret_cast<const cei4*>(st + L::INFO + which * 256 + at * 4);
            }
            return w4;
          };
          bool hit = false;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            cef4 rm, rr;
            if constexpr (MODE == CE_DW) {
              rm = __builtin_bit_cast(cef4, info(0, q));
              rr = __builtin_bit_cast(cef4, info(2, q));
              const cei4 rb = info(1, q);
              hit |= rb[0] == lab[j] || rb[1] == lab[j] || rb[2] == lab[j] || rb[3] == lab[j];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[4 * q + e] = __builtin_amdgcn_exp2f(
                  ce_exponent<P>(z[j][4 * q + e], unit, MODE == CE_DW ? rm[e] : mx[j], kappa, MODE == CE_DW ? rr[e] : rest[j]));
          }
          if constexpr (MODE == CE_DW) {
            if (__any(hit))
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const cei4 rb = info(1, q);
                const cef4 rg = __builtin_bit_cast(cef4, info(3, q));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * q + e] = rb[e] == lab[j] ? rg[e] : v[4 * q + e];
              }
          }
          if constexpr (MODE == CE_DX) {
            const int rel = lab[j] - o0;
            if (__any(rel >= 0 && rel < 32))
#pragma unroll
              for (int r = 0; r < 16; ++r) v[r] = (r & 3) + 8 * (r >> 2) + 4 * lh == rel ? gl[j] : v[r];
          }
          if constexpr (NATIVE) {                       // register r holds the others 8 (r / 4) + r % 4 of either half
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int64_t o = o0 + (r & 3) + 8 * (r >> 2) + 4 * lh;
              const float* at = reinterpret_cast<const float*>(p.a + (o < p.ra ? o : p.ra - 1) * 2 * p.lda) + li;
#pragma unroll
              for (int d = 0; d < AT; ++d) acc[d][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(at[d * 32], v[r], acc[d][j], 0, 0, 0);
            }
            continue;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const short h = ce_cvt<DT>(v[r]);
            g[0][j][r >> 3][r & 7] = h;
            if constexpr (P == 2) g[P - 1][j][r >> 3][r & 7] = ce_cvt<DT>(v[r] - (float)__builtin_bit_cast(_Float16, h));
          }
        }
      }
      if constexpr (MODE != CE_LOSS && !NATIVE) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < AT; ++d)
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            ces8 a[P];
#pragma unroll
            for (int q = 0; q < P; ++q) a[q] = L::across(smem, stage + q * L::PIECE + k2 * 16 * L::ROWB + abase, d);
#pragma unroll
            for (int j = 0; j < AN; ++j) {
              if constexpr (P == 2) {
                acc[d][j] = ce_mfma<DT>(a[1], g[0][j][k2], acc[d][j]);
                acc[d][j] = ce_mfma<DT>(a[0], g[P - 1][j][k2], acc[d][j]);
              }
              acc[d][j] = ce_mfma<DT>(a[0], g[0][j][k2], acc[d][j]);
            }
          }
        ce_interleave<AT * 4 * P, AN * (P == 2 ? 3 : 1) * AT * 2>();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    cur = cur + 1 == NS ? 0 : cur + 1;
    nxt = nxt + 1 == NS ? 0 : nxt + 1;
  }
  if constexpr (MODE == CE_LOSS) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int row = own0 + j * 32 + li;
      top[j][0].add(top[j][1]);
      const float2 mine = top[j][0].stat(mx[j]);
      const float2 m = ce_merge(mine, make_float2(__shfl_xor(mine.x, 32, 64), __shfl_xor(mine.y, 32, 64)), c2);
      if (row >= p.n) continue;
      if (lh == 0) p.part[(int64_t)split * p.n + row] = m;
      if (lab[j] >= kb && lab[j] < ke && ((lab[j] >> 2) & 1) == lh) p.zlab[row] = zl[j];
    }
  } else {
    __syncthreads();
    ce_store<DT, DP / 32, NT>(p, acc, smem + wave * (32 * 512), own0, 0, split, lane);
  }
}

// own items per wave / 32: two where the registers hold them (for LOSS their features alone)
constexpr int ce_nt(int mode, int P, int DP) { return P == 1 && (mode == CE_LOSS || DP == 64) ? 2 : 1; }

template <int MODE, int DT, int P, int DP>
__device__ __forceinline__ void ce_stream_either(const CeArgs& p, int block, int blocks) {
  if (ce_native<P>(p)) {
    if constexpr (P == 2) ce_stream_body<MODE, DT, P, DP, ce_nt(MODE, P, DP), true>(p, block, blocks);
  } else {
    ce_stream_body<MODE, DT, P, DP, ce_nt(MODE, P, DP), false>(p, block, blocks);
  }
}

template <int DT, int P, int DP>
__global__ __launch_bounds__(512, 2) void ce_loss_kernel(CeArgs p) {
  ce_stream_either<CE_LOSS, DT, P, DP>(p, blockIdx.x, gridDim.x);
}

// both gradients in one launch, the first nx workgroups dx: small problems leave CUs to each other
template <int DT, int P, int DP>
__global__ __launch_bounds__(512, 2) void ce_grad_kernel(CeArgs dx, CeArgs dw, int nx) {
  if ((int)blockIdx.x < nx) ce_stream_either<CE_DX, DT, P, DP>(dx, blockIdx.x, nx);
  else ce_stream_either<CE_DW, DT, P, DP>(dw, blockIdx.x - nx, gridDim.x - nx);
}

// ------------------------------------------------------------------------------------------------------- few rows
// LOSS for at most 32 rows: bound by reading w once, so no LDS and no copy of the operands -- a wave streams 64 classes from
// memory straight into the matrix instructions, one group of loads (128 bytes of each class row) ahead.  fp32 goes through
// the fp32 matrix instruction (32 x 32 x 2, 157 TF: 32 rows need 16 products a loaded element, well below it).  The lane
// halves take alternate 16-byte pieces of the contraction in both operands, which for fp32 makes a 16-byte load feed four instructions.
// 16 x 65536 x 512 fp32: 30 us, 4.5 TB/s (through copies and the streaming kernel: 152 us for the whole call, now 43)
// Whole calls of 16 x 65536 x 512 fp32 / 8 x 100000 x 1024 bf16, back to back: 37 / 61 us; 8 waves of 32 classes 44 / 57, workgroups of
// 128 classes 52 / 58, of 64 classes 42 / 59
template <int DT>
__global__ __launch_bounds__(256) void ce_few_kernel(CeArgs p, int D) {
  constexpr int EB = DT == CRESTE_DT_F32 ? 4 : 2, STEP = 32 / EB;      // elements both halves take per load
  typedef int iv4 __attribute__((ext_vector_type(4)));
  __shared__ float2 sh[4][32];
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;
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
  mx = fmaxf(mx, -3.0e38f);
  float own = -1.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float t = acc[i][r] - mx;
      sum += t == 0.f ? 0.f : __builtin_amdgcn_exp2f(t * c2);
      own += t == 0.f ? 1.f : 0.f;
    }
  float2 st = make_float2(mx, sum + own);
  st = ce_merge(st, make_float2(__shfl_xor(st.x, 32, 64), __shfl_xor(st.y, 32, 64)), c2);
  if (lh == 0) sh[wave][li] = st;
  if (lab >= 0 && ((lab >> 2) & 1) == lh) p.zlab[li] = z;
  __syncthreads();
  if (threadIdx.x < 32 && (int)threadIdx.x < p.n) {
    for (int j = 1; j < 4; ++j) st = ce_merge(st, sh[j][li], c2);
    p.part[(int64_t)blockIdx.x * p.n + li] = st;
  }
}

// ---------------------------------------------------------------------------------------------------- small kernels
// both operands at once: blocks below `split` take the first, the others the second.  Rows of x that do not count are taken as zeros,
// whatever they hold (0 * NaN would reach dw, a large value fp32's scale): named by their labels, behind the forward by the infinite
// rest it left
struct CeSide {
  const void* x;
  int64_t rows, ld;
  short* out;
  int64_t piece;
  const int64_t* labels;
  int64_t ignore;
  const float* counts;
  __device__ __forceinline__ bool off(int64_t r) const { return labels ? labels[r] == ignore : counts && counts[r] == INFINITY; }
};

// What the blocks of ce_amax_kernel leave of an operand: max |x|, and the smallest exponent of a row's largest magnitude (rows of zeros
// aside; 255: none)
struct CeMax { unsigned bits; int low; };

__device__ __forceinline__ CeMax ce_max_join(CeMax a, CeMax b) { return CeMax{max(a.bits, b.bits), min(a.low, b.low)}; }

// over the 256 threads of a block
__device__ __forceinline__ CeMax ce_max_block(CeMax m, CeMax (&sh)[4]) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = ce_max_join(m, CeMax{(unsigned)__shfl_xor((int)m.bits, o, 64), __shfl_xor(m.low, o, 64)});
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  return ce_max_join(ce_max_join(sh[0], sh[1]), ce_max_join(sh[2], sh[3]));
}

// Each 16 lanes take whole rows, 4 columns a lane and step (no division by the row length).  Magnitudes as bit patterns: they order
// alike, and a NaN counts as the largest
__global__ __launch_bounds__(256) void ce_amax_kernel(CeSide u, CeSide v, int cols, int split, unsigned* __restrict__ bmax,
                                                      uint8_t* __restrict__ blow) {
  __shared__ CeMax sh[4];
  const bool second = (int)blockIdx.x >= split;
  const CeSide s = second ? v : u;
  const int blk = second ? blockIdx.x - split : blockIdx.x, nb = second ? gridDim.x - split : split;
  const int c0 = (threadIdx.x & 15) * 4;
  CeMax m{0, 255};
  for (int64_t r = (int64_t)blk * 16 + (threadIdx.x >> 4); r < s.rows; r += (int64_t)nb * 16) {
    const unsigned* x = (const unsigned*)s.x + r * s.ld;
    if (s.off(r)) continue;
    unsigned row = 0;
    for (int c = c0; c < cols; c += 64)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < cols) row = max(row, x[c + e] & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) row = max(row, (unsigned)__shfl_xor((int)row, o, 64));      // (the 16 lanes of a row are here together)
    m = ce_max_join(m, CeMax{row, row ? (int)(row >> 23) : 255});
  }
  m = ce_max_block(m, sh);
  if (threadIdx.x == 0) {
    bmax[blockIdx.x] = m.bits;
    blow[blockIdx.x] = (uint8_t)m.low;
  }
}

// Do two fp16 pieces under one power of two hold an operand's rows to 22 bits of each row's largest magnitude?  That magnitude may lie 17
// binades below the tensor's (its low piece's steps are 2^-24 where the tensor's largest is 2^14 .. 2^15), nothing may be infinite or
// NaN, and the tensor's largest not so small that no power of two brings it there
__device__ __forceinline__ bool ce_even(CeMax m) {
  const int e = m.bits >> 23;
  return m.bits == 0 || (e >= 15 && e < 255 && e - m.low <= 17);
}

// 16-bit copy of the features with rows of cp (a multiple of 64) elements, zero behind the last column.  fp32: two pieces under
// the power of two of the operand's max |x| (from the na0 + na1 blocks' maxima; left in amax[0 / 1]).  Where that does not hold either
// operand's rows (ce_even), or the logits' unit leaves fp32's range, the copies are fp32 and amax[2] says so: the kernels then multiply
// with the fp32 matrix instruction.  Pieces / one row 10^9 times the others, us a step: 19584 x 4096 x 128 376 / 1194, 4096 x 65536 x 256
// 2062 / 6610
template <typename T>
__global__ __launch_bounds__(256) void ce_pack_kernel(CeSide u, CeSide v, int cols, int cp, int split, const unsigned* __restrict__ bmax,
                                                      const uint8_t* __restrict__ blow, int na0, int na1, float inv_tau, bool force,
                                                      float* __restrict__ amax) {
  const bool second = (int)blockIdx.x >= split;
  const CeSide s = second ? v : u;
  const int blk = second ? blockIdx.x - split : blockIdx.x, nb = second ? gridDim.x - split : split;
  float scale = 1.f;
  bool native = false;
  if constexpr (sizeof(T) == 4) {
    __shared__ CeMax sh[4];
    CeMax m[2] = {{0, 255}, {0, 255}};
    for (int i = threadIdx.x; i < na0; i += 256) m[0] = ce_max_join(m[0], CeMax{bmax[i], blow[i]});
    for (int i = threadIdx.x; i < na1; i += 256) m[1] = ce_max_join(m[1], CeMax{bmax[na0 + i], blow[na0 + i]});
    float inv[2], sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = ce_max_block(m[i], sh);
      sc[i] = f16_operand_scale(__uint_as_float(m[i].bits), &inv[i]);
    }
    const float unit = inv[0] * inv[1], c2 = unit * inv_tau * kCeLog2e;
    native = force || !ce_even(m[0]) || !ce_even(m[1]) || !(unit >= 0x1p-126f && unit < INFINITY && c2 >= 0x1p-125f && c2 < INFINITY);
    scale = sc[second];
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      amax[0] = native ? 0.f : __uint_as_float(m[0].bits);
      amax[1] = native ? 0.f : __uint_as_float(m[1].bits);
      amax[2] = native ? 1.f : 0.f;
    }
  }
  const int c0 = (threadIdx.x & 15) * 4;
  for (int64_t r = (int64_t)blk * 16 + (threadIdx.x >> 4); r < s.rows; r += (int64_t)nb * 16) {
    const T* x = (const T*)s.x + r * s.ld;
    const int there = s.off(r) ? 0 : cols;
    for (int c = c0; c < cp; c += 64) {
      ces4 hi, lo;
      cef4 whole;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const T v = c + e < there ? x[c + e] : (T)0;
        if constexpr (sizeof(T) == 4) {
          whole[e] = v;
          const float a = v * scale;
          const short h = ce_cvt<CRESTE_DT_F16>(a);       // (a scalar: bit casts of vector elements are miscompiled)
          hi[e] = h;
          lo[e] = ce_cvt<CRESTE_DT_F16>(a - (float)__builtin_bit_cast(_Float16, h));
        } else {
          hi[e] = (short)v;
        }
      }
      if constexpr (sizeof(T) == 4)
        if (native) {
          *reinterpret_cast<cef4*>((float*)s.out + r * cp + c) = whole;
          continue;
        }
      *reinterpret_cast<ces4*>(s.out + r * cp + c) = hi;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<ces4*>(s.out + s.piece + r * cp + c) = lo;
    }
  }
}

// per row: join the class tiles' (maximum, rest); 64 rows x 16 slices of the tiles per block and turn (blocks of rows).  Leaves nll, what
// the gradient kernels ask of a row (padded to whole tiles: rows that do not count get an infinite rest, hence G = 0, a label that
// names no class a NaN), and, from the last block to finish, the loss: sums of the blocks' sums in their order, so the result does not
// depend on which that was.  Maxima and label logits come in the units of the products
__global__ __launch_bounds__(1024) void ce_join_kernel(const float2* __restrict__ part, int tiles, int n, int blocks,
                                                       const float* __restrict__ zlab, const int64_t* __restrict__ labels, int64_t ignore,
                                                       int classes, const float* __restrict__ amax, float inv_tau,
                                                       float log2_scale, float* __restrict__ nll, float* __restrict__ rows,
                                                       uint64_t* __restrict__ bsum, unsigned* __restrict__ done, int mean,
                                                       float* __restrict__ loss, float* __restrict__ stat) {
  __shared__ float2 sh[16][64];
  __shared__ bool last;
  const int li = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const int64_t n64 = blocks * 64ll;
  const float unit = ce_operand_inv(amax, 0) * ce_operand_inv(amax, 1), c2 = unit * inv_tau * kCeLog2e;      // (as the loss kernels')
  for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t row = blk * 64ll + li;
    float2 st = make_float2(-3.0e38f, -1.f);
    if (row < n)
#pragma unroll 4
      for (int t = sl; t < tiles; t += 16) st = ce_merge(st, part[(int64_t)t * n + row], c2);
    if (blk != (int)blockIdx.x) __syncthreads();        // (everybody has left the turn before)
    sh[sl][li] = st;
    __syncthreads();
    if (sl != 0) continue;
    for (int s = 1; s < 16; ++s) st = ce_merge(st, sh[s][li], c2);
    float l = 0.f, c = 0.f;
    const int64_t y = row < n ? labels[row] : ignore;
    const bool on = row < n && y != ignore, ok = y >= 0 && y < classes;
    const float lr = log1pf(st.y);
    if (on) {
      l = ok ? (st.x - zlab[row]) * c2 * kCeLn2 + lr : __builtin_nanf("");
      c = 1.f;
    }
    if (row < n) nll[row] = l;
    rows[row] = !on ? 0.f : ok ? st.x * unit : __builtin_nanf("");
    reinterpret_cast<int*>(rows)[n64 + row] = on && ok ? (int)y : -1;
    rows[2 * n64 + row] = on ? lr * kCeLog2e - log2_scale : INFINITY;
    rows[3 * n64 + row] = on ? expm1f(-l) * exp2f(log2_scale) : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      l += __shfl_xor(l, o, 64);
      c += __shfl_xor(c, o, 64);
    }
    if (li == 0)                                        // one word, written through; counted when it has arrived
      __hip_atomic_store(bsum + blk, (uint64_t)__float_as_uint(c) << 32 | __float_as_uint(l), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (threadIdx.x == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = atomicAdd(done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __shared__ double sl_[1024], sc_[1024];
  double l = 0., c = 0.;
  for (int i = threadIdx.x; i < blocks; i += 1024) {
    const uint64_t v = __hip_atomic_load(bsum + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    l += __uint_as_float((unsigned)v);
    c += __uint_as_float((unsigned)(v >> 32));
  }
  sl_[threadIdx.x] = l;
  sc_[threadIdx.x] = c;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) {
      sl_[threadIdx.x] += sl_[threadIdx.x + o];
      sc_[threadIdx.x] += sc_[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    stat[0] = (float)sl_[0];
    stat[1] = (float)sc_[0];
    *loss = (float)(mean ? sl_[0] / fmax(sc_[0], 1.) : sl_[0]);
  }
}

// out[n][m] = scale * sum over splits of partial[split][n][ldp], for up to two outputs (blocks below `split` take the first)
__global__ __launch_bounds__(256) void ce_reduce_kernel(CeArgs u, int su, CeArgs v, int sv, int split) {
  const bool second = (int)blockIdx.x >= split;
  const CeArgs& p = second ? v : u;
  const int splits = second ? sv : su, blk = second ? blockIdx.x - split : blockIdx.x, nb = second ? gridDim.x - split : split;
  const float fs = ce_out_scale(p);
  const int64_t total = (int64_t)p.n * p.ldp;
  const int ldp = (int)p.ldp;
  int64_t i = (blk * 256LL + threadIdx.x) * 4, row = i / ldp;
  int d = (int)(i - row * ldp);
  const int64_t step = nb * 1024LL, srow = step / ldp;
  const int sd = (int)(step - srow * ldp);
  for (; i < total; i += step, row += srow, d += sd) {
    if (d >= ldp) { d -= ldp; ++row; }
    cef4 a = *reinterpret_cast<const cef4*>(p.partial + i);
#pragma unroll 8
    for (int s = 1; s < splits; ++s) a += *reinterpret_cast<const cef4*>(p.partial + s * p.psplit + i);
    a *= fs;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (d + e >= p.m_out) continue;
      const int64_t o = row * p.ldo + d + e;
      if (p.out_dt == CRESTE_DT_F32) ((float*)p.out)[o] = a[e];
      else if (p.out_dt == CRESTE_DT_BF16) ((short*)p.out)[o] = ce_cvt<CRESTE_DT_BF16>(a[e]);
      else ((short*)p.out)[o] = ce_cvt<CRESTE_DT_F16>(a[e]);
    }
  }
}

// --------------------------------------------------------------------------------------------------------- host side
namespace {

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Where everything sits in the caller's workspace.  The operands are used in place when a row is a multiple of 64 elements on
// 16-byte boundaries, else copied once (padded; fp32 into its two pieces unless x has few rows).  The gradients always have x from a copy, without what
// ignored rows hold (a training step of 8192 x 65536 x 256 bf16: 1215 -> 1219 us).
struct CePlan {
  int P, dt16, es, Dp, ldq, own;   // own: items a streaming workgroup holds
  bool packx, packw, stream;
  int64_t amax, xp, wp, part, zlab, bsum, done, g, dxp, dwp, total;
  int64_t packs;                   // bytes of the copied operands, at the front of the workspace
  int64_t vc, n64, ldg;            // classes per piece, rows of G, bytes between them
  int pieces, tiles, sl, sx, sw;   // class tiles of the loss, splits of LOSS / DX / DW
};

float ce_gscale_log2(const CePlan& q) { return q.dt16 == CRESTE_DT_F16 ? kCeF16Log2 : 0.f; }
int ce_own(const CePlan& q, int mode) { return 256 * ce_nt(mode, q.P, q.Dp); }

constexpr int kCeFewRows = 32;
constexpr int kCeJoinBlocks = 1 << 20;             // (a launch holds less than 2^32 threads: of 1024 a block)
constexpr int kCeMaxima = 512;                     // blocks that look for an operand's largest magnitude
// A piece of G takes 64 to 512 MiB: ce_pieces() weighs what the rounds of workgroups, the launches and dx's partial sums cost against
// the memory-side cache, which still holds 128 MiB when DX and DW read them.  Whole steps in us, always 128 MiB (16384 classes at least) /
// always 512 MiB / chosen: 4096 x 131072 x 1024 bf16 4805 / 4880 / 4790, 8192 x 50000 x 512 fp16 2476 / 2370 / 2366, 1000 x 100000 x 768
// bf16 930 / 877 / 874, 4096 x 65536 x 256 fp32 2195 / 2072 / 2070, 3000 x 30000 x 640 bf16 799 / 711 / 707
constexpr int64_t kCeCached = 128ll << 20;
constexpr int kCePieceMiB[] = {512, 384, 256, 192, 128, 64};

// Up to 256 feature columns (fp32's two pieces: 128) the streaming kernels hold the own side in registers; beyond, G in memory
bool ce_streams(int D, int dtype) { return D <= (dtype == CRESTE_DT_F32 ? 128 : 256); }
int ce_padded(int D, int dtype) { return ce_streams(D, dtype) ? (D <= 64 ? 64 : D <= 128 ? 128 : 256) : (int)up(D, 64); }

// 16-bit rows of whole padded widths are read in place, and fp32 ones where there are few rows of x (NATIVE then, ce_operands; a training
// step of 16 x 65536 x 512: 294 us, 353 with a copy of w)
bool ce_direct(const void* x, int64_t ld, int64_t N, int D, int dtype) {
  const int part = dtype == CRESTE_DT_F32 ? 4 : 8;
  return (dtype != CRESTE_DT_F32 || N <= kCeFewRows) && D == ce_padded(D, dtype) && ld % part == 0 && ld < (1 << 24) &&
         ((uintptr_t)x & 15) == 0;
}

// rows that the few-rows kernel can read in place: whole 32-byte steps on 16-byte boundaries
bool ce_few(const void* x, int64_t ld, int D, int dtype) {
  const int es = dtype == CRESTE_DT_F32 ? 4 : 2;
  return D * es % 32 == 0 && ld * es % 16 == 0 && ((uintptr_t)x & 15) == 0;
}

// splits of the contraction k, of those that fill one to eight rounds of workgroups: least rounds times the length of one (`start`: what its
// beginning and end cost, in units of k)
int ce_splits(int64_t tiles, int64_t k, int start, int64_t* least = nullptr) {
  int best = 1;
  int64_t cost = (tiles + 255) / 256 * (k + start);
  for (int r = 1; r <= 8; ++r) {
    int64_t s = 256 * r / tiles;
    const int64_t most = (k + 127) / 128;
    s = s > most ? most : s;
    if (s < 2) continue;
    const int64_t c = (tiles * s + 255) / 256 * (up((k + s - 1) / s, 64) + start);
    if (c < cost) { cost = c; best = (int)s; }
  }
  if (least) *least = cost;
  return best;
}

// classes per piece of G, and the splits of its DX and DW.  Costs in the time a workgroup takes for one step of the contraction (33 ns)
void ce_pieces(CePlan& q, int64_t N, int64_t V, int D) {
  const int64_t vall = up(V, kCeTile), col = q.n64 * 2 * q.P, mt = (D + kCeTile - 1) / kCeTile, nt = (N + kCeTile - 1) / kCeTile;
  const int work = q.P == 2 ? 3 : 1;                           // products a step
  double best = INFINITY;
  for (const int mib : kCePieceMiB) {
    int64_t vc = ((int64_t)mib << 20) / col / kCeTile * kCeTile;
    vc = vc < kCeTile ? kCeTile : vc > vall ? vall : vc;
    int64_t pieces = (vall + vc - 1) / vc;
    vc = up((vall + pieces - 1) / pieces, kCeTile);            // pieces of one size
    pieces = (vall + vc - 1) / vc;
    if (vc == q.vc) continue;
    int64_t cx, cw;
    const int sx = ce_splits(mt * nt, vc, 256, &cx), sw = ce_splits(mt * (vc / kCeTile), q.n64, 256, &cw);
    double cost = (double)((vc / kCeTile * nt + 255) / 256 * (q.Dp + 256) + cx + cw) * work + 450.;        // and three launches
    if (pieces > 1) cost += 8e-6 * sx * N * q.ldq * 6.;        // dx's partial sums, read and written: 6 steps a MB
    if (vc * col > kCeCached) cost += 1e-6 * vc * col * 9.;    // what the cache would have saved: 9 steps a MB of G
    if (cost * pieces >= best) continue;
    best = cost * pieces;
    q.vc = vc; q.pieces = (int)pieces; q.sx = sx; q.sw = sw;
  }
}

CePlan ce_plan(int64_t N, int64_t V, int D, int dtype, bool packx, bool packw, bool train) {
  CePlan q{};
  q.P = dtype == CRESTE_DT_F32 ? 2 : 1;
  q.dt16 = dtype == CRESTE_DT_BF16 ? CRESTE_DT_BF16 : CRESTE_DT_F16;
  q.es = dtype == CRESTE_DT_F32 ? 4 : 2;
  q.stream = ce_streams(D, dtype);
  q.Dp = ce_padded(D, dtype);
  q.ldq = (int)up(D, 4);
  q.packx = packx;
  q.packw = packw;
  int64_t o = 0;
  auto take = [&](int64_t bytes) { const int64_t at = o; o = up(o + bytes, 1024); return at; };
  q.amax = take(64 + 2 * kCeMaxima * 5);           // the two maxima and `native`; the blocks' maxima, and their lowest exponents
  q.xp = packx ? take(N * q.Dp * 2 * q.P) : 0;
  q.wp = packw ? take(V * q.Dp * 2 * q.P) : 0;
  q.packs = o + 32 * packw;                        // the size tells whether w is among them (all else is in whole 1024 bytes)
  q.tiles = (int)((V + kCeTile - 1) / kCeTile);
  if (!train) {
    q.own = ce_own(q, CE_LOSS);
    q.sl = q.stream ? ce_splits((N + q.own - 1) / q.own, V, 320) : 0;
    const bool tiles = !q.stream || N <= kCeFewRows;            // (few rows: which kernel depends on alignment too)
    q.part = take((int64_t)(tiles && q.tiles > q.sl ? q.tiles : q.sl) * N * 8);
    q.zlab = take(N * 4);
    q.bsum = take((N + 63) / 64 * 8);
    q.done = take(4);
    q.total = o;
    return q;
  }
  q.n64 = up(N, 64);
  if (q.stream) {
    q.own = ce_own(q, CE_DX);
    q.pieces = 1;
    q.vc = V;
    q.sx = ce_splits((N + q.own - 1) / q.own, V, 320);
    q.sw = ce_splits((V + q.own - 1) / q.own, N, 320);
  } else {
    ce_pieces(q, N, V, D);
    q.ldg = q.vc * 2 + 256;          // (rows a power of two apart would meet in the same memory channels)
    q.g = take(q.n64 * q.ldg * q.P);
  }
  if (q.sx > 1 || q.pieces > 1) q.dxp = take((int64_t)q.sx * N * q.ldq * 4);
  if (q.sw > 1) q.dwp = take((int64_t)q.sw * q.vc * q.ldq * 4);
  q.total = o;
  return q;
}

using CeBig = CeShape<256, 256, 2, 4, 64, 2>;          // 128 KB of LDS: one workgroup per CU

template <int MODE, int DT, int P, typename S>
int ce_launch(CeArgs a, int splits, hipStream_t s) {
  constexpr int bytes = S::NS * (S::BM + S::BN) * S::BK * 2;
  static std::atomic<uint64_t> mask{0};
  static_assert(S::BM == kCeTile, "");
  if (MODE != CE_GRAD) a.mt = cdiv(a.m, S::BM);          // (GRAD: given, the zeros behind the last class too)
  a.nt = cdiv(a.n, S::BN);
  const int64_t blocks = (int64_t)a.mt * a.nt * splits;
  CRESTE_REQUIRE(blocks * S::NW * 64 < (1ll << 32), "linear_ce: too many tiles for a launch");
  CRESTE_HIP(ensure_dyn_smem((const void*)ce_gemm_kernel<MODE, DT, P, S>, bytes, mask));
  ce_gemm_kernel<MODE, DT, P, S><<<(int)blocks, S::NW * 64, bytes, s>>>(a);
  CRESTE_CHECK_LAUNCH("linear_ce gemm");
  return CRESTE_OK;
}

template <int MODE>
int ce_gemm(const CePlan& q, const CeArgs& a, int splits, hipStream_t s) {
  if (q.P == 2) return ce_launch<MODE, CRESTE_DT_F16, 2, CeBig>(a, splits, s);
  if (q.dt16 == CRESTE_DT_BF16) return ce_launch<MODE, CRESTE_DT_BF16, 1, CeBig>(a, splits, s);
  return ce_launch<MODE, CRESTE_DT_F16, 1, CeBig>(a, splits, s);
}

// number of workgroups of one of the streaming kernels' halves; completes its arguments
int64_t ce_stream_blocks(CeArgs& a, int own, int splits) {
  a.nt = cdiv(a.n, own);
  a.k1 = a.m;
  a.ksplit = (int)up(cdiv(a.m, splits), kCeStage);
  return (int64_t)a.nt * splits;
}

// LOSS (loss given), or the gradients that are wanted (dx, dw: the others null)
template <int DT, int P, int DP>
int ce_stream_launch(const CePlan& q, CeArgs* loss, CeArgs* dx, CeArgs* dw, hipStream_t s) {
  constexpr int stages = 3 * CeStream<DP, kCeStage, P>::BYTES, out = 8 * 32 * 512, grad = stages > out ? stages : out;
  static std::atomic<uint64_t> mask_loss{0}, mask_grad{0};
  const int64_t nl = loss ? ce_stream_blocks(*loss, q.own, q.sl) : 0, nx = dx ? ce_stream_blocks(*dx, q.own, q.sx) : 0,
                nw = dw ? ce_stream_blocks(*dw, q.own, q.sw) : 0;
  CRESTE_REQUIRE((nl + nx + nw) * 512 < (1ll << 32), "linear_ce: too many tiles for a launch");
  if (loss) {
    CRESTE_HIP(ensure_dyn_smem((const void*)ce_loss_kernel<DT, P, DP>, stages, mask_loss));
    ce_loss_kernel<DT, P, DP><<<(int)nl, 512, stages, s>>>(*loss);
  } else {
    CRESTE_HIP(ensure_dyn_smem((const void*)ce_grad_kernel<DT, P, DP>, grad, mask_grad));
    ce_grad_kernel<DT, P, DP><<<(int)(nx + nw), 512, grad, s>>>(dx ? *dx : *dw, dw ? *dw : *dx, (int)nx);
  }
  CRESTE_CHECK_LAUNCH("linear_ce stream");
  return CRESTE_OK;
}

template <int DT, int P>
int ce_stream_typed(const CePlan& q, CeArgs* loss, CeArgs* dx, CeArgs* dw, hipStream_t s) {
  if (q.Dp == 64) return ce_stream_launch<DT, P, 64>(q, loss, dx, dw, s);
  if constexpr (P == 1)
    if (q.Dp == 256) return ce_stream_launch<DT, P, 256>(q, loss, dx, dw, s);
  return ce_stream_launch<DT, P, 128>(q, loss, dx, dw, s);
}

int ce_stream(const CePlan& q, CeArgs* loss, CeArgs* dx, CeArgs* dw, hipStream_t s) {
  if (q.P == 2) return ce_stream_typed<CRESTE_DT_F16, 2>(q, loss, dx, dw, s);
  if (q.dt16 == CRESTE_DT_BF16) return ce_stream_typed<CRESTE_DT_BF16, 1>(q, loss, dx, dw, s);
  return ce_stream_typed<CRESTE_DT_F16, 1>(q, loss, dx, dw, s);
}

int ce_grid(int64_t items) { return (int)(items < 1 ? 1 : items > 2048 ? 2048 : items); }

struct CeOperand { const char* p; int64_t ld, piece; };

// the operands as the kernels read them, from `work` (the maxima and the copies at the offsets of the plan); copied there unless `ready`.
// labels, ignore, counts: see CeSide
int ce_operands(const CePlan& q, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int64_t V, int D, float inv_tau,
                bool ready, const int64_t* labels, int64_t ignore, const float* counts, char* work, CeOperand* X, CeOperand* W, hipStream_t s) {
  float* amax = (float*)(work + q.amax);
  unsigned* bmax = (unsigned*)amax + 16;
  uint8_t* blow = (uint8_t*)(bmax + 2 * kCeMaxima);
  *X = {(const char*)x, ldx * 2, 0};
  *W = {(const char*)w, ldw * 2, 0};
  if (q.packx) *X = {work + q.xp, (int64_t)q.Dp * 2, N * q.Dp * 2};
  if (q.packw) *W = {work + q.wp, (int64_t)q.Dp * 2, V * q.Dp * 2};
  if (ready) return CRESTE_OK;
  const CeSide sx{x, N, ldx, (short*)(work + q.xp), N * q.Dp, labels, ignore, counts},
      sw{w, V, ldw, (short*)(work + q.wp), V * q.Dp, nullptr, 0, nullptr};
  auto blocks = [](int64_t rows, int most) { const int64_t b = (rows + 15) / 16; return (int)(b > most ? most : b); };
  const int px = q.packx ? blocks(N, 2048) : 0, pw = q.packw ? blocks(V, 2048) : 0;
  if (q.P == 2) {                                  // (x at least is copied where not the few-rows kernel takes both)
    const bool force = N <= kCeFewRows;            // (as the few-rows kernel multiplies: no magnitudes asked for)
    const int ax = force ? 0 : blocks(N, kCeMaxima), aw = force ? 0 : blocks(V, kCeMaxima);
    if (!force) ce_amax_kernel<<<ax + aw, 256, 0, s>>>(sx, sw, D, ax, bmax, blow);
    ce_pack_kernel<float><<<px + pw, 256, 0, s>>>(sx, sw, D, q.Dp, px, bmax, blow, ax, aw, inv_tau, force, amax);
  } else if (px + pw) {
    ce_pack_kernel<short><<<px + pw, 256, 0, s>>>(sx, sw, D, q.Dp, px, nullptr, nullptr, 0, 0, 0.f, false, nullptr);
  }
  CRESTE_CHECK_LAUNCH("linear_ce pack");
  return CRESTE_OK;
}

int ce_check(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* labels_or_rows, int64_t N, int64_t V, int D, int dtype,
             float tau) {
  CRESTE_REQUIRE(x && w && labels_or_rows, "linear_ce: null pointer");
  CRESTE_REQUIRE(dtype >= CRESTE_DT_F32 && dtype <= CRESTE_DT_F16, "linear_ce: dtype %d", dtype);
  CRESTE_REQUIRE(N > 0 && V > 0 && D > 0 && N < (1ll << 30) && V < (1ll << 30) && D <= 65536, "linear_ce: N %lld V %lld D %d",
                 (long long)N, (long long)V, D);
  CRESTE_REQUIRE((ldx >= D || (ldx == 0 || N == 1)) && ldx >= 0 && (ldw >= D || V == 1 || ldw == 0) && ldw >= 0,
                 "linear_ce: row strides %lld %lld", (long long)ldx, (long long)ldw);
  CRESTE_REQUIRE(tau > 0.f && tau < INFINITY && 1.f / tau * kCeLog2e < INFINITY,
                 "linear_ce: temperature must be positive and finite, its inverse (in units of log 2) too");
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

// whether the forward takes the few-rows kernel, which copies nothing
static bool ce_takes_few(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int D, int dtype) {
  return N <= kCeFewRows && ce_few(x, ldx, D, dtype) && ce_few(w, ldw, D, dtype);
}

extern "C" int64_t creste_linear_ce_packs_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t N, int64_t V, int D,
                                                int dtype) {
  if (creste_linear_ce_workspace_bytes(N, V, D, dtype, 0) < 0) return -1;
  if (ce_takes_few(x, ldx, w, ldw, N, D, dtype)) return 0;
  return ce_plan(N, V, D, dtype, true, !ce_direct(w, ldw, N, D, dtype), false).packs;
}

extern "C" int creste_linear_ce_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* labels, int64_t N,
                                        int64_t V, int D, int dtype, int64_t ignore_index, float temperature, int mean,
                                        float* loss, float* nll, float* rows, float* stat, void* packs, void* work,
                                        int64_t work_bytes, void* stream) {
  const int bad = ce_check(x, ldx, w, ldw, labels, N, V, D, dtype, temperature);
  if (bad) return bad;
  const bool few = ce_takes_few(x, ldx, w, ldw, N, D, dtype);
  // (a row of x only reaches its own softmax, so x need not be copied for what ignored rows hold -- unless the backward is to have it)
  const CePlan q = ce_plan(N, V, D, dtype, !few && (packs || !ce_direct(x, ldx, N, D, dtype)), !few && !ce_direct(w, ldw, N, D, dtype),
                           false);
  CRESTE_REQUIRE(loss && nll && rows && stat && work && work_bytes >= q.total, "linear_ce_forward: outputs / workspace (%lld of %lld bytes)",
                 (long long)work_bytes, (long long)q.total);
  CRESTE_REQUIRE(q.stream || few || (int64_t)q.tiles * ((N + 255) / 256) * 512 < (1ll << 32),
                 "linear_ce_forward: too many tiles for a launch (2^23 of 256 x 256) at N %lld V %lld", (long long)N, (long long)V);
  CRESTE_REQUIRE((((uintptr_t)work | (uintptr_t)packs) & 15) == 0, "linear_ce_forward: work and packs on 16-byte boundaries");
  hipStream_t s = (hipStream_t)stream;
  char* wk = (char*)work;
  CeOperand X{(const char*)x, ldx * q.es, 0}, W{(const char*)w, ldw * q.es, 0};
  char* const copies = packs ? (char*)packs : wk;
  if (!few) {
    const int rc = ce_operands(q, x, ldx, w, ldw, N, V, D, 1.f / temperature, false, labels, ignore_index, nullptr, copies, &X, &W, s);
    if (rc) return rc;
  }
  CeArgs a{};
  a.a = W.p; a.lda = W.ld; a.pa = W.piece; a.ra = V;
  a.b = X.p; a.ldb = X.ld; a.pb = X.piece; a.rb = N;
  a.m = (int)V; a.n = (int)N;
  a.k1 = q.Dp;
  a.labels = labels; a.classes = (int)V;
  a.inv_tau = 1.f / temperature;
  a.amax = q.P == 2 ? (const float*)(copies + q.amax) : nullptr;
  a.part = (float2*)(wk + q.part); a.zlab = (float*)(wk + q.zlab); a.done = (unsigned*)(wk + q.done);
  if (few) {
    if (dtype == CRESTE_DT_F32) ce_few_kernel<CRESTE_DT_F32><<<q.tiles, 256, 0, s>>>(a, D);
    else if (dtype == CRESTE_DT_BF16) ce_few_kernel<CRESTE_DT_BF16><<<q.tiles, 256, 0, s>>>(a, D);
    else ce_few_kernel<CRESTE_DT_F16><<<q.tiles, 256, 0, s>>>(a, D);
    CRESTE_CHECK_LAUNCH("linear_ce few rows");
  } else {
    const int rg = q.stream ? ce_stream(q, &a, nullptr, nullptr, s) : ce_gemm<CE_LOSS>(q, a, 1, s);
    if (rg) return rg;
  }
  const int nb = (int)((N + 63) / 64);
  ce_join_kernel<<<nb < kCeJoinBlocks ? nb : kCeJoinBlocks, 1024, 0, s>>>(
      a.part, q.stream && !few ? q.sl : q.tiles, (int)N, nb, a.zlab, labels, ignore_index, (int)V, few ? nullptr : a.amax, a.inv_tau,
      ce_gscale_log2(q), nll, rows, (uint64_t*)(wk + q.bsum), a.done, mean, loss, stat);
  CRESTE_CHECK_LAUNCH("linear_ce join");
  return CRESTE_OK;
}

extern "C" int creste_linear_ce_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* rows, int64_t N, int64_t V,
                                         int D, int dtype, float temperature, int mean, const float* stat, const float* g_loss,
                                         const void* packs, void* gx, void* gw, void* work, int64_t work_bytes, void* stream) {
  const int bad = ce_check(x, ldx, w, ldw, rows, N, V, D, dtype, temperature);
  if (bad) return bad;
  const CePlan q = ce_plan(N, V, D, dtype, true, !ce_direct(w, ldw, N, D, dtype), true);
  CRESTE_REQUIRE(stat && g_loss && (gx || gw) && work && work_bytes >= q.total, "linear_ce_backward: inputs / workspace (%lld of %lld bytes)",
                 (long long)work_bytes, (long long)q.total);
  CRESTE_REQUIRE((((uintptr_t)gx | (uintptr_t)gw | (uintptr_t)work | (uintptr_t)packs) & 15) == 0,
                 "linear_ce_backward: gx, gw, packs and work on 16-byte boundaries");
  hipStream_t s = (hipStream_t)stream;
  char* wk = (char*)work;
  CeOperand X, W;
  const bool kept = packs && !ce_takes_few(x, ldx, w, ldw, N, D, dtype);
  char* const copies = kept ? (char*)packs : wk;
  const int rc = ce_operands(q, x, ldx, w, ldw, N, V, D, 1.f / temperature, kept, nullptr, 0, rows + 2 * q.n64, copies, &X, &W, s);
  if (rc) return rc;
  CeArgs c{};                                       // what every product shares
  c.classes = (int)V;
  c.inv_tau = 1.f / temperature;
  c.amax = q.P == 2 ? (const float*)(copies + q.amax) : nullptr;
  c.stat = stat; c.gl = g_loss; c.mean = mean;
  c.gscale = exp2f(ce_gscale_log2(q));
  c.row_max = rows; c.row_lab = (const int*)(rows + q.n64); c.row_rest = rows + 2 * q.n64; c.row_g = rows + 3 * q.n64;
  c.n64 = (int)q.n64;
  c.out_dt = dtype;
  c.ldo = c.m_out = D;
  c.ldp = q.ldq;
  auto reduce = [&](const CeArgs* u, int su, const CeArgs* v, int sv) {      // one or two sums of partials in one launch
    auto blocks = [&](const CeArgs& a) { return ce_grid((int64_t)a.n * q.ldq / 1024 + 1); };
    const int bu = u ? blocks(*u) : 0, bv = v ? blocks(*v) : 0;
    ce_reduce_kernel<<<bu + bv, 256, 0, s>>>(u ? *u : *v, su, v ? *v : *u, sv, bu);
    CRESTE_CHECK_LAUNCH("linear_ce reduce");
    return CRESTE_OK;
  };
  CeArgs dx = c, dw = c;
  dx.n = (int)N; dx.out = gx; dx.which = 1; dx.psplit = N * q.ldq;
  if (q.dxp) dx.partial = (float*)(wk + q.dxp);
  dw.which = 0; dw.psplit = q.vc * q.ldq;
  if (q.dwp) dw.partial = (float*)(wk + q.dwp);
  if (q.stream) {
    dx.a = W.p; dx.lda = W.ld; dx.pa = W.piece; dx.ra = V; dx.m = (int)V;
    dx.b = X.p; dx.ldb = X.ld; dx.pb = X.piece;
    dw.a = X.p; dw.lda = X.ld; dw.pa = X.piece; dw.ra = N; dw.m = (int)N;
    dw.b = W.p; dw.ldb = W.ld; dw.pb = W.piece; dw.n = (int)V;
    dw.out = gw;
    const int rg = ce_stream(q, nullptr, gx ? &dx : nullptr, gw ? &dw : nullptr, s);
    if (rg) return rg;
  } else {
    for (int piece = 0; piece < q.pieces; ++piece) {
      const int64_t v0 = piece * q.vc, nv = V - v0 < q.vc ? V - v0 : q.vc;
      CeArgs a = c;                                 // G of the piece
      a.g = wk + q.g; a.ldg = q.ldg; a.pg = q.n64 * q.ldg; a.mt = (int)(q.vc / kCeTile);
      a.a = W.p + v0 * W.ld; a.lda = W.ld; a.pa = W.piece; a.ra = nv;
      a.b = X.p; a.ldb = X.ld; a.pb = X.piece; a.rb = N;
      a.m = (int)nv; a.n = (int)N; a.class0 = (int)v0;
      a.k1 = q.Dp;
      int rg = ce_gemm<CE_GRAD>(q, a, 1, s);
      if (rg) return rg;
      if (gx) {
        dx.a = a.a; dx.lda = W.ld; dx.pa = W.piece; dx.ra = nv; dx.ca = q.Dp * 2;
        dx.b = a.g; dx.ldb = a.ldg; dx.pb = a.pg; dx.rb = q.n64;
        dx.m = D; dx.class0 = (int)v0;
        dx.k1 = (int)up(nv, 64);
        dx.ksplit = q.sx > 1 ? (int)up(cdiv(q.vc, q.sx), 64) : 0;
        dx.accumulate = piece > 0;
        rg = ce_gemm<CE_DX>(q, dx, q.sx, s);
        if (rg) return rg;
      }
      if (gw) {
        dw.a = X.p; dw.lda = X.ld; dw.pa = X.piece; dw.ra = N; dw.ca = q.Dp * 2;
        dw.b = a.g; dw.ldb = a.ldg; dw.pb = a.pg; dw.rb = q.n64; dw.cb = (int)(q.vc * 2);
        dw.m = D; dw.n = (int)nv;
        dw.k1 = (int)q.n64;
        dw.ksplit = q.sw > 1 ? (int)up(cdiv(q.n64, q.sw), 64) : 0;
        dw.out = (char*)gw + v0 * D * q.es;
        rg = ce_gemm<CE_DW>(q, dw, q.sw, s);
        if (rg) return rg;
        if (dw.partial && q.pieces > 1 && reduce(nullptr, 0, &dw, q.sw)) return CRESTE_ERR_HIP;
      }
    }
  }
  const bool rx = gx && dx.partial, rw = gw && dw.partial && q.pieces == 1;
  return rx || rw ? reduce(rx ? &dx : nullptr, q.sx, rw ? &dw : nullptr, q.sw) : CRESTE_OK;
}
