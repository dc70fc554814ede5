// The experts' products (moe_topk.hip) on operands of two fp16 pieces (split2.h),
// for layers whose experts hold enough slots that the products outweigh the
// passes that lay their operands out.
//
// Every product is C = A B^T with both operands as [piece][K / 8][R][8]:
//   hidden   u^T [H, pos] = W1[e]^T x^T      A rows (e, h), k = d;  B rows pos
//   slots    o^T [D, pos] = W2[e]^T h^T      A rows (e, d), k = h;  B rows pos
//   back     dh^T [H, pos] = W2[e] dy^T      A rows (e, h), k = d;  B rows pos
//   slots    dx^T [D, pos] = W1[e] du^T      A rows (e, d), k = h;  B rows pos
//   weights  dW1[e] = x^T du, dW2[e] = (w h)^T dy     k = the expert's positions
// Positions are the slots sorted by expert, every segment padded to 32 with
// zeros (perm -1), so that a segment is whole chunks as a contraction too.  The
// positions are a product's columns: a lane then holds four consecutive h (or d)
// of one position, half a chunk of the next product's operand, and stores its
// floats as float4s.
//
// Scales.  Rows of x, dy and the weights are scaled by the power of two that
// brings their largest finite entry to [2^14, 2^15), so that 22 bits are kept of
// every entry down to 2^-17 of its row's largest, an absolute 2^-40 of that
// below; an infinity or NaN stays in its row's products.  act(u) and du are
// written as pieces by the epilogue that makes them, before their largest entry
// is known: their scale is the Cauchy-Schwarz bound |x| max |W1 column| (2-norms,
// rounded up to powers of two), some 2^4 above the largest entry.  Where
// positions are the contraction, one scale serves an expert's segment, with the
// features and hidden units far below its largest: there the low pieces are held
// times 2^11 (split2.h), 22 bits down to 2^-28 and an absolute 2^-51 below.  Relative
// errors of the rows and columns of the weights' gradients of units at 1e-4, 1e-6
// and 1e-8 of the others, by themselves, 500 tokens of 136 x 160: 2.7e-7, 2.7e-7,
// 1.0e-5 (three pieces 3e-7); with low pieces beside the high ones 2.0e-6, 1.8e-4,
// 1.9e-2, in 1.6% less of a training step.
//
// Passes beside the products: the weights' layouts (read twice, written once),
// x and dy gathered by position, and for the gradient both once more with
// positions as k.  They are bound by HBM.
#include <algorithm>
#include <atomic>

#include "common.h"
#include "kernels.h"
#include "moe_act.h"
#include "split2.h"

namespace nship {
namespace {

// 256 rows x 128 columns, two workgroups on a CU: one's epilogue runs beside the
// other's products.  131072 slots of 64 experts of 1024 x 1024, us, hidden and slots
// products: 1172, 949 (235 and 290 TFLOP/s); 256 x 256, one workgroup of eight waves
// on a CU: 1308, 1050.
// The weights' gradients have accumulators for the products with a low piece beside
// the others, and eight waves of half the blocks: 16384 tokens, 2 of 64 experts of
// 1024 x 1024, 273 us a product (290 with the two sums in turn on the waves above,
// 253 with one sum).
constexpr int kWN = 2, kTN = 2;
using Tile = Split2Tile<2, kWN, 4, kTN, 16>;
using FarTile = Split2Tile<4, kWN, 2, kTN, 16, true>;  // the weights' gradients
constexpr int kPad = 32;      // positions a segment is padded to
constexpr int kNoExp = -300;  // "the logarithm of 0"
constexpr int kPitch = 40;    // halves of a transposing tile's row
constexpr int kTurnBytes = 2 * 32 * kPitch * 2;

// v = h + l (FAR: h + 2^-11 l, split2.h), with l = 0 beside an infinite h (not inf - inf).
template <bool FAR = false>
__device__ __forceinline__ void split2_any(float v, _Float16& h, _Float16& l) {
  h = (_Float16)v;
  const float r = (v - (float)h) * (FAR ? kLowUp : 1.f);
  l = (_Float16)(fabsf(v) > 65504.f ? 0.f : r);
}
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}
// Smallest n with a <= 2^n, for a > 0.
__device__ __forceinline__ int log2_up(double a) {
  int n;
  const double m = frexp(a, &n);  // a = m 2^n, m in [1/2, 1)
  return m == 0.5 ? n - 1 : n;
}
// The exponent that scales a row of largest entry `top` into [2^14, 2^15].
__device__ __forceinline__ int row_exp(float top) { return top > 0.f ? 14 - ilogbf(top) : 0; }
// The exponent of a segment's operand from the largest -exponent of its rows.
__device__ __forceinline__ int seg_exp(int top) { return top > kNoExp ? -top : 0; }
__device__ __forceinline__ int log2_norm(double sq) { return sq > 0. ? log2_up(sqrt(sq)) : kNoExp; }

template <bool FAR = false>
__device__ __forceinline__ void put_chunk(_Float16* __restrict__ to, int64_t piece, const float (&v)[8]) {
  half8 h, l;
#pragma unroll
  for (int u = 0; u < 8; u++) {
    _Float16 hh, ll;
    split2_any<FAR>(v[u], hh, ll);
    h[u] = hh;
    l[u] = ll;
  }
  *reinterpret_cast<half8*>(to) = h;
  *reinterpret_cast<half8*>(to + piece) = l;
}

// ---- layouts -----------------------------------------------------------------------

// Rows of `src` (row r: src + (tok ? tok[r] : r) * K) as operand rows r of [2][Kp /
// 8][rows][8], with their exponents and the logarithms of their 2-norms.  32 rows
// a workgroup.  blk: the expert of every 32 rows; then for each expert the largest
// -exponent (top), and of norm + log2 |weight| (wnorm) if asked for.
struct RowsArgs {
  const float* src;
  const int* tok;
  const int* perm;
  const int* blk;
  const int* nrows;   // rows in use (device), or null: all
  const float* weight;
  _Float16* out;
  int* exps;
  int* norm;
  int* top;
  int* wnorm;
  int64_t rows, K, Kp;
  int per_expert;     // rows an expert (weights): norm[r / per_expert] is the largest norm instead
};
// Lane (row, part) of a wave's 8 rows takes the octets part, part + 8, .. of its
// row: 256-byte runs of eight rows are read, 128-byte runs of chunks written.
// REGS: a row's share stays in registers (K up to 1024), else it is read twice.
constexpr int kRowOctets = 16;  // octets a lane
template <bool VEC, bool REGS>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, part = lane >> 3;
  const int64_t r0 = (int64_t)blockIdx.x * 32;
  if (a.nrows && r0 >= *a.nrows) return;
  const int64_t r = r0 + w * 8 + (lane & 7);
  const bool in = r < a.rows;
  const int64_t from = !in ? -1 : a.tok ? (int64_t)a.tok[r] : r;
  const float* __restrict__ p = a.src + (from >= 0 ? from : 0) * a.K;
  const int oct = (int)(a.Kp / 8);
  auto load = [&](int o, float (&v)[8]) {
    if (VEC) {
#pragma unroll
      for (int u = 0; u < 8; u += 4) {
        const bool ok = from >= 0 && o * 8 + u < a.K;
        const float4 f = *reinterpret_cast<const float4*>(p + (ok ? o * 8 + u : 0));
        v[u] = ok ? f.x : 0.f; v[u + 1] = ok ? f.y : 0.f; v[u + 2] = ok ? f.z : 0.f; v[u + 3] = ok ? f.w : 0.f;
      }
    } else {
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const bool ok = from >= 0 && o * 8 + u < a.K;
        const float f = p[ok ? o * 8 + u : 0];
        v[u] = ok ? f : 0.f;
      }
    }
  };
  float top = 0.f;
  double sq = 0.;
  auto look = [&](const float (&v)[8]) {
    float s[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      s[u] = finite_abs(v[u]);
      top = fmaxf(top, s[u]);
      sq += (double)s[u] * s[u];
    }
  };
  float keep[REGS ? kRowOctets : 1][8];
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kRowOctets; i++)
      if (8 * i < oct) load(part + 8 * i, keep[i]);  // (uniform; past the row's end: zeros)
#pragma unroll
    for (int i = 0; i < kRowOctets; i++)
      if (8 * i < oct) look(keep[i]);
  } else {
    for (int o = part; o < oct; o += 8) {
      load(o, keep[0]);
      look(keep[0]);
    }
  }
#pragma unroll
  for (int o = 8; o < 64; o <<= 1) {
    top = fmaxf(top, __shfl_xor(top, o, kWave));
    sq += __shfl_xor(sq, o, kWave);
  }
  const int ex = row_exp(top), n = log2_norm(sq);
  if (part == 0 && in) {
    a.exps[r] = ex;
    if (!a.per_expert) a.norm[r] = n;
  }
  if (a.per_expert) {  // (one atomic a wave where its rows are one expert's: those of an expert queue up)
    const int64_t first = min(r0 + w * 8, a.rows - 1) / a.per_expert, end = min(r0 + w * 8 + 7, a.rows - 1) / a.per_expert;
    int big = in ? n : kNoExp;
    if (first == end) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) big = max(big, __shfl_xor(big, o, kWave));
      if (lane == 0) atomicMax(&a.norm[first], big);
    } else if (part == 0 && in) {
      atomicMax(&a.norm[r / a.per_expert], n);
    }
  }
  if (a.blk) {
    int big_e = from >= 0 && top > 0.f ? -ex : kNoExp, big_n = kNoExp;  // over the wave's 8 rows
    if (a.weight && from >= 0) {
      const float wt = finite_abs(a.weight[a.perm[r]]);
      big_n = wt > 0.f && n > kNoExp ? n + log2_up(wt) : kNoExp;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      big_e = max(big_e, __shfl_xor(big_e, o, kWave));
      big_n = max(big_n, __shfl_xor(big_n, o, kWave));
    }
    if (lane == 0) {
      const int e = a.blk[blockIdx.x];
      if (a.top && big_e > kNoExp) atomicMax(&a.top[e], big_e);
      if (a.wnorm && big_n > kNoExp) atomicMax(&a.wnorm[e], big_n);
    }
  }
  if (!in) return;
  const int64_t piece = a.Kp * a.rows;
  auto store = [&](int o, float (&v)[8]) {
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = ldexpf(v[u], ex);
    put_chunk(a.out + (o * a.rows + r) * 8, piece, v);
  };
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kRowOctets; i++)
      if (part + 8 * i < oct) store(part + 8 * i, keep[i]);
  } else {
    for (int o = part; o < oct; o += 8) {
      load(o, keep[0]);
      store(o, keep[0]);
    }
  }
}

// Columns of W[e] [K, C] as operand rows e C + c of [2][Kp / 8][E C][8], their
// exponents, and each expert's largest column norm.  64 columns a workgroup of 16
// waves, each the octets w, w + 16, .. of them.  REGS: as above.
constexpr int kColOctets = 8;
template <bool REGS>
__global__ __launch_bounds__(1024) void cols_kernel(const float* __restrict__ W, _Float16* __restrict__ out,
                                                    int* __restrict__ exps, int* __restrict__ norm, int64_t K,
                                                    int64_t Kp, int64_t C, int64_t rows) {
  __shared__ float st[16][64];
  __shared__ double sn[16][64];
  const int t = threadIdx.x, c = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t col = (int64_t)blockIdx.x * 64 + c, e = blockIdx.y;
  const bool in = col < C;
  const float* __restrict__ p = W + e * K * C + (in ? col : 0);
  const int oct = (int)(Kp / 8);
  float top = 0.f;
  double sq = 0.;
  auto load = [&](int o, float (&v)[8]) {
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = p[(o * 8 + u < K ? o * 8 + u : 0) * C];  // (uniform)
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = o * 8 + u < K ? v[u] : 0.f;
  };
  auto look = [&](const float (&v)[8]) {
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const float s = finite_abs(v[u]);
      top = fmaxf(top, s);
      sq += (double)s * s;
    }
  };
  float keep[REGS ? kColOctets : 1][8];
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kColOctets; i++)
      if (w + 16 * i < oct) load(w + 16 * i, keep[i]);
#pragma unroll
    for (int i = 0; i < kColOctets; i++)
      if (w + 16 * i < oct) look(keep[i]);
  } else {
    for (int o = w; o < oct; o += 16) {
      load(o, keep[0]);
      look(keep[0]);
    }
  }
  st[w][c] = top;
  sn[w][c] = sq;
  __syncthreads();
  sq = 0.;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    top = fmaxf(top, st[i][c]);
    sq += sn[i][c];
  }
  const int ex = row_exp(top);
  if (w == 0) {
    int n = in ? log2_norm(sq) : kNoExp;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n = max(n, __shfl_xor(n, o, kWave));
    if (c == 0) atomicMax(&norm[e], n);
    if (in) exps[e * C + col] = ex;
  }
  if (!in) return;
  const int64_t piece = Kp * rows;
  auto store = [&](int o, float (&v)[8]) {
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = ldexpf(v[u], ex);
    put_chunk(out + (o * rows + e * C + col) * 8, piece, v);
  };
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kColOctets; i++)
      if (w + 16 * i < oct) store(w + 16 * i, keep[i]);
  } else {
    for (int o = w; o < oct; o += 16) {
      load(o, keep[0]);
      store(o, keep[0]);
    }
  }
}

// src by position as the operand [2][np / 8][C][8] (rows: its columns, k: the
// positions), scaled by -top of the position's expert.  Workgroup: 64 columns, 32
// positions.
__global__ __launch_bounds__(256) void turn_kernel(const float* __restrict__ src, const int* __restrict__ tok,
                                                   const int* __restrict__ blk, const int* __restrict__ nrows,
                                                   const int* __restrict__ top, _Float16* __restrict__ out, int64_t C,
                                                   int64_t np) {
  const int ctiles = (int)((C + 63) / 64), b = blockIdx.x / ctiles;
  const int64_t p0 = (int64_t)b * kPad;
  if (p0 >= *nrows) return;
  const int c = threadIdx.x & 63, o = threadIdx.x >> 6;
  const int64_t col = (int64_t)(blockIdx.x % ctiles) * 64 + c;
  if (col >= C) return;
  const int ex = seg_exp(top[blk[b]]);
  float v[8];
#pragma unroll
  for (int u = 0; u < 8; u++) {
    const int t = tok[p0 + 8 * o + u];
    const float f = src[(int64_t)(t < 0 ? 0 : t) * C + col];
    v[u] = t < 0 ? 0.f : ldexpf(f, ex);
  }
  put_chunk<true>(out + ((p0 / 8 + o) * C + col) * 8, np * C, v);
}

// xw[e] = the largest log2 of |weight| times the bound of |act(u)|'s factor by
// position: |x|, or 1 where act is bounded by 1.
__global__ __launch_bounds__(256) void weight_norm_kernel(const int* __restrict__ xnorm, const int* __restrict__ perm,
                                                          const int* __restrict__ blk, const int* __restrict__ nrows,
                                                          const float* __restrict__ weight, bool one,
                                                          int* __restrict__ xw) {
  const int64_t pos = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int n = kNoExp;
  if (pos < *nrows) {
    const int slot = perm[pos];
    const float w = slot >= 0 ? finite_abs(weight[slot]) : 0.f;
    const int b = one ? 0 : xnorm[pos];
    n = w > 0.f && b > kNoExp ? b + log2_up(w) : kNoExp;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n = max(n, __shfl_xor(n, o, kWave));  // (32 positions: one expert)
  if ((threadIdx.x & 31) == 0 && n > kNoExp) atomicMax(&xw[blk[pos / kPad]], n);
}

__global__ void preset_kernel(int* __restrict__ p, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = kNoExp;
}

// ---- products ------------------------------------------------------------------------

struct Stats {     // of the positions and experts (int arrays)
  int *xexp, *xnorm, *dexp, *dnorm;  // [np]
  int *xtop, *xw, *dtop, *dw;        // [E] largest -exponent, norm + log2 |weight|
  int *w1norm, *w2norm;              // [E] largest column norm of W1[e], row norm of W2[e]
  int *w1c, *w2c, *w1r, *w2r;        // exponents of the weights' operands' rows
};

enum Mode : int { kHidden = 0, kSlots, kBack, kWeight };

struct SplitArgs {
  const _Float16* A;    // weights (kWeight: a transposed operand)
  const _Float16* B;
  int64_t arows, brows, kp;  // rows of the operands, contraction (kWeight: np)
  int64_t M;            // rows of C (of an expert)
  const int *seg, *perm, *tiles, *ntiles, *items, *nitems;
  int mt, nt;           // tiles of M, kWeight: of the columns too
  const int* aexp;      // exponents of A's rows
  const int* bexp;      // of B's rows (kSlots from kHidden's or kBack's: null, by the bound)
  Stats st;
  int act, sigmoid;     // sigmoid: act(u) is bounded by 1, not by |u|
  int back;             // kSlots: B is du, not act(u)
  const float* weight;  // [slot]
  float* f;             // kHidden: u [np, M] or null; kSlots: [slot, M]; kWeight: [E][M, N]
  const float* pre;     // kBack: u
  _Float16* out;        // kHidden: act(u), kBack: du, as rows of positions
  _Float16* turn1;      // kBack: du with positions as k
  _Float16* turn2;      // kBack: weight act(u) alike
  float* dot;           // kBack: [2 mt][np] partial sums of act(u) . dh
  float* kpart;         // kWeight: partial sums of items with a slot
  int64_t np, N;
  bool vec;
};

// The exponents of act(u), du (rows) and of their segments' (positions as k).
__device__ __forceinline__ int hidden_exp(const SplitArgs& g, int64_t pos, int e) {
  const int b = g.sigmoid ? 0 : g.st.xnorm[pos] + g.st.w1norm[e];
  return b > kNoExp ? 15 - b : 0;
}
__device__ __forceinline__ int grad_exp(const SplitArgs& g, int64_t pos, int e, float w) {
  const float a = finite_abs(w);
  const int b = g.st.dnorm[pos] + g.st.w2norm[e] + 1;  // (every activation's slope is below 2)
  return a > 0.f && b > kNoExp ? 15 - b - log2_up(a) : 0;
}
__device__ __forceinline__ int grad_seg_exp(const SplitArgs& g, int e) {
  const int b = g.st.dw[e] + g.st.w2norm[e] + 1;
  return b > kNoExp ? 15 - b : 0;
}
__device__ __forceinline__ int hidden_seg_exp(const SplitArgs& g, int e) {
  // (sigmoid: act is below 1 and so below every weight's own size)
  const int b = g.st.xw[e] + (g.sigmoid ? 0 : g.st.w1norm[e]);
  return b > kNoExp ? 15 - b : 0;
}

constexpr int waves_of(int mode) { return mode == kWeight ? FarTile::NT / 64 : Tile::NT / 64; }

template <int MODE>
__global__ __launch_bounds__(waves_of(MODE) * 64, 2) void split_kernel(SplitArgs g) {
  constexpr int kWaves = waves_of(MODE), kTM = 16 / kWaves;
  static_assert(kTurnBytes * kWaves + 4 * Tile::RA <= Tile::kLds, "the transposing tiles and the exponents fit");
  __shared__ __attribute__((aligned(16))) char smem[Tile::kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / kWN, wn = wave % kWN;
  const int l32 = lane & 31, kh = lane >> 5;
  int e, mt;
  int64_t n0, nend;       // columns: positions, or kWeight the second matrix's
  int64_t arow, kbeg = 0;
  int nk;
  float* f = g.f;
  if (MODE == kWeight) {
    const int per = g.mt * g.nt, T = *g.nitems * per;
    if ((int)blockIdx.x >= T) return;
    const int L = split2_xcd_linear(blockIdx.x, T);
    const int* it = g.items + 4 * (L / per);
    e = it[0];
    kbeg = it[1];
    nk = (it[2] - it[1]) / 16;  // (whole chunks; 0: an expert without slots)
    mt = L % per / g.nt;
    n0 = (int64_t)(L % g.nt) * Tile::RB;
    nend = g.N;
    arow = 0;
    f = it[3] < 0 ? f + (int64_t)e * g.M * g.N : g.kpart + (int64_t)it[3] * g.M * g.N;
  } else {
    const int T = *g.ntiles * g.mt;
    if ((int)blockIdx.x >= T) return;
    const int L = split2_xcd_linear(blockIdx.x, T);
    e = g.tiles[2 * (L / g.mt)];
    mt = L % g.mt;
    n0 = g.seg[e] + (int64_t)g.tiles[2 * (L / g.mt) + 1] * Tile::RB;
    nend = g.seg[e + 1];
    arow = (int64_t)e * g.M;
    nk = (int)(g.kp / 16);
  }
  const int64_t m0 = (int64_t)mt * Tile::RA;
  floatx16 acc[kTM][kTN];
  if (MODE == kWeight && nk == 0) {
#pragma unroll
    for (int r = 0; r < kTM; r++)
#pragma unroll
      for (int c = 0; c < kTN; c++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[r][c][v] = 0.f;
  } else {
    const Split2Operand A{reinterpret_cast<const uintx4*>(g.A) + kbeg / 8 * g.arows, g.arows, g.kp / 8 * g.arows,
                          arow + m0, arow + g.M - 1};
    const Split2Operand B{reinterpret_cast<const uintx4*>(g.B) + kbeg / 8 * g.brows, g.brows, g.kp / 8 * g.brows, n0,
                          nend - 1};
    std::conditional_t<MODE == kWeight, FarTile, Tile>::run(A, B, nk, smem, acc);
  }
  const int64_t mw = m0 + wm * kTM * 32, nw = n0 + wn * kTN * 32;
  if constexpr (MODE == kWeight) {
    // (turn_kernel's scale and the epilogue's of kBack; st.xtop: of A, st.dtop: of B)
    const int ex = g.back ? seg_exp(g.st.xtop[e]) + grad_seg_exp(g, e) : hidden_seg_exp(g, e) + seg_exp(g.st.dtop[e]);
#pragma unroll
    for (int r = 0; r < kTM; r++)
#pragma unroll
      for (int c = 0; c < kTN; c++) {
        const int64_t col = nw + c * 32 + l32;
        if (col >= g.N) continue;
#pragma unroll
        for (int v = 0; v < 16; v++) {
          const int64_t row = mw + r * 32 + 8 * (v >> 2) + 4 * kh + (v & 3);
          if (row < g.M) f[row * g.N + col] = ldexpf(acc[r][c][v], -ex);
        }
      }
    return;
  } else {
    char* turn = smem + wave * kTurnBytes;
    int* aexp = reinterpret_cast<int*>(smem + kWaves * kTurnBytes);  // of the tile's rows
    for (int i = threadIdx.x; i < Tile::RA; i += 64 * kWaves) aexp[i] = g.aexp[arow + min(m0 + i, g.M - 1)];
    __syncthreads();
    // what a lane knows of its column (position) in block column c
    struct Column {
      int64_t pos;
      int slot, be, oe;  // exponents: of B's row, of the output's
      float wt, dot;
    } col[kTN];
#pragma unroll
    for (int c = 0; c < kTN; c++) {
      const int64_t p = nw + c * 32 + l32, at = p < nend ? p : nend - 1;
      const int sl = p < nend ? g.perm[at] : -1;
      const float w = MODE != kHidden && sl >= 0 ? g.weight[sl] : 0.f;
      col[c].pos = p;
      col[c].slot = sl;
      col[c].wt = w;
      col[c].be = MODE == kHidden ? g.st.xexp[at]
                  : MODE == kBack ? g.st.dexp[at]
                                  : (g.back ? grad_exp(g, at, e, w) : hidden_exp(g, at, e));
      col[c].oe = MODE == kHidden ? hidden_exp(g, at, e) : MODE == kBack ? grad_exp(g, at, e, w) : 0;
      col[c].dot = 0.f;
    }
    const int se1 = MODE == kBack ? grad_seg_exp(g, e) : 0, se2 = MODE == kBack ? hidden_seg_exp(g, e) : 0;
    const int64_t Mp = (g.M + 31) / 32 * 32;
    // One block at a time, in a loop that stays a loop: unrolled, the activations
    // of 128 values a lane are more code than the compiler unrolls, and the
    // accumulators would go to scratch.
#pragma unroll 1
    for (int blk = 0; blk < kTM * kTN; blk++) {
      const int r = blk / kTN;
      floatx16 x16 = acc[0][0];
      Column cl = col[0];
#pragma unroll
      for (int i = 1; i < kTM * kTN; i++)
        if (blk == i) x16 = acc[i / kTN][i % kTN];
#pragma unroll
      for (int i = 1; i < kTN; i++)
        if (blk % kTN == i) cl = col[i];
      const int64_t row0 = mw + r * 32, pos = cl.pos;
      const bool in = pos < nend;
      half4 th[4], tl[4];
      float pre[4][4];  // the block's pre-activations, all loads in flight at once
      if constexpr (MODE == kBack) {
        const float* p = g.pre + (in ? pos : nend - 1) * g.M;
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int64_t k = row0 + 8 * q + 4 * kh;
          if (g.vec) {
            const float4 v = *reinterpret_cast<const float4*>(p + min(k, g.M - 4));
            pre[q][0] = v.x; pre[q][1] = v.y; pre[q][2] = v.z; pre[q][3] = v.w;
          } else {
#pragma unroll
            for (int u = 0; u < 4; u++) pre[q][u] = p[min(k + u, g.M - 1)];
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int64_t k = row0 + 8 * q + 4 * kh;  // four rows of C: k .. k + 3
        float x[4];
        const int* ae = aexp + wm * kTM * 32 + r * 32 + 8 * q + 4 * kh;
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = k + u < g.M ? ldexpf(x16[4 * q + u], -(ae[u] + cl.be)) : 0.f;
        if constexpr (MODE == kSlots) {
          if (cl.slot < 0) continue;
          float* p = f + (int64_t)cl.slot * g.M + k;
          const float w = g.back ? 1.f : cl.wt;
          if (g.vec) {
            if (k < g.M) *reinterpret_cast<float4*>(p) = make_float4(w * x[0], w * x[1], w * x[2], w * x[3]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; u++)
              if (k + u < g.M) p[u] = w * x[u];
          }
        } else {
          half4 h, l;
          if constexpr (MODE == kHidden) {
            if (g.f && in) {
              float* p = f + pos * g.M + k;
              if (g.vec) {
                if (k < g.M) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
              } else {
#pragma unroll
                for (int u = 0; u < 4; u++)
                  if (k + u < g.M) p[u] = x[u];
              }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
              const float a = cl.slot >= 0 && k + u < g.M ? ldexpf(act_apply(x[u], g.act), cl.oe) : 0.f;
              _Float16 hh, ll;
              split2_any(a, hh, ll);
              h[u] = hh;
              l[u] = ll;
            }
          } else {
            const float* up = pre[q];
#pragma unroll
            for (int u = 0; u < 4; u++) {
              const bool ok = cl.slot >= 0 && k + u < g.M;
              float a, slope;
              act_both(up[u], g.act, a, slope);
              const float du = cl.wt * x[u] * slope, hw = cl.wt * a;
              cl.dot += ok ? a * x[u] : 0.f;
              _Float16 hh, ll;
              split2_any(ok ? ldexpf(du, cl.oe) : 0.f, hh, ll);
              h[u] = hh;
              l[u] = ll;
              // with positions as k: du now, weight act(u) after it
              _Float16* to = reinterpret_cast<_Float16*>(turn) + (8 * q + 4 * kh + u) * kPitch + l32;
              split2_any<true>(ok ? ldexpf(du, se1) : 0.f, hh, ll);
              to[0] = hh;
              to[32 * kPitch] = ll;
              split2_any<true>(ok ? ldexpf(hw, se2) : 0.f, hh, ll);
              th[q][u] = hh;
              tl[q][u] = ll;
            }
          }
          if (in && k < Mp) {
            _Float16* p = g.out + ((k / 8) * g.np + pos) * 8 + 4 * kh;
            *reinterpret_cast<half4*>(p) = h;
            *reinterpret_cast<half4*>(p + Mp * g.np) = l;
          }
        }
      }
      if constexpr (MODE == kBack) {
        auto flush = [&](_Float16* __restrict__ out) {
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
          for (int q = 0; q < 2; q++) {
            const int o = 2 * q + kh;
            const int64_t row = row0 + l32, k = nw + blk % kTN * 32 + 8 * o;
            const _Float16* from = reinterpret_cast<const _Float16*>(turn) + l32 * kPitch + 8 * o;
            const half8 h = *reinterpret_cast<const half8*>(from);
            const half8 l = *reinterpret_cast<const half8*>(from + 32 * kPitch);
            if (row < g.M && k < nend) {
              _Float16* to = out + ((k / 8) * g.M + row) * 8;
              *reinterpret_cast<half8*>(to) = h;
              *reinterpret_cast<half8*>(to + g.np * g.M) = l;
            }
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        flush(g.turn1);
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int u = 0; u < 4; u++) {
            _Float16* to = reinterpret_cast<_Float16*>(turn) + (8 * q + 4 * kh + u) * kPitch + l32;
            to[0] = th[q][u];
            to[32 * kPitch] = tl[q][u];
          }
        flush(g.turn2);
      }
      if constexpr (MODE == kBack) {
#pragma unroll
        for (int i = 0; i < kTN; i++)
          if (blk % kTN == i) col[i].dot = cl.dot;
      }
    }
    if constexpr (MODE == kBack) {
#pragma unroll
      for (int c = 0; c < kTN; c++) {
        const float d = col[c].dot + __shfl_xor(col[c].dot, 32, kWave);
        if (kh == 0 && col[c].pos < nend) g.dot[(int64_t)(2 * mt + wm) * g.np + col[c].pos] = d;
      }
    }
  }
}

// dweight[slot] = the sum of its position's partial sums
__global__ __launch_bounds__(256) void dot_kernel(const float* __restrict__ dot, const int* __restrict__ perm,
                                                  const int* __restrict__ nrows, float* __restrict__ dweight,
                                                  int parts, int64_t np) {
  const int64_t pos = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (pos >= *nrows) return;
  const int slot = perm[pos];
  if (slot < 0) return;
  float d = 0.f;
  for (int p = 0; p < parts; p++) d += dot[p * np + pos];
  dweight[slot] = d;
}

constexpr int64_t round64(int64_t n) { return (n + 63) / 64 * 64; }
constexpr int64_t round32(int64_t n) { return (n + 31) / 32 * 32; }

struct Sizes {
  int64_t N, np, Dp, Hp;
  explicit Sizes(const MoeShape& m) {
    N = m.T * m.K;
    np = round32(N + (kPad - 1) * std::min(m.E, N));
    Dp = round32(m.D);
    Hp = round32(m.H);
  }
};

// A bump allocator over a workspace of 256-byte pieces (base null: sizes only).
struct Room {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = reinterpret_cast<T*>(base ? base + used : nullptr);
    used += ((size_t)n * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

// What the gradient needs of the forward.
struct State {
  SlotTables t;
  int *xexp, *xnorm, *xtop, *w1norm;
  float* pre;
};
State state_at(Room& r, const MoeShape& m) {
  const Sizes z(m);
  State s;
  s.t.seg = r.take<int>(m.E + 1);
  s.t.perm = r.take<int>(z.np);
  s.t.tok = r.take<int>(z.np);
  s.t.expert = r.take<int>(z.N);
  s.t.tiles = r.take<int>(2 * (ceil_div(z.N, Tile::RB) + m.E));
  s.t.ntiles = r.take<int>(1);
  s.t.blk = r.take<int>(z.np / kPad);
  s.xexp = r.take<int>(z.np);
  s.xnorm = r.take<int>(z.np);
  s.xtop = r.take<int>(m.E);
  s.w1norm = r.take<int>(m.E);
  return s;
}

int rows_pass(RowsArgs a, hipStream_t s) {
  const dim3 g((unsigned)ceil_div(a.rows, 32));
  const bool vec = a.K % 4 == 0 && (reinterpret_cast<uintptr_t>(a.src) & 15) == 0, regs = a.Kp <= 64 * kRowOctets;
  if (vec && regs) hipLaunchKernelGGL((rows_kernel<true, true>), g, dim3(256), 0, s, a);
  else if (vec) hipLaunchKernelGGL((rows_kernel<true, false>), g, dim3(256), 0, s, a);
  else if (regs) hipLaunchKernelGGL((rows_kernel<false, true>), g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rows_kernel<false, false>), g, dim3(256), 0, s, a);
  NSH_LAUNCHED();
  return 0;
}
int cols_pass(const float* W, _Float16* out, int* exps, int* norm, int64_t K, int64_t Kp, int64_t C, int64_t E,
              hipStream_t s) {
  const dim3 g((unsigned)ceil_div(C, 64), (unsigned)E);
  if (Kp <= 128 * kColOctets)
    hipLaunchKernelGGL(cols_kernel<true>, g, dim3(1024), 0, s, W, out, exps, norm, K, Kp, C, E * C);
  else
    hipLaunchKernelGGL(cols_kernel<false>, g, dim3(1024), 0, s, W, out, exps, norm, K, Kp, C, E * C);
  NSH_LAUNCHED();
  return 0;
}
int preset(int* p, int64_t n, hipStream_t s) {
  hipLaunchKernelGGL(preset_kernel, dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, s, p, (int)n);
  NSH_LAUNCHED();
  return 0;
}

bool sigmoid_bound(int act) { return act == kActSigmoid; }

// Tests' choice of the least slots an expert (any size above 128); 0: the rule.
std::atomic<int64_t> g_split_least{0};

}  // namespace

void set_split_least(int64_t slots) { g_split_least.store(std::max<int64_t>(0, slots), std::memory_order_relaxed); }

// Both products on pieces cost the layouts of the weights (24 bytes an element,
// forward) and some 50 us of passes, and save half of the products' time.  Sorted
// fp32 operands -> this, us, forward and training step: 64 experts of 1024 x 1024,
// slots an expert 192: 473, 1423 -> 511, 1521; 256: 611, 1861 -> 646, 1864; 384:
// 813, 2519 -> 756, 2221; 1024: 1839, 5948 -> 1407, 4327.  16 of 512 x 2048, 384:
// 307, 854 -> 296, 840.  8 of 256 x 256, 1024: 74, 219 -> 136, 359.  Where a size is
// no multiple of 4 the others read it float by float: 10 of 200 x 333, 96: 123, 288
// -> 122, 303; 192: 130, 328 -> 125, 317; 1024: 159, 420 -> 143, 388.
bool split_takes(const MoeShape& m) {
  if (m.D <= 128 || m.H <= 128) return false;
  const int64_t N = m.T * m.K;
  if (const int64_t least = g_split_least.load(std::memory_order_relaxed)) return N >= least * m.E;
  const bool odd = m.D % 4 || m.H % 4;
  return N >= (odd ? 192 : 288) * m.E && (double)N * m.D * m.H >= (odd ? 0x1p28 : 6 * 0x1p30);
}

static size_t split_forward(const MoeShape& m, Room& r, bool state, State* st, int** count, _Float16** xa,
                            _Float16** ha, _Float16** w1, _Float16** w2, int** w1e, int** w2e, float** slots) {
  const Sizes z(m);
  if (!state) *st = state_at(r, m);
  *count = r.take<int>(sort_count_ints(z.N, m.E));
  *xa = r.take<_Float16>(2 * z.Dp * z.np);
  *ha = r.take<_Float16>(2 * z.Hp * z.np);
  *w1 = r.take<_Float16>(2 * z.Dp * m.E * m.H);
  *w2 = r.take<_Float16>(2 * z.Hp * m.E * m.D);
  *w1e = r.take<int>(m.E * m.H);
  *w2e = r.take<int>(m.E * m.D + m.E);  // (and W2's norms, which nothing reads)
  *slots = r.take<float>(z.N * m.D);
  return r.used;
}

struct Backward {
  int *dexp, *dnorm, *dtop, *dw, *xw, *w2norm, *w1norm2, *w1r, *w2r, *kitems;
  _Float16 *da, *du, *xt, *dyt, *dut, *hwt, *wr;
  float *slots, *dot, *kpart;
};
static Backward split_backward(const MoeShape& m, Room& r) {
  const Sizes z(m);
  Backward b;
  b.dexp = r.take<int>(z.np);
  b.dnorm = r.take<int>(z.np);
  b.dtop = r.take<int>(5 * m.E);  // dtop, dw, xw, w2norm, w1norm2: preset together
  b.dw = b.dtop + m.E;
  b.xw = b.dw + m.E;
  b.w2norm = b.xw + m.E;
  b.w1norm2 = b.w2norm + m.E;
  b.w1r = r.take<int>(m.E * m.D);
  b.w2r = r.take<int>(m.E * m.H);
  b.kitems = r.take<int>(moe_bwd_kitem_ints(z.np, m.D, m.H, m.E));
  b.da = r.take<_Float16>(2 * z.Dp * z.np);
  b.du = r.take<_Float16>(2 * z.Hp * z.np);
  b.xt = r.take<_Float16>(2 * z.np * m.D);
  b.dyt = r.take<_Float16>(2 * z.np * m.D);
  b.dut = r.take<_Float16>(2 * z.np * m.H);
  b.hwt = r.take<_Float16>(2 * z.np * m.H);
  // W2's rows, then (its product done) W1's
  b.wr = r.take<_Float16>(std::max(2 * z.Dp * m.E * m.H, 2 * z.Hp * m.E * m.D));
  b.slots = r.take<float>(z.N * m.D);
  b.dot = r.take<float>(2 * ceil_div(m.H, Tile::RA) * z.np);
  b.kpart = r.take<float>(moe_bwd_kpart_floats(z.np, m.D, m.H));
  return b;
}

size_t split_state_bytes(const MoeShape& m) {
  Room r{nullptr};
  state_at(r, m);
  r.take<float>(Sizes(m).np * m.H);
  return r.used;
}

size_t split_workspace_bytes(const MoeShape& m, bool grad) {
  Room f{nullptr}, b{nullptr};
  State st;
  int *count, *w1e, *w2e;
  _Float16 *xa, *ha, *w1, *w2;
  float* slots;
  split_forward(m, f, false, &st, &count, &xa, &ha, &w1, &w2, &w1e, &w2e, &slots);
  if (grad) split_backward(m, b);
  return std::max(f.used, b.used);
}

static SplitArgs split_args(const MoeShape& m, const State& st, int64_t M, int act) {
  const Sizes z(m);
  SplitArgs g{};
  g.M = M;
  g.seg = st.t.seg; g.perm = st.t.perm; g.tiles = st.t.tiles; g.ntiles = st.t.ntiles;
  g.mt = (int)ceil_div(M, Tile::RA);
  g.act = act;
  g.sigmoid = sigmoid_bound(act);
  g.np = z.np;
  g.st.xexp = st.xexp; g.st.xnorm = st.xnorm; g.st.xtop = st.xtop; g.st.w1norm = st.w1norm;
  return g;
}

template <int MODE>
static int split_product(const SplitArgs& g, int64_t entries, hipStream_t s) {
  hipLaunchKernelGGL(split_kernel<MODE>, dim3((unsigned)(entries * g.mt * (MODE == kWeight ? g.nt : 1))),
                     dim3(64 * waves_of(MODE)), 0, s, g);
  NSH_LAUNCHED();
  return 0;
}

static bool float4_rows(int64_t M, const void* p) { return M % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int launch_experts_split(const float* x, const int32_t* idx, const float* weight, const float* W1, const float* W2,
                         float* y, const MoeShape& m, int act, void* state, void* workspace, hipStream_t s) {
  const Sizes z(m);
  Room r{static_cast<char*>(workspace)}, rs{static_cast<char*>(state)};
  State st;
  int *count, *w1e, *w2e;
  _Float16 *xa, *ha, *w1, *w2;
  float *slots, *pre = nullptr;
  if (state) {
    st = state_at(rs, m);
    pre = rs.take<float>(z.np * m.H);
  }
  split_forward(m, r, state != nullptr, &st, &count, &xa, &ha, &w1, &w2, &w1e, &w2e, &slots);
  if (launch_sort_slots(idx, st.t, count, z.N, (int)m.K, (int)m.E, kPad, Tile::RB, z.np, s) != 0) return -1;
  if (preset(st.w1norm, m.E, s) != 0 || preset(st.xtop, m.E, s) != 0) return -1;
  RowsArgs a{};
  a.src = x; a.tok = st.t.tok; a.perm = st.t.perm; a.blk = st.t.blk; a.nrows = st.t.seg + m.E;
  a.out = xa; a.exps = st.xexp; a.norm = st.xnorm; a.top = st.xtop;
  a.rows = z.np; a.K = m.D; a.Kp = z.Dp;
  if (rows_pass(a, s) != 0) return -1;
  if (cols_pass(W1, w1, w1e, st.w1norm, m.D, z.Dp, m.H, m.E, s) != 0) return -1;
  const int64_t entries = ceil_div(z.N, Tile::RB) + m.E;
  SplitArgs g = split_args(m, st, m.H, act);
  g.A = w1; g.arows = m.E * m.H; g.aexp = w1e;
  g.B = xa; g.brows = z.np; g.kp = z.Dp;
  g.f = pre; g.vec = float4_rows(m.H, pre);
  g.out = ha;
  if (split_product<kHidden>(g, entries, s) != 0) return -1;
  if (cols_pass(W2, w2, w2e, w2e + m.E * m.D, m.H, z.Hp, m.D, m.E, s) != 0) return -1;
  SplitArgs o = split_args(m, st, m.D, act);
  o.A = w2; o.arows = m.E * m.D; o.aexp = w2e;
  o.B = ha; o.brows = z.np; o.kp = z.Hp;
  o.weight = weight;
  o.f = slots; o.vec = float4_rows(m.D, slots);
  if (split_product<kSlots>(o, entries, s) != 0) return -1;
  return launch_combine(slots, st.t.expert, y, m, s);
}

int launch_experts_split_grad(const float* dy, const float* x, const float* weight, const float* W1, const float* W2,
                              const void* state, float* dx, float* dweight, float* dW1, float* dW2, const MoeShape& m,
                              int act, void* workspace, hipStream_t s) {
  const Sizes z(m);
  Room rs{static_cast<char*>(const_cast<void*>(state))}, r{static_cast<char*>(workspace)};
  const State st = state_at(rs, m);
  const float* pre = rs.take<float>(z.np * m.H);
  const Backward b = split_backward(m, r);
  const int* nrows = st.t.seg + m.E;
  const int64_t entries = ceil_div(z.N, Tile::RB) + m.E;
  if (preset(b.dtop, 5 * m.E, s) != 0) return -1;
  // dy by position, with the largest norm times weight of each expert; W2's rows
  RowsArgs a{};
  a.src = dy; a.tok = st.t.tok; a.perm = st.t.perm; a.blk = st.t.blk; a.nrows = nrows; a.weight = weight;
  a.out = b.da; a.exps = b.dexp; a.norm = b.dnorm; a.top = b.dtop; a.wnorm = b.dw;
  a.rows = z.np; a.K = m.D; a.Kp = z.Dp;
  if (rows_pass(a, s) != 0) return -1;
  RowsArgs w{};
  w.src = W2; w.out = b.wr; w.exps = b.w2r; w.norm = b.w2norm; w.per_expert = (int)m.H;
  w.rows = m.E * m.H; w.K = m.D; w.Kp = z.Dp;
  if (rows_pass(w, s) != 0) return -1;
  hipLaunchKernelGGL(weight_norm_kernel, dim3((unsigned)ceil_div(z.np, 256)), dim3(256), 0, s, st.xnorm, st.t.perm,
                     st.t.blk, nrows, weight, sigmoid_bound(act), b.xw);
  NSH_LAUNCHED();
  auto with_stats = [&](SplitArgs g) {
    g.weight = weight;
    g.st.dexp = b.dexp; g.st.dnorm = b.dnorm; g.st.dtop = b.dtop; g.st.dw = b.dw; g.st.xw = b.xw;
    g.st.w2norm = b.w2norm;
    return g;
  };
  SplitArgs g = with_stats(split_args(m, st, m.H, act));
  g.A = b.wr; g.arows = m.E * m.H; g.aexp = b.w2r;
  g.B = b.da; g.brows = z.np; g.kp = z.Dp;
  g.pre = pre; g.vec = float4_rows(m.H, pre);
  g.out = b.du; g.turn1 = b.dut; g.turn2 = b.hwt; g.dot = b.dot;
  if (split_product<kBack>(g, entries, s) != 0) return -1;
  if (dweight) {
    if (launch_fill(dweight, z.N, 0.f, s) != 0) return -1;
    hipLaunchKernelGGL(dot_kernel, dim3((unsigned)ceil_div(z.np, 256)), dim3(256), 0, s, b.dot, st.t.perm, nrows, dweight,
                       2 * g.mt, z.np);
    NSH_LAUNCHED();
  }
  if (dx) {
    RowsArgs v{};
    v.src = W1; v.out = b.wr; v.exps = b.w1r; v.norm = b.w1norm2; v.per_expert = (int)m.D;
    v.rows = m.E * m.D; v.K = m.H; v.Kp = z.Hp;
    if (rows_pass(v, s) != 0) return -1;
    SplitArgs o = with_stats(split_args(m, st, m.D, act));
    o.A = b.wr; o.arows = m.E * m.D; o.aexp = b.w1r;
    o.B = b.du; o.brows = z.np; o.kp = z.Hp;
    o.back = 1;
    o.f = b.slots; o.vec = float4_rows(m.D, b.slots);
    if (split_product<kSlots>(o, entries, s) != 0) return -1;
    if (launch_combine(b.slots, st.t.expert, dx, m, s) != 0) return -1;
  }
  if (!dW1 && !dW2) return 0;
  if (launch_moe_kitems(st.t.seg, b.kitems, nullptr, z.np, m.D, m.H, m.E, s) != 0) return -1;
  const int64_t items = moe_bwd_most_items(z.np, m.D, m.H, m.E);
  auto weight_grad = [&](const float* src, const int* top, _Float16* turned, const _Float16* A, const _Float16* B,
                         int64_t M, int64_t N, int back, float* out) -> int {
    hipLaunchKernelGGL(turn_kernel, dim3((unsigned)(z.np / kPad * ceil_div(m.D, 64))), dim3(256), 0, s, src,
                       st.t.tok, st.t.blk, nrows, top, turned, m.D, z.np);
    NSH_LAUNCHED();
    SplitArgs k = with_stats(split_args(m, st, M, act));
    k.A = A; k.arows = M;
    k.B = B; k.brows = N; k.kp = z.np; k.N = N;
    k.nt = (int)ceil_div(N, Tile::RB);
    k.items = b.kitems + 2; k.nitems = b.kitems; k.kpart = b.kpart;
    k.back = back;
    k.f = out;
    if (split_product<kWeight>(k, items, s) != 0) return -1;
    return launch_moe_kpart_sum(out, M * N, b.kitems, b.kpart, z.np, m.D, m.H, m.E, s);
  };
  if (dW1 && weight_grad(x, st.xtop, b.xt, b.xt, b.dut, m.D, m.H, 1, dW1) != 0) return -1;
  if (dW2 && weight_grad(dy, b.dtop, b.dyt, b.hwt, b.dyt, m.H, m.D, 0, dW2) != 0) return -1;
  return 0;
}

}  // namespace nship
