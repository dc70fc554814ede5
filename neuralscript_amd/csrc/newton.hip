// Newton-Schulz orthogonalisation of n matrices [r, c], and the Muon step that
// takes its update from it.
//
//   X = G / (|G|_F + 1e-7);  steps times: S = X X^T, P = a I + b S + c S S, X = P X
//
// with X held wide ([m, N], m = min(r, c) <= N): each step maps every singular
// value s to a s + b s^3 + c s^5, which in five steps ends between about 0.7
// and 1.2 for all but the smallest.
//
// Three products a step, m^2 N (half of a symmetric result), m^3 (half again)
// and 2 m^2 N FLOP; bound by the matrix cores from some hundred rows on, below
// by launches and the latency of a slab's loads.
//
// Products of two fp16 pieces (split2.h).  The map keeps |X| and |S| (entries and
// singular values) below 1.21^2 and |P| below 3.45 whatever G is, so one power of
// two per operand puts every entry into fp16's range.  Measured against 64 bits,
// relative, fp32 products and these: 8 of 64 x 256 1.5e-6, 1.3e-6; 333 x 1000
// 2.2e-6, 1.1e-6.
//
// One scale a matrix leaves the entries of a small row or column of G (an embedding's
// row that few tokens read) far below it, so the low pieces are held times 2^11: an
// entry of X keeps its 22 bits down to 2^-29, and below that an absolute 2^-51.
// Relative errors of every third row of 512 x 2048 at 1e-4, 1e-6, 1e-8 of the others,
// by themselves: 3.2e-7, 4.0e-7, 2.7e-5 (fp32 3.3e-7); with low pieces beside the high
// ones 4.9e-6, 4.9e-4, 4.9e-2, for which the products of 64 of 1024 x 1024 took 4% less.
//
// The norm's 1e-7 leaves X0 small where G is.  X is then held times 2^e, e = e0 -
// 2 k at step k and not below 0 (a step grows X by at most 3.4445), so that its
// entries keep their bits.
//
// Operands are padded with zeros to a contraction length of 32 k.  X is kept both
// ways, as the Gram product's operand (rows m, contraction N) and as the update's
// (rows N, contraction m); S and P are symmetric and need one.
#include <algorithm>
#include <atomic>

#include "common.h"
#include "kernels.h"
#include "split2.h"

namespace nship {
namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr double kNsEps = 1e-7;
constexpr int kNormParts = 256;  // partial sums of a matrix's norm
// the operands' powers of two: X and S below 2 x 2^15 = fp16's range, P below 4 x 2^14
constexpr float kUpX = 0x1p15f, kUpS = 0x1p15f, kUpP = 0x1p14f;

// What a product is for, i.e. its epilogue.
enum NsMode : int { kGram = 0, kPoly, kUpdate, kLast };

struct NsArgs {
  const _Float16* A;   // rows ra, contraction k (a multiple of 32)
  const _Float16* B;   // rows rb
  int64_t ra, rb, k;
  int64_t sA, sB;      // matrix to matrix, halves
  int tiles_m, tiles_n, tiles;  // of a matrix (symmetric: its lower triangle)
  int n;
  _Float16* out;       // kGram: S, kPoly: P, kUpdate: X as the Gram's operand [.][kout2 / 8][ra][8]
  _Float16* out2;      // kUpdate: X as the update's operand [.][kout / 8][rb][8]
  const _Float16* S;   // kPoly
  int64_t sOut, sOut2;
  int64_t kout, kout2; // padded contraction lengths of the outputs: of rows ra as k, of rows rb as k
  float* f;            // kLast: q or w [ra][rb] per matrix
  float le, decay;
  int weights;         // kLast: f = f - le x - decay f
  const int* ex;       // e0 of every matrix
  int step;
};

// Tile of linear index t: by rows, or of a lower triangle (tn <= tm) by rows.
template <bool SYM>
__device__ __forceinline__ void ns_tile(int t, int tiles_n, int& tm, int& tn) {
  if (SYM) {
    tm = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((int64_t)tm * (tm + 1) / 2 > t) tm--;
    while ((int64_t)(tm + 1) * (tm + 2) / 2 <= t) tm++;
    tn = t - tm * (tm + 1) / 2;
  } else {
    tm = t / tiles_n;
    tn = t - tm * tiles_n;
  }
}

constexpr int kPitch = 40;                       // halves of a transposing tile's row
constexpr int kTurnBytes = 2 * 32 * kPitch * 2;  // of a wave's transposing tile

// One wave's TM x TN blocks of 32x32 from (mw, nw), by what the product is for.
// turn: kTurnBytes of LDS of the wave's own.  diagonal: a symmetric result's
// tile on the diagonal.
template <int MODE, int TM, int TN>
__device__ __forceinline__ void ns_epilogue(const NsArgs& g, const floatx16 (&acc)[TM][TN], char* turn, int mat,
                                            int64_t mw, int64_t nw, int l32, int kh, bool diagonal) {
  constexpr bool kSym = MODE == kGram || MODE == kPoly;
  // Accumulator v of lane (l32, kh) in a 32x32 block: row 8 (v / 4) + 4 kh + v % 4, column l32.
  const int ex = max(0, g.ex[mat] - 2 * g.step);  // X = 2^-ex times what is held
  if constexpr (MODE == kLast) {
    float* __restrict__ f = g.f + mat * g.ra * g.rb;
#pragma unroll
    for (int r = 0; r < TM; r++)
#pragma unroll
      for (int c = 0; c < TN; c++) {
        const int64_t col = nw + c * 32 + l32, row0 = mw + r * 32 + 4 * kh;
        if (col >= g.rb) continue;
        float* p = f + row0 * g.rb + col;
        float w[16];  // (all loads before the stores, which may alias them for all the compiler knows)
#pragma unroll
        for (int v = 0; v < 16; v++) {
          const int dr = 8 * (v >> 2) + (v & 3);
          w[v] = g.weights && row0 + dr < g.ra ? p[dr * g.rb] : 0.f;
        }
#pragma unroll
        for (int v = 0; v < 16; v++) {
          const int dr = 8 * (v >> 2) + (v & 3);
          // (not times 2^-ex 2^-29, which underflows where X still does not)
          const float x = ldexpf(acc[r][c][v] * (1.f / (kUpX * kUpP)), -ex);
          if (row0 + dr < g.ra) p[dr * g.rb] = g.weights ? w[v] - g.le * x - g.decay * w[v] : x;
        }
      }
    return;
  } else {
    // (S is held times 2^2ex)
    const float by = MODE == kGram     ? kUpS / (kUpX * kUpX)
                     : MODE == kUpdate ? ldexpf(1.f / kUpP, max(0, ex - 2) - ex)
                                       : ldexpf(kNsC * kUpP / (kUpS * kUpS), -4 * ex);
    const float bs = ldexpf(kNsB * kUpP / kUpS, -2 * ex);
    _Float16* __restrict__ out = g.out + mat * g.sOut;
    _Float16* __restrict__ out2 = (kSym ? g.out : g.out2) + mat * (kSym ? g.sOut : g.sOut2);
    const int64_t piece2 = g.kout * g.rb, piece = g.kout2 * g.ra;
#pragma unroll
    for (int r = 0; r < TM; r++)
#pragma unroll
      for (int c = 0; c < TN; c++) {
        const int64_t row0 = mw + r * 32, col0 = nw + c * 32, col = col0 + l32;
        // as [k = row][col]: four consecutive k of a column, half a chunk
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int64_t k = row0 + 8 * q + 4 * kh;
          const int64_t at = ((k / 8) * g.rb + col) * 8 + 4 * kh;
          const bool in = col < g.rb && k < g.kout;
          half4 h, l;
          half4 sh = {0, 0, 0, 0}, sl = {0, 0, 0, 0};
          if (MODE == kPoly && in) {  // (S is symmetric: its [k = row][col] is its (row, col))
            const _Float16* s = g.S + mat * g.sOut + at;
            sh = *reinterpret_cast<const half4*>(s);
            sl = *reinterpret_cast<const half4*>(s + piece2);
          }
#pragma unroll
          for (int u = 0; u < 4; u++) {
            float x = acc[r][c][4 * q + u] * by;
            if (MODE == kPoly)
              x += (k + u == col ? kNsA * kUpP : 0.f) + bs * join2_far(sh[u], sl[u]);
            x = k + u < g.ra && col < g.rb ? x : 0.f;  // (padding)
            _Float16 hh, ll;
            split2_far(x, hh, ll);
            h[u] = hh;
            l[u] = ll;
          }
          if (in) {
            *reinterpret_cast<half4*>(out2 + at) = h;
            *reinterpret_cast<half4*>(out2 + piece2 + at) = l;
          }
          _Float16* to = reinterpret_cast<_Float16*>(turn) + (8 * q + 4 * kh) * kPitch + l32;
#pragma unroll
          for (int u = 0; u < 4; u++) {
            to[u * kPitch] = h[u];
            to[u * kPitch + 32 * kPitch] = l[u];
          }
        }
        if (diagonal) continue;  // (the other way round lies in the same tile)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // as [k = col][row]: a whole chunk of a row
#pragma unroll
        for (int q = 0; q < 2; q++) {
          const int o = 2 * q + kh;
          const int64_t row = row0 + l32, k = col0 + 8 * o;
          const _Float16* from = reinterpret_cast<const _Float16*>(turn) + l32 * kPitch + 8 * o;
          const half8 h = *reinterpret_cast<const half8*>(from);
          const half8 l = *reinterpret_cast<const half8*>(from + 32 * kPitch);
          if (row < g.ra && k < g.kout2) {
            _Float16* to = out + ((k / 8) * g.ra + row) * 8;
            *reinterpret_cast<half8*>(to) = h;
            *reinterpret_cast<half8*>(to + piece) = l;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
  }
}

// One tile of C = A B^T (split2.h).
template <int MODE, int WM, int WN, int TM, int TN, int KS>
__global__ __launch_bounds__(64 * WM * WN, 2) void ns_gemm_kernel(NsArgs g) {
  using Tile = Split2Tile<WM, WN, TM, TN, KS, true>;
  static_assert(kTurnBytes * WM * WN <= Tile::kLds, "the transposing tiles fit");
  constexpr bool kSym = MODE == kGram || MODE == kPoly;
  static_assert(!kSym || Tile::RA == Tile::RB, "a symmetric result's tiles are square");
  __shared__ __attribute__((aligned(16))) char smem[Tile::kLds];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int L = split2_xcd_linear(blockIdx.x, g.tiles * g.n);
  const int mat = L / g.tiles;
  int tm, tn;
  ns_tile<kSym>(L % g.tiles, g.tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * Tile::RA, n0 = (int64_t)tn * Tile::RB;
  floatx16 acc[TM][TN];
  const Split2Operand A{reinterpret_cast<const uintx4*>(g.A + mat * g.sA), g.ra, g.k / 8 * g.ra, m0, g.ra - 1};
  const Split2Operand B{reinterpret_cast<const uintx4*>(g.B + mat * g.sB), g.rb, g.k / 8 * g.rb, n0, g.rb - 1};
  Tile::run(A, B, (int)(g.k / KS), smem, acc);
  ns_epilogue<MODE, TM, TN>(g, acc, smem + wave * kTurnBytes, mat, m0 + wm * TM * 32, n0 + wn * TN * 32, lane & 31,
                            lane >> 5, kSym && tm == tn);
}

// The same product where larger tiles leave most CUs idle: 32 x 32 outputs a
// workgroup, whose K is dealt out in 16-steps to eight waves that take their
// operands straight into registers, kFewU steps at a time and without barriers;
// the eight sums meet in LDS.  Bound by what a CU can pull from the L2 (64 rows
// of K a tile) and its one or two round trips.  Measured and not kept: 64 x 64
// tiles with K dealt out to four waves of each 32 x 32 block (fewer CUs pull
// more; 3 of 1000 x 333: Gram product 15 us).
constexpr int kFewU = 8;
template <int MODE>
__global__ __launch_bounds__(512) void ns_few_kernel(NsArgs g) {
  constexpr bool kSym = MODE == kGram || MODE == kPoly;
  __shared__ __attribute__((aligned(16))) float part[7][1024];
  const int t = threadIdx.x, lane = t & 63, l32 = lane & 31, kh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int L = split2_xcd_linear(blockIdx.x, g.tiles * g.n);
  const int mat = L / g.tiles;
  int tm, tn;
  ns_tile<kSym>(L % g.tiles, g.tiles_n, tm, tn);
  const int64_t mw = (int64_t)tm * 32, nw = (int64_t)tn * 32;
  floatx16 acc, low;
#pragma unroll
  for (int v = 0; v < 16; v++) acc[v] = low[v] = 0.f;
  {
    // chunk (piece, octet 2 s + kh, row) of step s
    const half8* pa = reinterpret_cast<const half8*>(g.A + mat * g.sA) + kh * g.ra + min(mw + l32, g.ra - 1);
    const half8* pb = reinterpret_cast<const half8*>(g.B + mat * g.sB) + kh * g.rb + min(nw + l32, g.rb - 1);
    const int64_t la = g.k / 8 * g.ra, lb = g.k / 8 * g.rb;  // to the other piece
    const int all = (int)(g.k / 16);
    // steps s, s + 8, .. of this wave
    auto steps = [&](int s0, auto count) {
      constexpr int CNT = decltype(count)::value;
      half8 a[CNT][2], b[CNT][2];
#pragma unroll
      for (int u = 0; u < CNT; u++) {
        const int64_t o = 2 * ((int64_t)s0 + 8 * u);
        a[u][0] = pa[o * g.ra];
        a[u][1] = pa[o * g.ra + la];
        b[u][0] = pb[o * g.rb];
        b[u][1] = pb[o * g.rb + lb];
      }
      __builtin_amdgcn_sched_barrier(0);  // (all loads first)
#pragma unroll
      for (int u = 0; u < CNT; u++) {
        low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[u][1], b[u][0], low, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[u][0], b[u][0], acc, 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[u][0], b[u][1], low, 0, 0, 0);
      }
    };
    int s = wave;
    for (; s + 8 * (kFewU - 1) < all; s += 8 * kFewU) steps(s, std::integral_constant<int, kFewU>{});
    if (s + 8 * 3 < all) {
      steps(s, std::integral_constant<int, 4>{});
      s += 32;
    }
    if (s + 8 < all) {
      steps(s, std::integral_constant<int, 2>{});
      s += 16;
    }
    if (s < all) steps(s, std::integral_constant<int, 1>{});
  }
#pragma unroll
  for (int v = 0; v < 16; v++) acc[v] += kLowDown * low[v];
  if (wave > 0) {
#pragma unroll
    for (int v = 0; v < 16; v++) part[wave - 1][v * 64 + lane] = acc[v];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int q = 0; q < 7; q++)
#pragma unroll
    for (int v = 0; v < 16; v++) acc[v] += part[q][v * 64 + lane];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  floatx16 one[1][1] = {{acc}};
  ns_epilogue<MODE, 1, 1>(g, one, reinterpret_cast<char*>(part), mat, mw, nw, l32, kh, kSym && tm == tn);
}

// ... and between the two: 64 x 64 outputs a workgroup, each of the eight waves
// with the whole tile over its share of K (half of the loads a product that 32 x
// 32 outputs take), the eight sums met in LDS, where wave (i, j) of the first four
// takes its block's.
constexpr int kMidU = 2;
template <int MODE>
__global__ __launch_bounds__(512) void ns_mid_kernel(NsArgs g) {
  constexpr bool kSym = MODE == kGram || MODE == kPoly;
  __shared__ __attribute__((aligned(16))) float part[4][4][1024];  // [wave pair][block]
  const int t = threadIdx.x, lane = t & 63, l32 = lane & 31, kh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int L = split2_xcd_linear(blockIdx.x, g.tiles * g.n);
  const int mat = L / g.tiles;
  int tm, tn;
  ns_tile<kSym>(L % g.tiles, g.tiles_n, tm, tn);
  const int64_t mw = (int64_t)tm * 64, nw = (int64_t)tn * 64;
  floatx16 acc[2][2], low[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] = low[i][j][v] = 0.f;
  {
    const half8 *pa[2], *pb[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      pa[i] = reinterpret_cast<const half8*>(g.A + mat * g.sA) + kh * g.ra + min(mw + 32 * i + l32, g.ra - 1);
      pb[i] = reinterpret_cast<const half8*>(g.B + mat * g.sB) + kh * g.rb + min(nw + 32 * i + l32, g.rb - 1);
    }
    const int64_t la = g.k / 8 * g.ra, lb = g.k / 8 * g.rb;  // to the other piece
    const int all = (int)(g.k / 16);
    auto steps = [&](int s0, auto count) {
      constexpr int CNT = decltype(count)::value;
      half8 a[CNT][2][2], b[CNT][2][2];
#pragma unroll
      for (int u = 0; u < CNT; u++) {
        const int64_t o = 2 * ((int64_t)s0 + 8 * u);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          a[u][i][0] = pa[i][o * g.ra];
          a[u][i][1] = pa[i][o * g.ra + la];
          b[u][i][0] = pb[i][o * g.rb];
          b[u][i][1] = pb[i][o * g.rb + lb];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < CNT; u++)
#pragma unroll
        for (int q = 0; q < 3; q++)  // l h, h h, h l
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
              floatx16& to = q == 1 ? acc[i][j] : low[i][j];
              to = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[u][i][q == 0], b[u][j][q == 2], to, 0, 0, 0);
            }
    };
    int s = wave;
    for (; s + 8 * (kMidU - 1) < all; s += 8 * kMidU) steps(s, std::integral_constant<int, kMidU>{});
    if (s < all) steps(s, std::integral_constant<int, 1>{});
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] += kLowDown * low[i][j][v];
  if (wave >= 4) {
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int v = 0; v < 16; v++) part[wave - 4][q][v * 64 + lane] = acc[q >> 1][q & 1][v];
  }
  __syncthreads();
  if (wave < 4) {
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int v = 0; v < 16; v++) {
        acc[q >> 1][q & 1][v] += part[wave][q][v * 64 + lane];
        part[wave][q][v * 64 + lane] = acc[q >> 1][q & 1][v];
      }
  }
  __syncthreads();
  floatx16 one[1][1];
  if (wave < 4) {
#pragma unroll
    for (int v = 0; v < 16; v++)
      one[0][0][v] = (part[0][wave][v * 64 + lane] + part[1][wave][v * 64 + lane]) +
                     (part[2][wave][v * 64 + lane] + part[3][wave][v * 64 + lane]);
  }
  __syncthreads();
  if (wave >= 4) return;
  ns_epilogue<MODE, 1, 1>(g, one, reinterpret_cast<char*>(part) + wave * kTurnBytes, mat, mw + (wave >> 1) * 32,
                          nw + (wave & 1) * 32, l32, kh, kSym && tm == tn);
}

__device__ __forceinline__ float update_of(float g, float m, float mu, int nesterov) {
  return nesterov ? g + mu * m : m;
}

// part[matrix][block] = sum of squares of the update's elements, in 64 bits:
// gradients of 1e-25 and 1e25 have squares that 32 bits cannot hold.
__global__ __launch_bounds__(256) void ns_norm_kernel(const float* __restrict__ g, float* __restrict__ m, float mu,
                                                      int nesterov, int64_t elems, double* __restrict__ part) {
  __shared__ double red[4];
  const int64_t base = (int64_t)blockIdx.y * elems;
  double sum = 0.;
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < elems; i0 += 8 * step) {
    float u[8], mm[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t i = min(i0 + j * step, elems - 1);
      u[j] = g[base + i];
      if (m) mm[j] = m[base + i];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int64_t i = i0 + j * step;
      if (i >= elems) break;
      if (m) {
        mm[j] = mu * mm[j] + u[j];
        m[base + i] = mm[j];
        u[j] = update_of(u[j], mm[j], mu, nesterov);
      }
      sum += (double)u[j] * u[j];
    }
  }
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)blockIdx.y * kNormParts + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// e0: 2^e0 |X0| in (1/2, 1].  (|X0| is at least 1e-38.)
__device__ __forceinline__ int ns_exponent(double x0) { return x0 > 0. ? max(0, min(126, ilogb(1. / x0))) : 0; }

// 1 / (|u|_F + 1e-7) from the partial sums; NaN where the norm is not finite,
// so that the whole matrix is.
__device__ __forceinline__ double ns_scale(const double* __restrict__ part, int parts, int* ex = nullptr) {
  const int lane = threadIdx.x & 63;
  double x[kNormParts / 64], some = 0.;
#pragma unroll
  for (int i = 0; i < kNormParts / 64; i++) x[i] = part[min(lane + 64 * i, parts - 1)];
#pragma unroll
  for (int i = 0; i < kNormParts / 64; i++) some += lane + 64 * i < parts ? x[i] : 0.;
  const double sq = wave_sum(some);
  const double norm = sqrt(sq), by = sq < __builtin_inf() ? 1. / (norm + kNsEps) : __builtin_nan("");
  if (ex) *ex = ns_exponent(norm * by);
  return by;
}

// X = the update over its norm in both layouts, a tile of 64 x 64 of X a
// workgroup: gram [.][Np / 8][m][8], upd [.][mp / 8][N][8].
struct NsStart {
  const float* g;
  const float* m;
  float mu;
  int nesterov;
  int64_t r, c;
  int parts, tiles_n;
  const double* part;
  int* ex;
  _Float16* gram;
  _Float16* upd;
  int64_t M, N, mp, np;
};
__global__ __launch_bounds__(256) void ns_start_kernel(NsStart a) {
  __shared__ float x[64][65];  // [i][j] of X
  const int64_t elems = a.r * a.c, base = (int64_t)blockIdx.y * elems;
  const int64_t i0 = (int64_t)(blockIdx.x / a.tiles_n) * 64, j0 = (int64_t)(blockIdx.x % a.tiles_n) * 64;
  const int t = threadIdx.x, lo = t & 63, hi = t >> 6;
  const bool tall = a.r > a.c;
  float u[16];
#pragma unroll
  for (int q = 0; q < 16; q++) {
    const int h = hi + 4 * q;  // (lanes run along g's rows)
    const int64_t i = i0 + (tall ? lo : h), j = j0 + (tall ? h : lo);
    u[q] = 0.f;
    if (i < a.M && j < a.N) {
      const int64_t at = base + (tall ? j * a.c + i : i * a.c + j);
      u[q] = a.g[at];
      if (a.m) u[q] = update_of(u[q], a.m[at], a.mu, a.nesterov);
    }
  }
  int ex;
  const double by = ns_scale(a.part + (int64_t)blockIdx.y * kNormParts, a.parts, &ex);
  const double up = ldexp(by * kUpX, ex);
  if (blockIdx.x == 0 && t == 0) a.ex[blockIdx.y] = ex;
#pragma unroll
  for (int q = 0; q < 16; q++) {
    const int h = hi + 4 * q;
    const float v = (float)(u[q] * up);
    if (tall) x[lo][h] = v;
    else x[h][lo] = v;
  }
  __syncthreads();
  const int64_t pg = a.np * a.M, pu = a.mp * a.N;
  _Float16* __restrict__ gram = a.gram + blockIdx.y * 2 * pg;
  _Float16* __restrict__ upd = a.upd + blockIdx.y * 2 * pu;
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const int o = hi + 4 * q;
    half8 h, l;
    if (i0 + lo < a.M && j0 + 8 * o < a.np) {
#pragma unroll
      for (int u = 0; u < 8; u++) {
        _Float16 hh, ll;
        split2_far(x[lo][8 * o + u], hh, ll);
        h[u] = hh;
        l[u] = ll;
      }
      _Float16* to = gram + ((j0 / 8 + o) * a.M + i0 + lo) * 8;
      *reinterpret_cast<half8*>(to) = h;
      *reinterpret_cast<half8*>(to + pg) = l;
    }
    if (j0 + lo < a.N && i0 + 8 * o < a.mp) {
#pragma unroll
      for (int u = 0; u < 8; u++) {
        _Float16 hh, ll;
        split2_far(x[8 * o + u][lo], hh, ll);
        h[u] = hh;
        l[u] = ll;
      }
      _Float16* to = upd + ((i0 / 8 + o) * a.N + j0 + lo) * 8;
      *reinterpret_cast<half8*>(to) = h;
      *reinterpret_cast<half8*>(to + pu) = l;
    }
  }
}

// No steps: the update over its norm itself.
__global__ __launch_bounds__(256) void ns_normalise_kernel(const float* g, const float* __restrict__ m, float mu,
                                                           int nesterov, int64_t elems, int parts,
                                                           const double* __restrict__ part, float* q,
                                                           float* __restrict__ w, float le, float decay) {
  const int64_t base = (int64_t)blockIdx.y * elems;
  const double by = ns_scale(part + (int64_t)blockIdx.y * kNormParts, parts);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (int64_t)gridDim.x * 256) {
    float u = g[base + i];
    if (m) u = update_of(u, m[base + i], mu, nesterov);
    const float x = (float)(u * by);
    if (w) w[base + i] = w[base + i] - le * x - decay * w[base + i];
    else q[base + i] = x;
  }
}

// A small matrix's whole orthogonalisation by one workgroup of 16 waves: X both
// ways and S (then P in its place) in LDS as the products above hold them, padded
// to 32 and with a row more between octets (the epilogues' stores along k then
// spread over the banks): up to 64 x 256.  A step is three products with a barrier
// between: S and P in 16 x 16 blocks (of 32 x 32 most waves would have none), X in
// 32 x 32 ones (half of the LDS reads).  Bound by LDS traffic and the waves'
// latency: 8 of 64 x 256 in 5 steps 36 us (84 with a launch for each product).
constexpr int kNsLds = 163840;
struct NsFused {
  const float* g;
  float* m;
  float mu;
  int nesterov, r, c, M, N, mp, np, steps;
  int vec;  // rows of g and m are read as float4
  float* f;
  float le, decay;
  int weights;
};
// LDS bytes of X (both ways) and S.
__host__ __device__ constexpr int64_t ns_fused_bytes(int64_t mp, int64_t np) {
  return 4 * (np * (mp + 1) + mp * (np + 1) + mp * (mp + 1));
}
__global__ __launch_bounds__(1024) void ns_fused_kernel(NsFused a) {
  extern __shared__ __attribute__((aligned(16))) char ns_lds[];
  __shared__ double red[16];
  constexpr int kW = 16, kSymBlocks = 2, kBlocks = 2;  // waves, blocks of S and of X a wave (ns_fused_fits)
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int mp = a.mp, np = a.np;
  int rm = mp + 1, rn = np + 1;  // rows between octets
  const int pg = np * rm, pu = mp * rn, ps = mp * rm;        // to the other piece, halves
  _Float16* gram = reinterpret_cast<_Float16*>(ns_lds);  // [2][np / 8][rm][8]
  _Float16* upd = gram + 2 * pg;                         // [2][mp / 8][rn][8]
  _Float16* sym = upd + 2 * pu;                          // [2][mp / 8][rm][8]
  const int elems = a.r * a.c;
  const int64_t base = (int64_t)blockIdx.x * elems;
  const float* __restrict__ g = a.g + base;
  float* __restrict__ m = a.m ? a.m + base : nullptr;
  const bool tall = a.r > a.c;
  double sq = 0.;
  for (int i0 = t; i0 < elems; i0 += 8 * 64 * kW) {
    float u[8], mm[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int i = min(i0 + j * 64 * kW, elems - 1);
      u[j] = g[i];
      if (m) mm[j] = m[i];
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int i = i0 + j * 64 * kW;
      if (i >= elems) break;
      if (m) {
        mm[j] = a.mu * mm[j] + u[j];
        m[i] = mm[j];
        u[j] = update_of(u[j], mm[j], a.mu, a.nesterov);
      }
      sq += (double)u[j] * u[j];
    }
  }
  sq = wave_sum(sq);
  if (lane == 0) red[wave] = sq;
  for (int i = t; i < (pg + pu) / 4; i += 64 * kW) reinterpret_cast<uintx4*>(gram)[i] = uintx4{0u, 0u, 0u, 0u};
  __syncthreads();  // (m is written: other threads read it below)
  sq = wave_sum(lane < kW ? red[lane] : 0.);
  const double norm = sqrt(sq), by = sq < __builtin_inf() ? 1. / (norm + kNsEps) : __builtin_nan("");
  const int e0 = ns_exponent(norm * by);
  const double up = ldexp(by * kUpX, e0);
  // X into an operand a chunk at a time: eight k of a row
  auto chunk = [&](_Float16* to, int rows, int piece, int ks, int row_step, int k_step, int row, int o) {
    float v[8];
    if (a.vec && k_step == 1) {  // (uniform; rows of a multiple of 4)
#pragma unroll
      for (int u = 0; u < 8; u += 4) {
        const int at = row * row_step + min(8 * o + u, ks - 4);
        float4 f = *reinterpret_cast<const float4*>(g + at);
        if (m) {
          const float4 h = *reinterpret_cast<const float4*>(m + at);
          f = make_float4(update_of(f.x, h.x, a.mu, a.nesterov), update_of(f.y, h.y, a.mu, a.nesterov),
                          update_of(f.z, h.z, a.mu, a.nesterov), update_of(f.w, h.w, a.mu, a.nesterov));
        }
        v[u] = f.x; v[u + 1] = f.y; v[u + 2] = f.z; v[u + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int at = row * row_step + min(8 * o + u, ks - 1) * k_step;
        v[u] = g[at];
        if (m) v[u] = update_of(v[u], m[at], a.mu, a.nesterov);
      }
    }
    half8 h, l;
#pragma unroll
    for (int u = 0; u < 8; u++) {
      _Float16 hh, ll;
      split2_far(8 * o + u < ks ? (float)(v[u] * up) : 0.f, hh, ll);
      h[u] = hh;
      l[u] = ll;
    }
    _Float16* p = to + (o * rows + row) * 8;
    *reinterpret_cast<half8*>(p) = h;
    *reinterpret_cast<half8*>(p + piece) = l;
  };
  // a wave takes 64 rows of an octet where rows lie next to each other in g, else 8
  // rows of 8 octets
  auto chunks = [&](_Float16* to, int rows, int piece, int nrows, int ks, int row_step, int k_step) {
    const int octs = (ks + 7) >> 3;
    if (k_step == 1) {
      const int across = (octs + 7) >> 3;
      for (int b = wave; b < across * ((nrows + 7) >> 3); b += kW) {
        const int o = b % across * 8 + (lane >> 3), row = b / across * 8 + (lane & 7);
        if (o < octs && row < nrows) chunk(to, rows, piece, ks, row_step, k_step, row, o);
      }
    } else {
      const int across = (nrows + 63) >> 6;
      for (int b = wave; b < across * octs; b += kW) {
        const int row = b % across * 64 + lane;
        if (row < nrows) chunk(to, rows, piece, ks, row_step, k_step, row, b / across);
      }
    }
  };
  const int si1 = tall ? 1 : a.c, sj1 = tall ? a.c : 1;  // X (i, j) is g[i si1 + j sj1]
  chunks(gram, rm, pg, a.M, a.N, si1, sj1);
  chunks(upd, rn, pu, a.N, a.M, sj1, si1);
  __syncthreads();
  // 16 x 16 block (bi, bj) of A A^T, A of rows rm, over `steps` of 32: lane (l16, kq)
  // holds octet kq of a step, then column l16 of rows 4 kq ..
  int l16 = lane & 15, kq = lane >> 4;
  auto block16 = [&](const _Float16* A, int piece, int bi, int bj, int steps) {
    const half8* pa = reinterpret_cast<const half8*>(A) + kq * rm + bi * 16 + l16;
    const half8* pb = reinterpret_cast<const half8*>(A) + kq * rm + bj * 16 + l16;
    piece /= 8;
    floatx4 hi = {0.f, 0.f, 0.f, 0.f}, lo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < steps; s++) {
      const half8 a0 = pa[4 * s * rm], a1 = pa[4 * s * rm + piece], b0 = pb[4 * s * rm], b1 = pb[4 * s * rm + piece];
      hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b0, hi, 0, 0, 0);
      lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b0, lo, 0, 0, 0);
      lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b1, lo, 0, 0, 0);
    }
    return hi + kLowDown * lo;
  };
  // its values into S's or P's operand, both ways unless on the diagonal
  auto put16 = [&](const floatx4& x, int bi, int bj) {
    const int col = bj * 16 + l16, row = bi * 16 + 4 * kq;
    half4 h, l;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      _Float16 hh, ll;
      split2_far(x[u], hh, ll);
      h[u] = hh;
      l[u] = ll;
      if (bi != bj) {
        _Float16* p = sym + ((col >> 3) * rm + row + u) * 8 + (col & 7);
        p[0] = hh;
        p[ps] = ll;
      }
    }
    _Float16* p = sym + ((row >> 3) * rm + col) * 8 + (row & 7);
    *reinterpret_cast<half4*>(p) = h;
    *reinterpret_cast<half4*>(p + ps) = l;
  };
  const int mb = mp / 16, tri = mb * (mb + 1) / 2;
  int si[kSymBlocks], sj[kSymBlocks];
#pragma unroll
  for (int q = 0; q < kSymBlocks; q++) ns_tile<true>(wave + kW * q, 0, si[q], sj[q]);
  const int xb = mp / 32, nb = np / 32;
  int l32 = lane & 31, kh = lane >> 5;
  for (int step = 0; step < a.steps; step++) {
    // (keeps the compiler from holding every address of a step in registers)
    asm volatile("" : "+s"(rm), "+s"(rn), "+v"(l16), "+v"(kq), "+v"(l32), "+v"(kh));
    const int ex = max(0, e0 - 2 * step);
    floatx4 S[kSymBlocks];
#pragma unroll
    for (int q = 0; q < kSymBlocks; q++)
      if (wave + kW * q < tri) {
        __builtin_amdgcn_sched_barrier(0);  // (a block at a time: registers)
        S[q] = block16(gram, pg, si[q], sj[q], np / 32);
#pragma unroll
        for (int v = 0; v < 4; v++) {
          // (as P's square sees it: a rounding of S in one term alone would reach P four times as large)
          _Float16 h, l;
          split2_far(S[q][v] * (kUpS / (kUpX * kUpX)), h, l);
          S[q][v] = join2_far(h, l);
        }
        put16(S[q], si[q], sj[q]);
      }
    __syncthreads();
    const float bs = ldexpf(kNsB * kUpP / kUpS, -2 * ex), bss = ldexpf(kNsC * kUpP / (kUpS * kUpS), -4 * ex);
#pragma unroll
    for (int q = 0; q < kSymBlocks; q++)
      if (wave + kW * q < tri) {
        __builtin_amdgcn_sched_barrier(0);
        const floatx4 x = block16(sym, ps, si[q], sj[q], mp / 32);
        const int col = sj[q] * 16 + l16, row = si[q] * 16 + 4 * kq;
#pragma unroll
        for (int v = 0; v < 4; v++)
          S[q][v] = x[v] * bss + (row + v == col && col < a.M ? kNsA * kUpP : 0.f) + bs * S[q][v];
      }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kSymBlocks; q++)
      if (wave + kW * q < tri) put16(S[q], si[q], sj[q]);
    __syncthreads();
    // X: 32 x 32 block (b / nb, b % nb) of P X over the 16-steps of m
    floatx16 x[kBlocks], low;
#pragma unroll
    for (int q = 0; q < kBlocks; q++) {
      const int b = wave + kW * q;
      if (b < xb * nb) {
        __builtin_amdgcn_sched_barrier(0);
        const half8* pa = reinterpret_cast<const half8*>(sym) + kh * rm + b / nb * 32 + l32;
        const half8* pb = reinterpret_cast<const half8*>(upd) + kh * rn + b % nb * 32 + l32;
#pragma unroll
        for (int v = 0; v < 16; v++) x[q][v] = low[v] = 0.f;
#pragma unroll 4
        for (int s = 0; s < mp / 16; s++) {
          const half8 a0 = pa[2 * s * rm], a1 = pa[2 * s * rm + ps / 8], b0 = pb[2 * s * rn], b1 = pb[2 * s * rn + pu / 8];
          low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1, b0, low, 0, 0, 0);
          x[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, b0, x[q], 0, 0, 0);
          low = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, b1, low, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; v++) x[q][v] += kLowDown * low[v];
      }
    }
    const bool last = step + 1 == a.steps;
    const float xs = last ? 1.f / (kUpX * kUpP) : ldexpf(1.f / kUpP, max(0, ex - 2) - ex);
    if (!last) __syncthreads();
#pragma unroll
    for (int q = 0; q < kBlocks; q++) {
      const int b = wave + kW * q;
      if (b >= xb * nb) continue;
      __builtin_amdgcn_sched_barrier(0);
      const int row0 = b / nb * 32 + 4 * kh, col = b % nb * 32 + l32;
      if (last) {
#pragma unroll
        for (int v = 0; v < 16; v++) {
          const int i = row0 + 8 * (v >> 2) + (v & 3);
          if (i >= a.M || col >= a.N) continue;
          float* p = a.f + base + (tall ? col * a.c + i : i * a.c + col);
          const float y = ldexpf(x[q][v] * xs, -ex);
          *p = a.weights ? *p - a.le * y - a.decay * *p : y;
        }
        continue;
      }
#pragma unroll
      for (int w = 0; w < 4; w++) {
        __builtin_amdgcn_sched_barrier(0);
        half4 h, l;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          _Float16 hh, ll;
          split2_far(x[q][4 * w + u] * xs, hh, ll);
          h[u] = hh;
          l[u] = ll;
          _Float16* p = gram + ((col >> 3) * rm + row0 + 8 * w + u) * 8 + (col & 7);
          p[0] = hh;
          p[pg] = ll;
        }
        _Float16* p = upd + ((row0 + 8 * w) / 8 * rn + col) * 8 + (row0 & 7);
        *reinterpret_cast<half4*>(p) = h;
        *reinterpret_cast<half4*>(p + pu) = l;
      }
    }
    if (!last) __syncthreads();
  }
}

// Whether a matrix fits ns_fused_kernel: its LDS, and its waves' blocks (which the LDS bounds: m is at
// most 96, 21 blocks of S on 16 waves, and m N at most 20480, 20 blocks of X).
bool ns_fused_fits(int64_t m, int64_t N) {
  const int64_t mp = (m + 31) / 32 * 32, np = (N + 31) / 32 * 32;
  return np <= 4096 && ns_fused_bytes(mp, np) + 128 <= kNsLds;
}

constexpr int64_t round64(int64_t n) { return (n + 63) / 64 * 64; }

struct NsSizes {
  int64_t m, N, mp, np, gram, upd, sym;  // halves of a matrix's operands
  NsSizes(int64_t r, int64_t c) {
    m = std::min(r, c);
    N = std::max(r, c);
    mp = (m + 31) / 32 * 32;
    np = (N + 31) / 32 * 32;
    gram = 2 * np * m;
    upd = 2 * mp * N;
    sym = 2 * mp * m;
  }
};

// Tiles of `side` of n results [ra, rb] (sym: their lower triangles).
int64_t tiles_of(int64_t n, int64_t ra, int64_t rb, int64_t side, bool sym) {
  const int64_t tm = ceil_div(ra, side);
  return n * (sym ? tm * (tm + 1) / 2 : tm * ceil_div(rb, side));
}

// Tests' choice of the tiles' side, also where one workgroup could take a matrix; 0: the rule.
std::atomic<int> g_tile_side{0};

// The side of a product's tiles, by the estimated us of each kernel from its
// workgroups and K, as measured on 512 x 512, 4 of 512 x 512, 512 x 2048, 8192 x
// 512, 2000 x 1500, 8 and 64 of 1024 x 1024: 32 x 32 outputs a workgroup 4 + 0.0031
// K, or 2.2e-5 K each once they fill the chip; 64 x 64 6 + 0.0075 K, or 6.5e-5 K;
// 128 x 128 9 + 0.0215 K on a CU by itself, 1.3 times as much for each of several;
// 256 x 256 8 + 0.107 K.  X of 64 of 1024 x 1024: 1700, 850, 462, 446 us; of 512 x
// 2048: 20, 11, 21, 48; S of 512 x 512: 6, 9.5, 18, 44.
int tile_side(int64_t n, int64_t ra, int64_t rb, int64_t K, bool sym) {
  if (const int side = g_tile_side.load(std::memory_order_relaxed)) return side;
  const double k = (double)K;
  const double t32 = (double)tiles_of(n, ra, rb, 32, sym), t64 = (double)tiles_of(n, ra, rb, 64, sym);
  const int64_t n128 = ceil_div(tiles_of(n, ra, rb, 128, sym), 256), n256 = ceil_div(tiles_of(n, ra, rb, 256, sym), 256);
  // (32 x 32 at most 2^22 workgroups: a launch takes fewer than 2^32 threads)
  const double us[4] = {t32 > 0x1p22 ? 1e30 : std::max(4 + 0.0031 * k, 3 + 2.2e-5 * k * t32),
                        std::max(6 + 0.0075 * k, 3 + 6.5e-5 * k * t64),
                        9 + 0.0215 * k * (n128 == 1 ? 1. : 1.3 * n128), 8 + 0.107 * k * n256};
  return 32 << (std::min_element(us, us + 4) - us);
}

template <int MODE>
int launch_product(NsArgs& g, hipStream_t s) {
  constexpr bool kSym = MODE == kGram || MODE == kPoly;
  const int side = tile_side(g.n, g.ra, g.rb, g.k, kSym);
  g.tiles_m = (int)ceil_div(g.ra, side);
  g.tiles_n = (int)ceil_div(g.rb, side);
  g.tiles = (int)tiles_of(1, g.ra, g.rb, side, kSym);
  const dim3 grid((unsigned)((int64_t)g.tiles * g.n));
  if (side == 32) hipLaunchKernelGGL((ns_few_kernel<MODE>), grid, dim3(512), 0, s, g);
  else if (side == 64) hipLaunchKernelGGL((ns_mid_kernel<MODE>), grid, dim3(512), 0, s, g);
  else if (side == 128) hipLaunchKernelGGL((ns_gemm_kernel<MODE, 2, 2, 2, 2, 32>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((ns_gemm_kernel<MODE, 2, 4, 4, 2, 16>), grid, dim3(512), 0, s, g);
  NSH_LAUNCHED();
  return 0;
}

}  // namespace

void set_ns_tile_side(int side) {
  g_tile_side.store(side == 32 || side == 64 || side == 128 || side == 256 ? side : 0, std::memory_order_relaxed);
}

// 0: one workgroup a matrix; else the side of the tiles of the products S (0), P (1), X (2) and the last (3).
int ns_tile_side(int product, int64_t n, int64_t r, int64_t c) {
  const NsSizes z(r, c);
  if (!g_tile_side.load(std::memory_order_relaxed) && ns_fused_fits(z.m, z.N)) return 0;
  if (product < 2) return tile_side(n, z.m, z.m, product ? z.mp : z.np, true);
  return product == 3 && r > c ? tile_side(n, z.N, z.m, z.mp, false) : tile_side(n, z.m, z.N, z.mp, false);
}

// the norms' partial sums; their exponents; X as the Gram's operand, twice as the update's; S and P
size_t newton_schulz_bytes(int64_t n, int64_t r, int64_t c) {
  const NsSizes z(r, c);
  return (size_t)round64(n) * 4 + (size_t)n * (kNormParts * 8 + 2 * (size_t)(z.gram + 2 * z.upd + 2 * z.sym));
}

int launch_newton_schulz(const float* g, float* q, const MuonNs* step, int64_t n, int64_t r, int64_t c, int steps,
                         void* workspace, hipStream_t s) {
  const NsSizes z(r, c);
  const int64_t elems = r * c;
  if (n <= 0 || elems <= 0) return 0;
  double* part = static_cast<double*>(workspace);
  int* ex = reinterpret_cast<int*>(part + n * kNormParts);
  _Float16* gram = reinterpret_cast<_Float16*>(ex + round64(n));
  _Float16* upd = gram + n * z.gram;
  _Float16* upd2 = upd + n * z.upd;
  _Float16* S = upd2 + n * z.upd;
  _Float16* P = S + n * z.sym;
  const int parts = (int)std::min<int64_t>(kNormParts, ceil_div(elems, 2048));
  float* mom = step ? step->m : nullptr;
  const float mu = step ? step->mu : 0.f;
  const int nesterov = step ? step->nesterov : 0;
  if (steps > 0 && ns_tile_side(0, n, r, c) == 0) {
    NsFused f{};
    f.g = g; f.m = mom; f.mu = mu; f.nesterov = nesterov;
    f.r = (int)r; f.c = (int)c; f.M = (int)z.m; f.N = (int)z.N;
    f.mp = (f.M + 31) / 32 * 32;
    f.np = (f.N + 31) / 32 * 32;
    f.steps = steps;
    f.f = step ? step->w : q;
    f.weights = step != nullptr;
    f.le = step ? step->le : 0.f;
    f.decay = step ? step->decay : 0.f;
    f.vec = c % 4 == 0 && ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(mom)) & 15) == 0;
    const unsigned lds = (unsigned)ns_fused_bytes(f.mp, f.np);
    hipLaunchKernelGGL(ns_fused_kernel, dim3((unsigned)n), dim3(1024), lds, s, f);
    NSH_LAUNCHED();
    return 0;
  }
  hipLaunchKernelGGL(ns_norm_kernel, dim3(parts, (unsigned)n), dim3(256), 0, s, g, mom, mu, nesterov, elems, part);
  NSH_LAUNCHED();
  if (steps == 0) {
    hipLaunchKernelGGL(ns_normalise_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(elems, 1024), 4096), (unsigned)n),
                       dim3(256), 0, s, g, mom, mu, nesterov, elems, parts, part, q, step ? step->w : nullptr,
                       step ? step->le : 0.f, step ? step->decay : 0.f);
    NSH_LAUNCHED();
    return 0;
  }
  NsStart a;
  a.g = g; a.m = mom; a.mu = mu; a.nesterov = nesterov;
  a.r = r; a.c = c;
  a.parts = parts; a.part = part; a.ex = ex;
  a.gram = gram; a.upd = upd;
  a.M = z.m; a.N = z.N; a.mp = z.mp; a.np = z.np;
  a.tiles_n = (int)ceil_div(z.np, 64);
  hipLaunchKernelGGL(ns_start_kernel, dim3((unsigned)(ceil_div(z.mp, 64) * a.tiles_n), (unsigned)n), dim3(256), 0, s, a);
  NSH_LAUNCHED();
  for (int k = 0; k < steps; k++) {
    NsArgs p{};
    p.n = (int)n;
    p.ex = ex; p.step = k;
    p.A = p.B = gram;
    p.ra = p.rb = z.m; p.k = z.np;
    p.sA = p.sB = z.gram;
    p.out = S; p.sOut = z.sym;
    p.kout = p.kout2 = z.mp;
    if (launch_product<kGram>(p, s) != 0) return -1;
    p.A = p.B = S; p.k = z.mp;
    p.sA = p.sB = z.sym;
    p.S = S; p.out = P;
    if (launch_product<kPoly>(p, s) != 0) return -1;
    const bool last = k + 1 == steps, tall = last && r > c;
    p.A = tall ? upd : P; p.sA = tall ? z.upd : z.sym; p.ra = tall ? z.N : z.m;
    p.B = tall ? P : upd; p.sB = tall ? z.sym : z.upd; p.rb = tall ? z.m : z.N;
    p.k = z.mp;
    if (last) {
      p.f = step ? step->w : q;
      p.weights = step != nullptr;
      p.le = step ? step->le : 0.f;
      p.decay = step ? step->decay : 0.f;
      return launch_product<kLast>(p, s);
    }
    p.out = gram; p.sOut = z.gram; p.kout2 = z.np;
    p.out2 = upd2; p.sOut2 = z.upd; p.kout = z.mp;
    if (launch_product<kUpdate>(p, s) != 0) return -1;
    std::swap(upd, upd2);
  }
  return 0;
}

}  // namespace nship
