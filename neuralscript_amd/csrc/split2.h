// Products of operands held as two fp16 pieces: v = h + l, h = fp16(v), l =
// fp16(v - h), 22 bits of v (23 with l's sign) while v is at least 2^-18 of
// fp16's largest value; below, an absolute 2^-25 (l's last place).  A product a b
// is accumulated in fp32 from ah bh + ah bl + al bh: three fp16 MFMAs a step of
// 16 (split3.h: six bf16 ones for the full 24 bits).  What that drops is at most
// 2^-23 of an operand (fp32: 2^-24) and 2^-22 of a product, 2^-23.6 of it
// rounding at random, where fp32 sums of 1024 terms lose 2^-20 and more.  The
// caller scales operands by powers of two so that they stay in fp16's range.
//
// An operand with rows R and contraction length K is stored as [piece][K / 8][R]
// [8]: the 16-byte chunk of 8 consecutive k of one row is what one lane of an
// MFMA takes, and a slab of a tile is contiguous runs of chunks, copied to LDS as
// they lie and read back conflict-free.
#pragma once
#include <type_traits>

#include "common.h"

namespace nship {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

// The low piece times 2^11: it then lies in the high one's range, and v keeps its
// 22 bits down to fp16's smallest normal, 2^-30 of its largest; below, an absolute
// 2^-36.  For operands whose rows lie far apart under one scale (newton.hip, moe_split.hip).
constexpr float kLowUp = 0x1p11f, kLowDown = 0x1p-11f;
__device__ __forceinline__ void split2_far(float v, _Float16& h, _Float16& l) {
  h = (_Float16)v;
  l = (_Float16)((v - (float)h) * kLowUp);
}
__device__ __forceinline__ float join2_far(_Float16 h, _Float16 l) { return (float)h + kLowDown * (float)l; }

// Workgroup b of T -> a linear index such that each of the 8 XCDs (ids are dealt
// to them in turn) owns one contiguous run; a bijection on [0, T).
__device__ __forceinline__ int split2_xcd_linear(int b, int T) {
  const int per = T >> 3, rem = T & 7, x = b & 7, i = b >> 3;
  return x * per + (x < rem ? x : rem) + i;
}

// One operand of a tile: chunks of `rows` rows, `piece` chunks to the other
// piece, the tile's rows from `first`, `last` the last that may be read (rows
// past it read that one: their results are not used).
struct Split2Operand {
  const uintx4* p;
  int64_t rows, piece, first, last;
};

// A tile of C = A B^T by WM x WN waves of TM x TN blocks of 32 x 32, in slabs of
// KS, double buffered in LDS, two slabs of loads in flight.  Accumulator v of
// lane (l32, kh) in a block: row 8 (v / 4) + 4 kh + v % 4, column l32.
//
// FAR: the low pieces are held times 2^11 (split2_far), so the products with one
// are summed apart: in accumulators of their own where these fit beside the others
// (up to 2 x 2 blocks a wave), else in a sweep over K of its own before that of the
// high pieces.
//
// Bound by the matrix cores and the power they draw: 64 products of 1024^3 on 256 x
// 256 tiles of eight 128 x 64 waves run at 308 TFLOP/s, 924 of fp16, with the sweep
// apart (317 and 950 in one sweep; the vendor's fp16 product: 1110).
template <int WM, int WN, int TM, int TN, int KS, bool FAR = false>
struct Split2Tile {
  static constexpr int NT = 64 * WM * WN, RA = 32 * WM * TM, RB = 32 * WN * TN, OCT = KS / 8;
  static constexpr int kBuf = 2 * OCT * (RA + RB) * 16, kLds = 2 * kBuf;

  // Slabs of PIECES pieces (the high one, or both) of O octets, nk of them (at least
  // one); `use` takes the pieces of a step of 16.  Ends with a barrier.
  template <int PIECES, int O, typename Use>
  __device__ __forceinline__ static void sweep(const Split2Operand& A, const Split2Operand& B, int nk,
                                               char* __restrict__ smem, Use use) {
    constexpr int CA = PIECES * O * RA / NT, CB = PIECES * O * RB / NT;  // chunks a thread
    static_assert(CA * NT == PIECES * O * RA && CB * NT == PIECES * O * RB, "the chunks divide evenly");
    static_assert(PIECES * O == 2 * OCT, "a slab fills its buffer");
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int wm = wave / WN, wn = wave % WN, l32 = lane & 31, kh = lane >> 5;
    // chunk i of thread t: (piece, octet, row), row fastest
    const uintx4* pa[CA];
    const uintx4* pb[CB];
#pragma unroll
    for (int i = 0; i < CA; i++) {
      const int c = t + NT * i, row = c % RA, o = c / RA % O, p = c / RA / O;
      pa[i] = A.p + p * A.piece + o * A.rows + min(A.first + row, A.last);
    }
#pragma unroll
    for (int i = 0; i < CB; i++) {
      const int c = t + NT * i, row = c % RB, o = c / RB % O, p = c / RB / O;
      pb[i] = B.p + p * B.piece + o * B.rows + min(B.first + row, B.last);
    }
    const int64_t stepa = O * A.rows, stepb = O * B.rows;
    uintx4 va[2][CA], vb[2][CB];
    int next = 0;  // slab to load; past the last it is loaded again
    auto load = [&](auto z) {
      constexpr int Z = decltype(z)::value;
#pragma unroll
      for (int i = 0; i < CA; i++) va[Z][i] = *pa[i];
#pragma unroll
      for (int i = 0; i < CB; i++) vb[Z][i] = *pb[i];
      const bool more = ++next < nk;
#pragma unroll
      for (int i = 0; i < CA; i++) pa[i] += more ? stepa : 0;
#pragma unroll
      for (int i = 0; i < CB; i++) pb[i] += more ? stepb : 0;
    };
    auto store = [&](auto z, char* to) {
      constexpr int Z = decltype(z)::value;
#pragma unroll
      for (int i = 0; i < CA; i++) *reinterpret_cast<uintx4*>(to + (t + NT * i) * 16) = va[Z][i];
#pragma unroll
      for (int i = 0; i < CB; i++) *reinterpret_cast<uintx4*>(to + 2 * OCT * RA * 16 + (t + NT * i) * 16) = vb[Z][i];
    };
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    load(Even{});
    load(Odd{});
    store(Even{}, smem);
    load(Even{});
    __syncthreads();
    auto slab = [&](int kt, auto z) {
      const char* as = smem + (kt & 1) * kBuf + (kh * RA + wm * TM * 32 + l32) * 16;
      const char* bs = smem + (kt & 1) * kBuf + 2 * OCT * RA * 16 + (kh * RB + wn * TN * 32 + l32) * 16;
#pragma unroll
      for (int s = 0; s < O / 2; s++) {
        half8 fa[TM][PIECES], fb[TN][PIECES];
#pragma unroll
        for (int c = 0; c < TN; c++)
#pragma unroll
          for (int p = 0; p < PIECES; p++)
            fb[c][p] = *reinterpret_cast<const half8*>(bs + ((p * O + 2 * s) * RB + c * 32) * 16);
#pragma unroll
        for (int r = 0; r < TM; r++)
#pragma unroll
          for (int p = 0; p < PIECES; p++)
            fa[r][p] = *reinterpret_cast<const half8*>(as + ((p * O + 2 * s) * RA + r * 32) * 16);
        use(fa, fb);
      }
      store(z, smem + ((kt + 1) & 1) * kBuf);
      load(z);
      __syncthreads();
    };
    for (int kt = 0; kt < nk; kt += 2) {
      slab(kt, Odd{});
      if (kt + 1 < nk) slab(kt + 1, Even{});
    }
  }

  // acc[r][c] += piece p of a row times piece q of b, over all blocks
  template <int PIECES>
  __device__ __forceinline__ static void products(const half8 (&fa)[TM][PIECES], const half8 (&fb)[TN][PIECES], int r,
                                                  int p, int q, floatx16 (&acc)[TM][TN]) {
#pragma unroll
    for (int c = 0; c < TN; c++) acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[r][p], fb[c][q], acc[r][c], 0, 0, 0);
  }

  // nk slabs of KS (FAR with more than 2 x 2 blocks: an even number)
  __device__ __forceinline__ static void run(const Split2Operand& A, const Split2Operand& B, int nk,
                                             char* __restrict__ smem, floatx16 (&acc)[TM][TN]) {
    auto each = [](auto f) {
#pragma unroll
      for (int r = 0; r < TM; r++)
#pragma unroll
        for (int c = 0; c < TN; c++)
#pragma unroll
          for (int v = 0; v < 16; v++) f(r, c, v);
    };
    each([&](int r, int c, int v) { acc[r][c][v] = 0.f; });
    if constexpr (!FAR) {
      sweep<2, OCT>(A, B, nk, smem, [&](const half8 (&fa)[TM][2], const half8 (&fb)[TN][2]) {
#pragma unroll
        for (int r = 0; r < TM; r++) {
          products(fa, fb, r, 1, 0, acc);
          products(fa, fb, r, 0, 1, acc);
          products(fa, fb, r, 0, 0, acc);
        }
      });
    } else if constexpr (TM * TN <= 4) {
      floatx16 low[TM][TN];
      each([&](int r, int c, int v) { low[r][c][v] = 0.f; });
      sweep<2, OCT>(A, B, nk, smem, [&](const half8 (&fa)[TM][2], const half8 (&fb)[TN][2]) {
#pragma unroll
        for (int r = 0; r < TM; r++) {
          products(fa, fb, r, 1, 0, low);
          products(fa, fb, r, 0, 0, acc);
          products(fa, fb, r, 0, 1, low);
        }
      });
      each([&](int r, int c, int v) { acc[r][c][v] += kLowDown * low[r][c][v]; });
    } else {
      sweep<2, OCT>(A, B, nk, smem, [&](const half8 (&fa)[TM][2], const half8 (&fb)[TN][2]) {
#pragma unroll
        for (int r = 0; r < TM; r++) {
          products(fa, fb, r, 1, 0, acc);
          products(fa, fb, r, 0, 1, acc);
        }
      });
      each([&](int r, int c, int v) { acc[r][c][v] *= kLowDown; });
      sweep<1, 2 * OCT>(A, B, nk / 2, smem, [&](const half8 (&fa)[TM][1], const half8 (&fb)[TN][1]) {
#pragma unroll
        for (int r = 0; r < TM; r++) products(fa, fb, r, 0, 0, acc);
      });
    }
  }
};

}  // namespace nship
