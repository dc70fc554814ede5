// The experts' products (moe_topk.hip) of a small layer: both products of 32 sorted
// slots in one workgroup, the hidden rows between them in LDS.
//
//   forward    u = x_rows W1[e], o = weight (act(u) W2[e])
//   backward   dh = dy_rows W2[e]^T, dweight = act(u) . dh, du = weight act'(u) dh,
//              o = du W1[e]^T
//
// A small layer's products are a few us of matrix instructions, and the grouped
// products that serve larger ones take 15 to 30 us each for their launch, their 128
// rows' staging and their epilogue on few workgroups; here two of them, the rows'
// pass between them and the gathering of the sorted rows are one launch.  fp32
// matrix instructions: the weights come straight from the L2 into registers, each
// value once a workgroup, with nothing to split or to stage.
#include <algorithm>

#include "common.h"
#include "kernels.h"
#include "moe_act.h"
#include "split2.h"

namespace nship {
namespace {

constexpr int kRows = 32, kWaves = 8, kThreads = 64 * kWaves;
constexpr int kMaxD = 256, kMaxH = 512;  // (LDS: 32 rows of both and the waves' sums, below 160 KB)

struct SmallArgs {
  const float* in;      // x, or dy [T, D]
  const float* W1;      // [E, D, H]
  const float* W2;      // [E, H, D]
  const float* weight;  // [slot]
  const int *seg, *tiles, *ntiles, *perm, *tok;
  float* pre;           // [pos, H]: the forward writes it (or null), the backward reads it
  float* slots;         // [slot, D] (backward: or null)
  const float* x;       // backward: x, and the rows that the weights' gradients take,
  float *dh, *hw;       // du, weight act(u) [pos, H],
  float *xs, *dys;      // x, dy [pos, D]; null: not wanted
  float* dweight;       // [slot] or null
  int D, H, act;
};

__host__ __device__ constexpr int round8(int n) { return (n + 7) / 8 * 8; }
// Floats between LDS rows: 4 times an odd number, so that 16 rows' float4s hit all banks.
__host__ __device__ constexpr int pitch_of(int n) { return round8(n) + 4; }
// Floats of the first region: the input rows, then the waves' partial sums.
__host__ __device__ constexpr int first_floats(int D) {
  return kRows * pitch_of(D) > kWaves * 1024 ? kRows * pitch_of(D) : kWaves * 1024;
}

// Column block `col` (a lane's column; past ncols: a copy of the last) of rows W
// over k0 .. k1 (multiples of 8) of K (a multiple of 4).  W [K, ncols], or turned
// [ncols, K].  a: the LDS row of the lane's row.  A lane's half kh takes the k 4 kh
// .. 4 kh + 3 of every octet on both sides.
template <bool TURNED>
__device__ __forceinline__ floatx16 block_product(const float* a, const float* __restrict__ W, int ncols, int K,
                                                  int col, int kh, int k0, int k1) {
  floatx16 acc;
#pragma unroll
  for (int v = 0; v < 16; v++) acc[v] = 0.f;
  const int c = min(col, ncols - 1);
  const float* __restrict__ p = TURNED ? W + (int64_t)c * K : W + c;
  for (int kk = k0; kk < k1; kk += 64) {
    float b[8][4];  // (64 steps of K in flight: a round trip to the L2 is longer than their products)
#pragma unroll
    for (int o = 0; o < 8; o++) {
      const int from = min(kk + 8 * o + 4 * kh, K - 4);
      if constexpr (TURNED) {
        const float4 f = *reinterpret_cast<const float4*>(p + from);
        b[o][0] = f.x; b[o][1] = f.y; b[o][2] = f.z; b[o][3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) b[o][j] = p[(int64_t)(from + j) * ncols];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int o = 0; o < 8; o++) {
      if (kk + 8 * o >= k1) break;  // (uniform)
      const int at = kk + 8 * o + 4 * kh;
      const bool in = at < K;
      const float4 x = *reinterpret_cast<const float4*>(a + at);
      const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(xs[j], in ? b[o][j] : 0.f, acc, 0, 0, 0);
    }
  }
  return acc;
}

template <bool BACK>
__global__ __launch_bounds__(kThreads) void small_kernel(SmallArgs g) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ int s_slot[kRows], s_tok[kRows];
  __shared__ float s_weight[kRows], s_dot[kWaves][kRows];
  const int entry = blockIdx.x >> 2;
  if (entry >= *g.ntiles) return;
  const int t = threadIdx.x, lane = t & 63, l32 = lane & 31, kh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int e = g.tiles[2 * entry];
  const int pos0 = g.seg[e] + g.tiles[2 * entry + 1] * 128 + (int)(blockIdx.x & 3) * kRows;
  const int rows = min(kRows, g.seg[e + 1] - pos0);
  if (rows <= 0) return;
  const int D = g.D, H = g.H, dp = pitch_of(D), hp = pitch_of(H);
  float* first = lds;
  float* hidden = lds + first_floats(D);
  if (t < kRows) {
    const int slot = t < rows ? g.perm[pos0 + t] : -1;
    s_slot[t] = slot;
    s_tok[t] = t < rows ? g.tok[pos0 + t] : -1;
    s_weight[t] = slot >= 0 ? g.weight[slot] : 0.f;
  }
  __syncthreads();
  // the input rows, zeros behind the last row and column
  const int d4 = round8(D) / 4;
  for (int i = t; i < kRows * d4; i += kThreads) {
    const int r = i / d4, c = (i - r * d4) * 4, tok = s_tok[r];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tok >= 0 && c < D) {
      v = *reinterpret_cast<const float4*>(g.in + (int64_t)tok * D + c);
      if (BACK && g.xs) {
        const int64_t to = (int64_t)(pos0 + r) * D + c;
        *reinterpret_cast<float4*>(g.dys + to) = v;
        *reinterpret_cast<float4*>(g.xs + to) = *reinterpret_cast<const float4*>(g.x + (int64_t)tok * D + c);
      }
    }
    *reinterpret_cast<float4*>(first + r * dp + c) = v;
  }
  __syncthreads();
  const int64_t DH = (int64_t)D * H;
  float dot[BACK ? 16 : 1];
#pragma unroll
  for (int v = 0; v < (BACK ? 16 : 1); v++) dot[v] = 0.f;
  for (int cb = wave; cb * 32 < H; cb += kWaves) {
    const int col = cb * 32 + l32;
    float u[16];
    if constexpr (BACK) {
#pragma unroll
      for (int v = 0; v < 16; v++) {
        const int r = 8 * (v >> 2) + 4 * kh + (v & 3);
        u[v] = g.pre[(int64_t)(pos0 + min(r, rows - 1)) * H + min(col, H - 1)];
      }
    }
    const float* W = (BACK ? g.W2 : g.W1) + (int64_t)e * DH;
    const floatx16 acc = block_product<BACK>(first + l32 * dp, W, H, D, col, kh, 0, round8(D));
#pragma unroll
    for (int v = 0; v < 16; v++) {
      const int r = 8 * (v >> 2) + 4 * kh + (v & 3);
      const bool in = r < rows && col < H;
      const int64_t at = (int64_t)(pos0 + r) * H + col;
      float h;
      if constexpr (BACK) {
        float a, slope;
        act_both(u[v], g.act, a, slope);
        const float w = s_weight[r];
        h = w * acc[v] * slope;
        dot[v] += in ? a * acc[v] : 0.f;
        if (in && g.xs) {
          g.dh[at] = h;
          g.hw[at] = w * a;
        }
      } else {
        if (in && g.pre) g.pre[at] = acc[v];
        h = act_apply(acc[v], g.act);
      }
      if (col < round8(H)) hidden[r * hp + col] = in ? h : 0.f;
    }
  }
  if constexpr (BACK) {
#pragma unroll
    for (int v = 0; v < 16; v++) {
      float d = row16_sum(dot[v]);
      d += __shfl_xor(d, 16, kWave);
      if (l32 == 0) s_dot[wave][8 * (v >> 2) + 4 * kh + (v & 3)] = d;
    }
  }
  __syncthreads();
  if (BACK && g.dweight && t < rows) {
    float d = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) d += s_dot[w][t];
    g.dweight[s_slot[t]] = d;
  }
  if (!g.slots) return;
  // the second product: column blocks times equal shares of K = H, one a wave
  const int nb = (D + 31) / 32, parts = kWaves / nb;
  const int share = round8((H + parts - 1) / parts);
  if (wave < nb * parts) {
    const int cb = wave % nb, k0 = min(round8(H), wave / nb * share), k1 = min(round8(H), k0 + share);
    const float* W = (BACK ? g.W1 : g.W2) + (int64_t)e * DH;
    const floatx16 acc = block_product<BACK>(hidden + l32 * hp, W, D, H, cb * 32 + l32, kh, k0, k1);
#pragma unroll
    for (int v = 0; v < 16; v++) first[wave * 1024 + (8 * (v >> 2) + 4 * kh + (v & 3)) * 32 + l32] = acc[v];
  }
  __syncthreads();
  for (int i = t; i < rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
    const float* p = first + c / 32 * 1024 + r * 32 + c % 32;
    float4 v = *reinterpret_cast<const float4*>(p);
    for (int s = 1; s < parts; s++) {
      const float4 w = *reinterpret_cast<const float4*>(p + s * nb * 1024);
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    const float w = BACK ? 1.f : s_weight[r];
    *reinterpret_cast<float4*>(g.slots + (int64_t)s_slot[r] * D + c) = make_float4(w * v.x, w * v.y, w * v.z, w * v.w);
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool BACK>
int launch(SmallArgs g, const SlotTables& t, const MoeShape& m, hipStream_t s) {
  g.seg = t.seg; g.tiles = t.tiles; g.ntiles = t.ntiles; g.perm = t.perm; g.tok = t.tok;
  g.D = (int)m.D; g.H = (int)m.H;
  const unsigned entries = (unsigned)(ceil_div(m.T * m.K, 128) + m.E);
  const unsigned lds = 4u * (unsigned)(first_floats(g.D) + kRows * pitch_of(g.H));
  hipLaunchKernelGGL(small_kernel<BACK>, dim3(4 * entries), dim3(kThreads), lds, s, g);
  NSH_LAUNCHED();
  return 0;
}

}  // namespace

// Up to N D H = 2^29, and any number of slots up to D = 64: a workgroup's 32 rows
// read the expert's weights from the L2, and the rate of fp32 matrix instructions is
// below that of three bf16 pieces.  Grouped products -> this, us, forward and
// training step, (tokens, choices, D, H, experts): 128, 4, 64, 256, 8: 56, 136 ->
// 27, 81; 1501: 59, 168 -> 29, 105; 32768: 186, 837 -> 168, 816.  1500, 2, 128, 256,
// 8: 64, 168 -> 33, 112; 16384: 104, 314 -> 94, 326; 65536: 239, 957 -> 278, 1108.
// 1500, 2, 256, 512, 8: 99, 274 -> 89, 253; 4000: 104, 308 -> 161, 421.
bool small_takes(const MoeShape& m, const void* x, const void* W1, const void* W2) {
  if (m.D > 64 && m.T * m.K * m.D * m.H > (1 << 29)) return false;
  return m.D <= kMaxD && m.H <= kMaxH && m.D % 4 == 0 && m.H % 4 == 0 && aligned(x) && aligned(W1) && aligned(W2);
}

int launch_small(const float* x, const float* weight, const float* W1, const float* W2, const SlotTables& t, float* pre,
                 float* slots, const MoeShape& m, int act, hipStream_t s) {
  SmallArgs g{};
  g.in = x; g.W1 = W1; g.W2 = W2; g.weight = weight;
  g.pre = pre; g.slots = slots; g.act = act;
  return launch<false>(g, t, m, s);
}

int launch_small_grad(const float* dy, const float* x, const float* weight, const float* W1, const float* W2,
                      const SlotTables& t, const float* pre, float* dh, float* hw, float* xs, float* dys, float* dweight,
                      float* slots, const MoeShape& m, int act, hipStream_t s) {
  SmallArgs g{};
  g.in = dy; g.x = x; g.W1 = W1; g.W2 = W2; g.weight = weight;
  g.pre = const_cast<float*>(pre); g.slots = slots; g.act = act;
  g.dh = dh; g.hw = hw; g.xs = xs; g.dys = dys; g.dweight = dweight;
  return launch<true>(g, t, m, s);
}

}  // namespace nship
