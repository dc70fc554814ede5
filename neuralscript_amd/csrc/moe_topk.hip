// Mixture of experts with K experts a token: routing from given logits and its
// gradient, and the experts' products forward and backward.
//
//   routing   s = softmax(l) or 1 / (1 + e^-l) over the live experts, c = s + bias;
//             the best groups stay, the K largest c of them are chosen, and
//             weight_k = scale s_k (/ sum_j s_j)
//   layer     y_t = sum_k weight_tk act(x_t W1[e]) W2[e],  e = idx_tk
//
// A (token, choice) pair t K + k is a slot.  Three ways through the layer, by its
// sizes alone:
//  * few slots an expert (few_slots): every workgroup lists its expert's slots and
//    streams the weights once for up to 8 of them, fp32 multiply-adds; bound by the
//    weights' bytes.
//  * many (split_takes, moe_split.hip): products of two fp16 pieces over operands
//    laid out for them; bound by the matrix cores.
//  * between: the slots are sorted by expert (stable, so every sum has one order).
//    A small layer's two products run in one kernel (small_takes, moe_small.hip),
//    bound by the latency of some ten launches; else gemm.hip's grouped products
//    (three bf16 pieces) run over the sorted rows, gathered and scattered as they
//    are, bound by the matrix cores.
// The slots of a token meet in a pass of their own, in the order of k.
#include <algorithm>

#include "common.h"
#include "kernels.h"
#include "moe_act.h"

namespace nship {
namespace {

constexpr double kNone = -__builtin_inf();

__device__ __forceinline__ double shfl_xor_f64(double v, int o) { return __shfl_xor(v, o, kWave); }

// The logit of expert e, -inf where the expert is not live.  Written without a
// branch on the lane: as `if (dead) x = -inf` hipcc 7.2 drops the assignment
// of every register but the first.
__device__ __forceinline__ float live_logit(const float* __restrict__ l, int e, int E,
                                            const uint8_t* __restrict__ active) {
  const bool in = e >= 0 && e < E;
  const int at = in ? e : 0;
  const float x = l[at];
  const int on = active ? active[at] : 1;  // (uniform)
  return (int)in & (int)(on != 0) & (int)(x > -__builtin_inff()) ? x : -__builtin_inff();  // (NaN > -inf is false)
}

// The larger value over the wave, the lower index on a tie.
__device__ __forceinline__ void wave_best(double& v, int& i) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double w = shfl_xor_f64(v, o);
    const int j = __shfl_xor(i, o, kWave);
    const bool take = w > v || (w == v && j < i);
    v = take ? w : v;
    i = take ? j : i;
  }
}

// One wave per token, expert v 64 + lane in register v.  The scores and what
// they are compared by are held in 64 bits: a choice is an integer, and two
// values 2^-24 apart, which 32 bits may order either way, turn up in every few
// thousand tokens.
template <int V>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
  __shared__ double by_expert[4][64 * V];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t tok = (int64_t)blockIdx.x * 4 + w;
  if (tok >= a.T) return;  // (uniform per wave; no barrier below)
  const float* __restrict__ l = a.logits + tok * a.E;
  double s[V], c[V];
  float x[V], mx = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < V; v++) {
    x[v] = live_logit(l, v * 64 + lane, a.E, a.active);
    mx = fmaxf(mx, x[v]);
  }
  mx = wave_max(mx);
  if (a.score == 0) {
    double sum = 0.;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const bool live = x[v] > -__builtin_inff();
      s[v] = !live ? 0. : x[v] == mx ? 1. : exp((double)x[v] - (double)mx);  // (a logit of +inf: 1)
      sum += s[v];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int v = 0; v < V; v++) s[v] = sum > 0. ? s[v] / sum : 0.;
  } else {
#pragma unroll
    for (int v = 0; v < V; v++) s[v] = x[v] > -__builtin_inff() ? 1. / (1. + exp(-(double)x[v])) : 0.;
  }
#pragma unroll
  for (int v = 0; v < V; v++) {
    const int e = v * 64 + lane;
    const double b = s[v] + (a.bias ? (double)a.bias[e < a.E ? e : 0] : 0.);
    c[v] = (int)(x[v] > -__builtin_inff()) & (int)(b > kNone) ? b : kNone;  // (a NaN bias: never chosen)
  }
  if (a.groups > 1) {
    const int per = a.E / a.groups;
    double* __restrict__ t = by_expert[w];
#pragma unroll
    for (int v = 0; v < V; v++) t[v * 64 + lane] = c[v];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    double one = kNone, two = kNone;
    if (lane < a.groups)
      for (int j = 0; j < per; j++) {
        const double b = t[lane * per + j];
        two = b > one ? one : b > two ? b : two;
        one = b > one ? b : one;
      }
    if (a.group_best == 2 && two > kNone) one += two;
    uint64_t keep = 0;
    for (int g = 0; g < a.top_groups; g++) {
      double v = one;
      int i = lane;
      wave_best(v, i);
      if (!(v > kNone)) break;
      keep |= 1ull << i;
      if (lane == i) one = kNone;
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int e = v * 64 + lane;
      c[v] = (keep >> (min(e, a.E - 1) / per)) & 1 ? c[v] : kNone;
    }
  }
  int mine = -1;
  double ms = 0.;
  for (int k = 0; k < a.K; k++) {
    double v = c[0], sv = s[0];
    int i = lane;
#pragma unroll
    for (int u = 1; u < V; u++) {
      const bool more = c[u] > v;
      v = more ? c[u] : v;
      sv = more ? s[u] : sv;
      i = more ? u * 64 + lane : i;
    }
    const int own = i;
    wave_best(v, i);
    if (!(v > kNone)) break;
    sv = __shfl(sv, i & 63, kWave);
    if (lane == k) {
      mine = i;
      ms = sv;
    }
#pragma unroll
    for (int u = 0; u < V; u++) c[u] = own == i && u == i >> 6 ? kNone : c[u];
  }
  double by = 1.;
  if (a.renorm) by = wave_sum(ms);
  if (lane < a.K) {
    a.idx[tok * a.K + lane] = mine;
    a.weight[tok * a.K + lane] = by > 0. ? (float)((double)a.scale * ms / by) : 0.f;
  }
}

// The gradient that one choice hands its own logit, in every mode but the softmax
// without renorm (whose sum reaches all experts): u = scale dweight, x the choice's
// logit (some: live, else u is 0), mx the token's largest.
//   sigmoid           u s (1 - s)
//   renorm, softmax   w (u - sum_j w_j u_j), w = s / sum_j s_j = e^(x - top) / sum_j ..
//   renorm, sigmoid   the same, times 1 - s
// 1 - s is taken from e^-|x|, and the shares w from differences to the largest
// chosen logit: neither cancels nor underflows where 1 - s or s do.  A sum of the
// scores that is 0 in 64 bits made weights of 0, whose gradient is 0.
template <class Sum, class Max>
__device__ __forceinline__ float choice_grad(bool some, float x, float u, float mx, int score, int renorm, Sum sum,
                                             Max max) {
  x = some ? x : 0.f;
  const float t = expf(-fabsf(x)), inv = 1.f / (1.f + t);
  if (!renorm) return u * (t * inv * inv);
  const float top = max(some ? x : -__builtin_inff());
  float f;
  if (score) f = x > 0.f ? inv : expf(x - fminf(top, 0.f)) * inv;  // s e^-min(top, 0)
  else f = x == top ? 1.f : expf(x - top);
  f = some ? f : 0.f;
  const float total = sum(f);
  const float w = total > 0.f ? f / total : 0.f;
  const float dot = sum(w * u);
  float g = w * (u - dot);
  if (score) g *= x > 0.f ? t * inv : inv;
  const bool none = score ? top < -709.78f : top - mx < -745.13f;
  return (int)some & (int)!none ? g : 0.f;
}

// One wave per token; lane k holds choice k.
template <int V>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteGradArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t tok = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tok >= a.T) return;
  const float* __restrict__ l = a.logits + tok * a.E;
  float x[V], s[V], mx = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < V; v++) {
    x[v] = live_logit(l, v * 64 + lane, a.E, a.active);
    mx = fmaxf(mx, x[v]);
  }
  mx = wave_max(mx);
  // this lane's choice
  int mine = -1;
  float u = 0.f, xm = -__builtin_inff();
  if (lane < a.K) {
    mine = a.idx[tok * a.K + lane];
    xm = live_logit(l, mine, a.E, a.active);
  }
  const bool some = xm > -__builtin_inff();
  mine = some ? mine : -1;
  if (some) u = a.dweight[tok * a.K + lane] * a.scale;
  const bool spread = !a.score && !a.renorm;  // (uniform) the softmax's sum reaches every expert
  float dot = 0.f;
  if (spread) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
      s[v] = !(x[v] > -__builtin_inff()) ? 0.f : x[v] == mx ? 1.f : expf(x[v] - mx);
      sum += s[v];
    }
    const float by = wave_sum(sum), p = by > 0.f ? 1.f / by : 0.f;  // (0: no expert is live)
#pragma unroll
    for (int v = 0; v < V; v++) s[v] *= p;
    dot = wave_sum(some ? u * ((xm == mx ? 1.f : expf(xm - mx)) * p) : 0.f);
  } else {
    u = choice_grad(some, xm, u, mx, a.score, a.renorm, [](float v) { return wave_sum(v); },
                    [](float v) { return wave_max(v); });
  }
  float ds[V];
#pragma unroll
  for (int v = 0; v < V; v++) ds[v] = 0.f;
  for (int k = 0; k < a.K; k++) {
    const int e = __builtin_amdgcn_readlane(mine, k);
    const float d = read_lane(u, k);
#pragma unroll
    for (int v = 0; v < V; v++) ds[v] += e == v * 64 + lane ? d : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; v++) {
    const int e = v * 64 + lane;
    if (e < a.E) a.dlogits[tok * a.E + e] = spread ? s[v] * (ds[v] - dot) : ds[v];
  }
}

// ---- up to 256 experts, up to 16 choices: 16 lanes a token ----
//
// Four tokens a wave: a row of 16 lanes holds a token's experts, V consecutive
// ones a lane, and reduces over itself by DPP moves alone (a whole wave's
// butterfly goes through LDS: six round trips a choice).  Bound by instruction issue:
// 16384 tokens, 8 of 256 experts in 8 groups 27 us (57 with a wave a token), 2460
// vector instructions a wave; the gradient by its bytes, 65536 tokens of 64 experts
// 9.8 us.  Measured and not kept: the choice in 32 bits first, and in 64 where two
// values of the order are near each other (30 us).
template <int CTRL>
__device__ __forceinline__ int dpp_int(int v) {
  return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)dpp_int<CTRL>((int)(uint32_t)b), hi = (uint32_t)dpp_int<CTRL>((int)(uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror: after each, all
// of 2, 4, 8, 16 lanes hold the same.
template <int CTRL>
__device__ __forceinline__ void best_step(double& v, int& i) {
  const double w = dpp_f64<CTRL>(v);
  const int j = dpp_int<CTRL>(i);
  const bool take = (int)(w > v) | ((int)(w == v) & (int)(j < i));
  v = take ? w : v;
  i = take ? j : i;
}
__device__ __forceinline__ void row_best(double& v, int& i) {
  best_step<0xB1>(v, i);
  best_step<0x4E>(v, i);
  best_step<0x141>(v, i);
  best_step<0x140>(v, i);
}
__device__ __forceinline__ double row_sum_f64(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  return v + dpp_f64<0x140>(v);
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v));
  v = fmaxf(v, dpp_mov<0x4E>(v));
  v = fmaxf(v, dpp_mov<0x141>(v));
  return fmaxf(v, dpp_mov<0x140>(v));
}

// Logits of V consecutive experts from e0, -inf where not live (see live_logit).
template <int V, bool VEC>
__device__ __forceinline__ void live_logits(const float* __restrict__ l, int e0, int E,
                                            const uint8_t* __restrict__ active, float (&x)[V]) {
  if constexpr (VEC) {  // (E % 4 == 0: a float4 is whole or out)
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      const bool in = e0 + v < E;
      const float4 f = *reinterpret_cast<const float4*>(l + (in ? e0 + v : 0));
      const float y[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int on = active ? active[in ? e0 + v + j : 0] : 1;
        x[v + j] = (int)in & (int)(on != 0) & (int)(y[j] > -__builtin_inff()) ? y[j] : -__builtin_inff();
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; v++) x[v] = live_logit(l, e0 + v, E, active);
  }
}

template <int V, bool VEC>
__global__ __launch_bounds__(256) void route_row_kernel(RouteArgs a) {
  __shared__ double by_expert[16][16 * V + 1];
  const int lane = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int64_t at = (int64_t)blockIdx.x * 16 + row;
  const bool in = at < a.T;
  const int64_t tok = in ? at : a.T - 1;  // (the rows past the end repeat the last token and store nothing)
  const int e0 = lane * V;
  float x[V], mx = -__builtin_inff();
  live_logits<V, VEC>(a.logits + tok * a.E, e0, a.E, a.active, x);
#pragma unroll
  for (int v = 0; v < V; v++) mx = fmaxf(mx, x[v]);
  mx = row_max(mx);
  double s[V], c[V], softmax_by = 0.;
  if (a.score == 0) {
    double sum = 0.;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const double z = x[v] == mx ? 0. : (double)x[v] - (double)mx;  // (a logit of +inf: 0)
      s[v] = x[v] > -__builtin_inff() ? exp(z) : 0.;
      sum += s[v];
    }
    sum = row_sum_f64(sum);
    softmax_by = sum > 0. ? 1. / sum : 0.;
#pragma unroll
    for (int v = 0; v < V; v++) s[v] *= softmax_by;
  } else {
#pragma unroll
    for (int v = 0; v < V; v++) s[v] = x[v] > -__builtin_inff() ? 1. / (1. + exp(-(double)x[v])) : 0.;
  }
#pragma unroll
  for (int v = 0; v < V; v++) {
    const double b = s[v] + (a.bias ? (double)a.bias[min(e0 + v, a.E - 1)] : 0.);
    c[v] = (int)(x[v] > -__builtin_inff()) & (int)(b > kNone) ? b : kNone;
  }
  if (a.groups > 1) {
    const int per = a.E / a.groups;
    uint64_t keep = 0;
    double one = kNone, two = kNone;
    auto merge = [&](double b) {
      two = b > one ? one : b > two ? b : two;
      one = b > one ? b : one;
    };
    if (per % V == 0) {  // (uniform) a lane's experts lie in one group, a group is `lanes` lanes
      const int lanes = per / V, g = lane / lanes, base = (threadIdx.x & 48) + g * lanes;
#pragma unroll
      for (int v = 0; v < V; v++) merge(c[v]);
      const double mine1 = one, mine2 = two;
      for (int o = 1; o < lanes; o++) {
        int from = lane - g * lanes + o;
        from = base + (from >= lanes ? from - lanes : from);
        const double b1 = __shfl(mine1, from, kWave), b2 = __shfl(mine2, from, kWave);
        merge(b1);
        merge(b2);
      }
      double value = (int)(a.group_best == 2) & (int)(two > kNone) ? one + two : one;
      value = g < a.groups ? value : kNone;
      for (int j = 0; j < a.top_groups; j++) {
        double v = value;
        int i = g;
        row_best(v, i);
        keep |= v > kNone ? 1ull << i : 0;
        value = i == g ? kNone : value;
      }
    } else {
      double* __restrict__ t = by_expert[row];
#pragma unroll
      for (int v = 0; v < V; v++) t[e0 + v] = c[v];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      double value[4];  // groups lane, lane + 16, ..
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int g = lane + 16 * q;
        one = two = kNone;
        if (g < a.groups)
          for (int j = 0; j < per; j++) merge(t[g * per + j]);
        value[q] = (int)(a.group_best == 2) & (int)(two > kNone) ? one + two : one;
      }
      for (int j = 0; j < a.top_groups; j++) {
        double v = value[0];
        int i = lane;
#pragma unroll
        for (int q = 1; q < 4; q++) {
          const bool more = value[q] > v;
          v = more ? value[q] : v;
          i = more ? lane + 16 * q : i;
        }
        row_best(v, i);
        keep |= v > kNone ? 1ull << i : 0;
#pragma unroll
        for (int q = 0; q < 4; q++) value[q] = i == lane + 16 * q ? kNone : value[q];
      }
    }
#pragma unroll
    for (int v = 0; v < V; v++) c[v] = (keep >> (min(e0 + v, a.E - 1) / per)) & 1 ? c[v] : kNone;
  }
  int mine = -1;
  for (int k = 0; k < a.K; k++) {
    double v = c[0];
    int i = e0;
#pragma unroll
    for (int u = 1; u < V; u++) {
      const bool more = c[u] > v;
      v = more ? c[u] : v;
      i = more ? e0 + u : i;
    }
    row_best(v, i);
    const bool some = v > kNone;
#pragma unroll
    for (int u = 0; u < V; u++) c[u] = i == e0 + u ? kNone : c[u];
    mine = (int)some & (int)(lane == k) ? i : mine;
  }
  // the score of this lane's choice, once more
  double ms = 0.;
  if (mine >= 0) {
    const float xm = a.logits[tok * a.E + mine];
    ms = a.score ? 1. / (1. + exp(-(double)xm)) : (xm == mx ? 1. : exp((double)xm - (double)mx)) * softmax_by;
  }
  const double by = a.renorm ? row_sum_f64(ms) : 1.;
  if (in && lane < a.K) {
    a.idx[tok * a.K + lane] = mine;
    a.weight[tok * a.K + lane] = by > 0. ? (float)((double)a.scale * ms / by) : 0.f;
  }
}

template <int V, bool VEC>
__global__ __launch_bounds__(256) void route_grad_row_kernel(RouteGradArgs a) {
  const int lane = threadIdx.x & 15;
  const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool in = at < a.T;
  const int64_t tok = in ? at : a.T - 1;
  const float* __restrict__ l = a.logits + tok * a.E;
  const int e0 = lane * V;
  // this lane's choice
  int mine = -1;
  float dw = 0.f, xm = -__builtin_inff();
  if (lane < a.K) {
    mine = a.idx[tok * a.K + lane];
    dw = a.dweight[tok * a.K + lane];
  }
  float x[V], s[V], mx = -__builtin_inff();
  live_logits<V, VEC>(l, e0, a.E, a.active, x);
  xm = live_logit(l, mine, a.E, a.active);
#pragma unroll
  for (int v = 0; v < V; v++) mx = fmaxf(mx, x[v]);
  mx = row_max(mx);
  const bool some = xm > -__builtin_inff();  // (false without a choice: mine -1 is not live)
  mine = some ? mine : -1;
  float u = some ? dw * a.scale : 0.f;
  const bool spread = !a.score && !a.renorm;
  float dot = 0.f;
  if (spread) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
      s[v] = !(x[v] > -__builtin_inff()) ? 0.f : x[v] == mx ? 1.f : expf(x[v] - mx);
      sum += s[v];
    }
    const float by = row16_sum(sum), p = by > 0.f ? 1.f / by : 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) s[v] *= p;
    dot = row16_sum(some ? u * ((xm == mx ? 1.f : expf(xm - mx)) * p) : 0.f);
  } else {
    u = choice_grad(some, xm, u, mx, a.score, a.renorm, [](float v) { return row16_sum(v); },
                    [](float v) { return row_max(v); });
  }
  float ds[V];
#pragma unroll
  for (int v = 0; v < V; v++) ds[v] = 0.f;
  for (int k = 0; k < a.K; k++) {
    const int from = (threadIdx.x & 48) + k;
    const int e = __shfl(mine, from, kWave) - e0;
    const float d = __shfl(u, from, kWave);
#pragma unroll
    for (int v = 0; v < V; v++) ds[v] += e == v ? d : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; v++) ds[v] = spread ? s[v] * (ds[v] - dot) : ds[v];
  if (!in) return;
  float* __restrict__ to = a.dlogits + tok * a.E;
  if constexpr (VEC) {
#pragma unroll
    for (int v = 0; v < V; v += 4)
      if (e0 + v < a.E) *reinterpret_cast<float4*>(to + e0 + v) = make_float4(ds[v], ds[v + 1], ds[v + 2], ds[v + 3]);
  } else {
#pragma unroll
    for (int v = 0; v < V; v++)
      if (e0 + v < a.E) to[e0 + v] = ds[v];
  }
}

// ---- slots sorted by expert -------------------------------------------------------

constexpr int kSortBlock = 1024;  // slots a workgroup

// A wave's lanes that hold the same expert (e in [0, E), E <= 1024; -1: none).
__device__ __forceinline__ uint64_t same_expert(int e) {
  uint64_t m = __ballot(e >= 0);
#pragma unroll
  for (int b = 0; b < 10; b++) {
    const uint64_t set = __ballot((e >> b) & 1);
    m &= (e >> b) & 1 ? set : ~set;
  }
  return e >= 0 ? m : 0;
}
__device__ __forceinline__ int slot_expert(const int32_t* __restrict__ idx, int64_t i, int64_t N, int E) {
  if (i >= N) return -1;
  const int e = idx[i];
  return e >= 0 && e < E ? e : -1;
}

// count[block][e]: the block's slots of each expert.  fill (not 0): perm and
// tok of positions 0 .. fill - 1 are set to -1.
__global__ __launch_bounds__(kSortBlock) void slots_count_kernel(const int32_t* __restrict__ idx, int64_t N, int E,
                                                                 int* __restrict__ count, int* __restrict__ perm,
                                                                 int* __restrict__ tok, int64_t fill) {
  __shared__ int c[kMoeMaxExperts];
  for (int64_t i = (int64_t)blockIdx.x * kSortBlock + threadIdx.x; i < fill; i += (int64_t)gridDim.x * kSortBlock) {
    perm[i] = -1;
    tok[i] = -1;
  }
  for (int e = threadIdx.x; e < E; e += kSortBlock) c[e] = 0;
  __syncthreads();
  const int e = slot_expert(idx, (int64_t)blockIdx.x * kSortBlock + threadIdx.x, N, E);
  const uint64_t m = same_expert(e);
  if (e >= 0 && (threadIdx.x & 63) == __builtin_ctzll(m)) atomicAdd(&c[e], __builtin_popcountll(m));
  __syncthreads();
  for (int i = threadIdx.x; i < E; i += kSortBlock) count[(int64_t)blockIdx.x * E + i] = c[i];
}

// Inclusive sum over the 1024 threads; `room`: 16 ints.
__device__ __forceinline__ int block_scan(int v, int* room) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int b = __shfl_up(v, o, kWave);
    v += lane >= o ? b : 0;
  }
  __syncthreads();  // (room's last use)
  if (lane == 63) room[w] = v;
  __syncthreads();
  int before = 0;
  for (int u = 0; u < w; u++) before += room[u];
  return before + v;
}

// Each expert's segment (its start rounded up to `pad` positions), the blocks'
// offsets in it (in place of their counts), the (expert, tile of bm rows) list
// and, blk not null, the expert of every `pad` positions.  One workgroup: thread
// (part, expert) sums a run of blocks, then the sums of all (expert, part) are
// scanned in that order.
__global__ __launch_bounds__(1024) void slots_scan_kernel(int* __restrict__ count, int nblk, int E, int pad, int bm,
                                                          int* __restrict__ seg, int* __restrict__ tiles,
                                                          int* __restrict__ ntiles, int* __restrict__ blk) {
  __shared__ int sum[1024], before[1024], start[1024], room[16];
  const int t = threadIdx.x;
  int ep = 1;
  while (ep < E) ep <<= 1;
  const int parts = 1024 / ep, e = t & (ep - 1), part = t / ep;
  const int run = (nblk + parts - 1) / parts, b0 = min(nblk, part * run), b1 = min(nblk, b0 + run);
  int c = 0;
  if (e < E) {
#pragma unroll 8
    for (int b = b0; b < b1; b++) c += count[(int64_t)b * E + e];
  }
  sum[e * parts + part] = c;
  __syncthreads();
  const int v = sum[t];
  before[t] = block_scan(v, room) - v;
  __syncthreads();
  // thread e: its expert's total, segment and tiles
  int total = 0;
  if (t < E) total = (t + 1 < ep ? before[(t + 1) * parts] : before[1023] + sum[1023]) - before[t * parts];
  const int padded = (total + pad - 1) / pad * pad, nt = (total + bm - 1) / bm;
  const int at = block_scan(padded, room) - padded, ta = block_scan(nt, room) - nt;
  if (t < E) {
    start[t] = at;
    seg[t] = at;
    if (t == E - 1) {
      seg[E] = at + padded;
      *ntiles = ta + nt;
    }
    for (int i = 0; i < nt; i++) {
      tiles[2 * (ta + i)] = t;
      tiles[2 * (ta + i) + 1] = i;
    }
    if (blk)
      for (int i = 0; i < padded / pad; i++) blk[at / pad + i] = t;
  }
  __syncthreads();
  if (e >= E) return;
  int off = start[e] + before[e * parts + part] - before[e * parts];
  for (int b = b0; b < b1; b++) {
    const int n = count[(int64_t)b * E + e];
    count[(int64_t)b * E + e] = off;
    off += n;
  }
}

// perm[position] = slot, tok[position] = its token (stable), expert[slot].
__global__ __launch_bounds__(kSortBlock) void slots_place_kernel(const int32_t* __restrict__ idx, int64_t N, int E,
                                                                 int K, const int* __restrict__ offset,
                                                                 int* __restrict__ perm, int* __restrict__ tok,
                                                                 int* __restrict__ expert) {
  __shared__ int c[16][kMoeMaxExperts];  // slots of each expert in the waves before
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < 16 * E; i += kSortBlock) c[i / E][i % E] = 0;
  __syncthreads();
  const int64_t slot = (int64_t)blockIdx.x * kSortBlock + threadIdx.x;
  const int e = slot_expert(idx, slot, N, E);
  if (slot < N) expert[slot] = e;
  const uint64_t m = same_expert(e);
  const int rank = __builtin_popcountll(m & ((1ull << lane) - 1));
  if (e >= 0 && rank == 0) c[w][e] = __builtin_popcountll(m);
  __syncthreads();
  if (e < 0) return;
  int at = offset[(int64_t)blockIdx.x * E + e] + rank;
  for (int u = 0; u < w; u++) at += c[u][e];
  perm[at] = (int)slot;
  tok[at] = (int)(slot / K);
}

// ---- rows ---------------------------------------------------------------------------

// y[t] = sum over the token's slots, in order, of o[slot]; slots without an
// expert add nothing (their rows of o are not written).
template <int W>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ o, const int* __restrict__ expert,
                                                      float* __restrict__ y, int64_t T, int K, int64_t DW) {
  const int64_t n = T * DW;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / DW, c = i - t * DW;
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j++) v[j] = 0.f;
    for (int k = 0; k < K; k++) {
      if (expert[t * K + k] < 0) continue;
      const float* p = o + ((t * K + k) * DW + c) * W;
#pragma unroll
      for (int j = 0; j < W; j++) v[j] += p[j];
    }
#pragma unroll
    for (int j = 0; j < W; j++) y[i * W + j] = v[j];
  }
}

// One wave per sorted row: dweight = act(u) . dh, du = weight act'(u) dh (in
// place of dh), hw = weight act(u).
__global__ __launch_bounds__(256) void bwd_rows_kernel(const float* __restrict__ pre, float* __restrict__ dh,
                                                       float* __restrict__ hw, const float* __restrict__ weight,
                                                       float* __restrict__ dweight, const int* __restrict__ perm,
                                                       const int* __restrict__ nrows, int H, int act) {
  const int lane = threadIdx.x & 63;
  const int64_t pos = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (pos >= *nrows) return;
  const int slot = perm[pos];
  const float w = weight[slot];
  float dot = 0.f;
  for (int a = lane; a < H; a += 64) {
    const float d = dh[pos * H + a];
    float h, slope;
    act_both(pre[pos * H + a], act, h, slope);
    dot += h * d;
    dh[pos * H + a] = w * d * slope;
    hw[pos * H + a] = w * h;
  }
  dot = wave_sum(dot);
  if (dweight && lane == 0) dweight[slot] = dot;
}

// a2[pos] = a[tok[pos]], b2 alike
__global__ __launch_bounds__(256) void gather_kernel(const float* __restrict__ a, const float* __restrict__ b,
                                                     const int* __restrict__ tok, const int* __restrict__ nrows,
                                                     float* __restrict__ a2, float* __restrict__ b2, int64_t D) {
  const int64_t n = (int64_t)*nrows * D;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / D, src = (int64_t)tok[r] * D + (i - r * D);
    a2[i] = a[src];
    b2[i] = b[src];
  }
}

// ---- few slots --------------------------------------------------------------------
//
// Where the experts hold a handful of slots each, a product is bound by its
// weights' bytes, and with one token by latency: no sort, fp32 multiply-adds (8
// rows cost a quarter of the time that the weights take to arrive).  Workgroup
// (column tile, expert, K chunk) lists the expert's slots itself and streams 64
// columns of its chunk once for up to 8 of them (with fewer slots than experts:
// (column tile, slot, K chunk), and the first of an expert's slots does it).  The
// chunks make enough workgroups to fill the chip and are summed, in their order, by
// whoever reads them: the second product as it stages act(u), the last pass as it
// weighs the slots.  64 experts of 1024 x 1024, two slots a token: one token 12 us
// (sorted 186), 37 tokens 90 us, 4.1 TB/s of weights (sorted 197).
constexpr int kFewSlots = 1024;  // most slots (a list in LDS)
constexpr int kFewRows = 8;      // rows a pass over the weights
constexpr int kFewK = 512;       // contraction staged at once

struct FewArgs {
  const float* in;     // FIRST: x [T, k]; else partial sums [parts][slots, k] of u
  const float* W;      // [E, k, cols]
  const int32_t* idx;
  float* out;          // [chunks][slots, cols]
  float* keep;         // second product: u [slots, k] for the gradient, or null
  int slots, choices, E, k, cols, chunk, parts, act;
  bool by_slot;
};

// Sum of p[0], p[stride], ... in order, four loads in flight.
__device__ __forceinline__ float sum_parts(const float* __restrict__ p, int64_t stride, int parts) {
  float v = 0.f;
  for (int z = 0; z < parts; z += 4) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = p[min(z + u, parts - 1) * stride];
#pragma unroll
    for (int u = 0; u < 4; u++) v += z + u < parts ? x[u] : 0.f;
  }
  return v;
}

// VEC: 16 lanes of four columns and four k a wave, else 64 columns.
template <bool FIRST, int VEC>
__global__ __launch_bounds__(256) void few_kernel(FewArgs a) {
  constexpr int KR = VEC == 4 ? 4 : 1, STEP = 4 * KR, UN = 8;
  __shared__ int list[kFewSlots];
  __shared__ int count;
  __shared__ __attribute__((aligned(16))) float xs[kFewK * kFewRows];
  __shared__ float red[4][kFewRows * 64];
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int e = a.by_slot ? a.idx[blockIdx.y] : (int)blockIdx.y;
  if (e < 0 || e >= a.E) return;
  if (w == 0) {
    int n = 0;
    for (int s = lane; s < a.slots + lane; s += 64) {
      const uint64_t m = __ballot(s < a.slots && a.idx[s < a.slots ? s : 0] == e);
      if ((m >> lane) & 1) list[n + __builtin_popcountll(m & ((1ull << lane) - 1))] = s;
      n += __builtin_popcountll(m);
    }
    if (lane == 0) count = n;
  }
  __syncthreads();
  const int n = count;
  if (n == 0 || (a.by_slot && list[0] != (int)blockIdx.y)) return;
  const int kbeg = blockIdx.z * a.chunk, kend = min(a.k, kbeg + a.chunk);
  const int lc = VEC == 4 ? (lane & 15) * 4 : lane, kr = VEC == 4 ? lane >> 4 : 0;
  const int col0 = blockIdx.x * 64;
  const int col = min(col0 + lc, a.cols - VEC);  // (columns past the end are not stored)
  const float* __restrict__ W = a.W + (int64_t)e * a.k * a.cols + col;
  float* __restrict__ out = a.out + (int64_t)blockIdx.z * a.slots * a.cols;
  auto pass = [&](int r0, auto rows) {
    constexpr int R = decltype(rows)::value;
    const int nr = min(R, n - r0);
    float acc[R][VEC];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int j = 0; j < VEC; j++) acc[r][j] = 0.f;
    for (int k0 = kbeg; k0 < kend; k0 += kFewK) {
      const int kn = min(kFewK, kend - k0);
      __syncthreads();  // (the last stage is read)
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int slot = list[r0 + min(r, nr - 1)];
        for (int k = t; k < kn; k += 256) {
          float v;
          if (FIRST) {
            v = a.in[(int64_t)(slot / a.choices) * a.k + k0 + k];
          } else {
            const float* p = a.in + (int64_t)slot * a.k + k0 + k;
            v = sum_parts(p, (int64_t)a.slots * a.k, a.parts);
            if (a.keep && blockIdx.x == 0 && r < nr) a.keep[(int64_t)slot * a.k + k0 + k] = v;
            v = act_apply(v, a.act);
          }
          xs[k * R + r] = r < nr ? v : 0.f;
        }
      }
      __syncthreads();
      auto steps = [&](int kk, auto count, auto check) {
        constexpr int CNT = decltype(count)::value;
        constexpr bool CHK = decltype(check)::value;
        float v[CNT][VEC];
#pragma unroll
        for (int u = 0; u < CNT; u++) {
          const int k = kk + u * STEP;
          const float* q = W + (int64_t)(k0 + (CHK ? min(k, kn - 1) : k)) * a.cols;
          if (VEC == 4) {
            const float4 f = *reinterpret_cast<const float4*>(q);
            v[u][0] = f.x; v[u][VEC / 4] = f.y; v[u][VEC / 2] = f.z; v[u][VEC - 1] = f.w;
          } else {
            v[u][0] = *q;
          }
        }
#pragma unroll
        for (int u = 0; u < CNT; u++) {
          const int k = kk + u * STEP;
          const float* x = xs + (CHK ? min(k, kn - 1) : k) * R;
#pragma unroll
          for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
              const float f = CHK && k >= kn ? 0.f : v[u][j];
              acc[r][j] = fmaf(CHK && k >= kn ? 0.f : x[r], f, acc[r][j]);
            }
        }
      };
      int kk = w * KR + kr, left = kn;
      for (; left >= UN * STEP; left -= UN * STEP, kk += UN * STEP)
        steps(kk, std::integral_constant<int, UN>{}, std::false_type{});
      for (; left > 0; left -= 2 * STEP, kk += 2 * STEP) steps(kk, std::integral_constant<int, 2>{}, std::true_type{});
    }
    if (VEC == 4) {
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          acc[r][j] += __shfl_xor(acc[r][j], 16, kWave);
          acc[r][j] += __shfl_xor(acc[r][j], 32, kWave);
        }
    }
    if (VEC == 1 || lane < 16) {
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < VEC; j++) red[w][r * 64 + lc + j] = acc[r][j];
    }
    __syncthreads();
    for (int i = t; i < nr * 64; i += 256) {
      const int c = col0 + (i & 63);
      if (c < a.cols)
        out[(int64_t)list[r0 + (i >> 6)] * a.cols + c] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    }
  };
  for (int r0 = 0; r0 < n; r0 += kFewRows) {
    const int left = n - r0;
    if (left == 1) pass(r0, std::integral_constant<int, 1>{});
    else if (left == 2) pass(r0, std::integral_constant<int, 2>{});
    else if (left <= 4) pass(r0, std::integral_constant<int, 4>{});
    else pass(r0, std::integral_constant<int, 8>{});
    __syncthreads();  // (red is read)
  }
}

// y[t] = sum over the token's slots of weight * (sum over the chunks of o);
// expert (not null): the slots' experts for the gradient, -1 where idx is out of
// range.
__global__ __launch_bounds__(256) void few_combine_kernel(const float* __restrict__ o, const int32_t* __restrict__ idx,
                                                          const float* __restrict__ weight, float* __restrict__ y,
                                                          int* __restrict__ expert, int64_t n, int choices, int cols,
                                                          int E, int slots, int parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int t = (int)(i / cols), c = (int)(i - (int64_t)t * cols);
  float y0 = 0.f;
  for (int k = 0; k < choices; k++) {
    const int slot = t * choices + k, e = idx[slot];
    const bool out = e < 0 || e >= E;
    if (expert && c == 0) expert[slot] = out ? -1 : e;
    if (out) continue;
    y0 += weight[slot] * sum_parts(o + (int64_t)slot * cols + c, (int64_t)slots * cols, parts);
  }
  y[i] = y0;
}

// The slots of an expert into `list`, by one wave; their number to *count.
__device__ __forceinline__ void list_slots(const int* __restrict__ expert, int slots, int e, int* list, int* count) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int s0 = 0; s0 < slots; s0 += 64) {
    const int s = s0 + lane;
    const uint64_t m = __ballot(s < slots && expert[min(s, slots - 1)] == e);
    if ((m >> lane) & 1) list[n + __builtin_popcountll(m & ((1ull << lane) - 1))] = s;
    n += __builtin_popcountll(m);
  }
  if (lane == 0) *count = n;
}

// out[slot, row] = sum_k in[slot, k] W[e][row, k]: rows of W along the lanes, four
// rows a wave, up to 8 slots a pass, each row's sums met by wave reductions.
// in: row slot (choices 0) or slot / choices.
struct FewRowsArgs {
  const float* in;
  const float* W;       // [E, rows, k]
  const int* expert;    // [slots]
  float* out;           // [slots, rows]
  int slots, choices, k, rows, E;
  bool by_slot;
};
template <bool VEC>
__global__ __launch_bounds__(256) void few_rows_kernel(FewRowsArgs a) {
  constexpr int R = kFewRows, W4 = VEC ? 4 : 1, CHUNK = 1024, STEPS = CHUNK / (64 * W4);
  __shared__ int list[kFewSlots];
  __shared__ int count;
  __shared__ __attribute__((aligned(16))) float xs[R][CHUNK];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int e = a.by_slot ? a.expert[blockIdx.y] : (int)blockIdx.y;
  if (e < 0) return;
  if (w == 0) list_slots(a.expert, a.slots, e, list, &count);
  __syncthreads();
  const int n = count;
  if (n == 0 || (a.by_slot && list[0] != (int)blockIdx.y)) return;
  const int row0 = blockIdx.x * 16 + w * 4;
  for (int r0 = 0; r0 < n; r0 += R) {
    const int nr = min(R, n - r0);
    float acc[4][R];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int r = 0; r < R; r++) acc[j][r] = 0.f;
    for (int k0 = 0; k0 < a.k; k0 += CHUNK) {
      const int kn = min(CHUNK, a.k - k0);
      __syncthreads();
      for (int r = 0; r < nr; r++) {
        const int slot = list[r0 + r], from = a.choices ? slot / a.choices : slot;
        for (int k = t; k < CHUNK; k += 256) xs[r][k] = k < kn ? a.in[(int64_t)from * a.k + k0 + k] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float* __restrict__ p = a.W + ((int64_t)e * a.rows + min(row0 + j, a.rows - 1)) * a.k + k0;
        float v[STEPS][W4];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
          const int k = (s * 64 + lane) * W4;
          const bool in = k < kn;
          if constexpr (VEC) {
            const float4 f = *reinterpret_cast<const float4*>(p + (in ? k : 0));
            v[s][0] = in ? f.x : 0.f; v[s][1] = in ? f.y : 0.f; v[s][2] = in ? f.z : 0.f; v[s][3] = in ? f.w : 0.f;
          } else {
            const float f = p[in ? k : 0];
            v[s][0] = in ? f : 0.f;
          }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
          if (r >= nr) break;  // (uniform)
#pragma unroll
          for (int s = 0; s < STEPS; s++) {
            const int k = (s * 64 + lane) * W4;
            if constexpr (VEC) {
              const float4 x = *reinterpret_cast<const float4*>(&xs[r][k]);
              acc[j][r] += (x.x * v[s][0] + x.y * v[s][1]) + (x.z * v[s][2] + x.w * v[s][3]);
            } else {
              acc[j][r] += xs[r][k] * v[s][0];
            }
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (r >= nr) break;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float d = wave_sum(acc[j][r]);
        if (lane == j && row0 + j < a.rows) a.out[(int64_t)list[r0 + r] * a.rows + row0 + j] = d;
      }
    }
  }
}

// One wave a slot: dweight = act(u) . dh, du = weight act'(u) dh (in place of dh),
// hw = weight act(u); slots without an expert get a dweight of 0.
__global__ __launch_bounds__(256) void few_back_kernel(const float* __restrict__ u, float* __restrict__ dh,
                                                       float* __restrict__ hw, const float* __restrict__ weight,
                                                       float* __restrict__ dweight, const int* __restrict__ expert,
                                                       int slots, int H, int act) {
  const int lane = threadIdx.x & 63, slot = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (slot >= slots) return;
  if (expert[slot] < 0) {
    if (dweight && lane == 0) dweight[slot] = 0.f;
    return;
  }
  const float w = weight[slot];
  float dot = 0.f;
  for (int i = lane; i < H; i += 64) {
    const int64_t at = (int64_t)slot * H + i;
    const float d = dh[at];
    float h, slope;
    act_both(u[at], act, h, slope);
    dot += h * d;
    dh[at] = w * d * slope;
    hw[at] = w * h;
  }
  dot = wave_sum(dot);
  if (dweight && lane == 0) dweight[slot] = dot;
}

// C[e] [M, N] = the sum over e's slots of A[slot] (column) B[slot] (row); zeros
// without slots.  A, B: row slot, or slot / choices where ca, cb.  A workgroup: 16
// rows by up to 1024 columns (256 without float4), eight rows a thread at a time.
struct FewOuterArgs {
  const float* A;
  const float* B;
  const int* expert;
  float* C;
  int slots, ca, cb, M, N, ctiles;
};
template <bool VEC>
__global__ __launch_bounds__(256) void few_outer_kernel(FewOuterArgs a) {
  constexpr int W4 = VEC ? 4 : 1, RT = 8;
  __shared__ int list[kFewSlots];
  __shared__ int count;
  const int t = threadIdx.x, e = blockIdx.y;
  if (t < 64) list_slots(a.expert, a.slots, e, list, &count);
  __syncthreads();
  const int n = count, col = (int)(blockIdx.x % a.ctiles * 256 + t) * W4;
  if (col >= a.N) return;
  for (int h = 0; h < 2; h++) {
    const int row0 = (int)(blockIdx.x / a.ctiles) * 16 + h * RT;
    if (row0 >= a.M) return;
    float acc[RT][W4];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int j = 0; j < W4; j++) acc[r][j] = 0.f;
    for (int s = 0; s < n; s++) {
      const int slot = __builtin_amdgcn_readfirstlane(list[s]);
      const float* __restrict__ p = a.A + (int64_t)(a.ca ? slot / a.ca : slot) * a.M;
      const float* __restrict__ q = a.B + (int64_t)(a.cb ? slot / a.cb : slot) * a.N + col;
      float b[W4];
      if constexpr (VEC) {
        const float4 f = *reinterpret_cast<const float4*>(q);
        b[0] = f.x; b[1] = f.y; b[2] = f.z; b[3] = f.w;
      } else {
        b[0] = *q;
      }
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const float x = p[min(row0 + r, a.M - 1)];  // (uniform)
#pragma unroll
        for (int j = 0; j < W4; j++) acc[r][j] = fmaf(x, b[j], acc[r][j]);
      }
    }
    float* __restrict__ c = a.C + (int64_t)e * a.M * a.N + col;
#pragma unroll
    for (int r = 0; r < RT; r++) {
      if (row0 + r >= a.M) break;
      float* to = c + (int64_t)(row0 + r) * a.N;
      if constexpr (VEC) *reinterpret_cast<float4*>(to) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
      else *to = acc[r][0];
    }
  }
}

constexpr int64_t round64(int64_t n) { return (n + 63) / 64 * 64; }
int64_t tables_ints(int64_t N, int64_t E) {
  return round64(E + 1) + 3 * round64(N) + round64(2 * (ceil_div(N, 128) + E)) + 64;
}
SlotTables tables_at(int* p, int64_t N, int64_t E) {
  SlotTables t;
  t.seg = p;
  t.perm = t.seg + round64(E + 1);
  t.tok = t.perm + round64(N);
  t.expert = t.tok + round64(N);
  t.tiles = t.expert + round64(N);
  t.ntiles = t.tiles + round64(2 * (ceil_div(N, 128) + E));
  return t;
}

unsigned stream_blocks(int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(n, 256), 8192)); }

GemmArgs grouped(const SlotTables& t, int64_t rows, int64_t N, int64_t K, const float* A, const float* B, float* C,
                 const MoeShape& m, bool tB) {
  GemmArgs g;
  g.A = A; g.B = B; g.C = C;
  g.M = (int)rows; g.N = (int)N; g.K = (int)K;
  g.lda = K; g.ldb = tB ? K : N; g.ldc = N;
  g.groups = (int)m.E; g.seg = t.seg; g.tiles = t.tiles; g.ntiles = t.ntiles; g.sBg = N * K;
  g.narrow = N <= 128;
  return g;
}

}  // namespace

static bool rows_of_16(int64_t E, int64_t K) { return E <= 256 && K <= 16; }
static bool logits_float4(int64_t E, const void* p, const void* q) {
  return E % 4 == 0 && ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15) == 0;
}

#define NSH_ROUTE_ROWS(KERNEL_)                                                                     \
  do {                                                                                              \
    const dim3 g((unsigned)ceil_div(a.T, 16));                                                      \
    if (a.E <= 16) hipLaunchKernelGGL((KERNEL_<1, false>), g, dim3(256), 0, s, a);                  \
    else if (vec && a.E <= 64) hipLaunchKernelGGL((KERNEL_<4, true>), g, dim3(256), 0, s, a);       \
    else if (vec && a.E <= 128) hipLaunchKernelGGL((KERNEL_<8, true>), g, dim3(256), 0, s, a);      \
    else if (vec) hipLaunchKernelGGL((KERNEL_<16, true>), g, dim3(256), 0, s, a);                   \
    else if (a.E <= 64) hipLaunchKernelGGL((KERNEL_<4, false>), g, dim3(256), 0, s, a);             \
    else hipLaunchKernelGGL((KERNEL_<16, false>), g, dim3(256), 0, s, a);                           \
  } while (0)

int launch_combine(const float* o, const int* expert, float* y, const MoeShape& m, hipStream_t s) {
  if (m.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(y)) & 15) == 0)
    hipLaunchKernelGGL(combine_kernel<4>, dim3(stream_blocks(m.T * m.D / 4)), dim3(256), 0, s, o, expert, y, m.T,
                       (int)m.K, m.D / 4);
  else
    hipLaunchKernelGGL(combine_kernel<1>, dim3(stream_blocks(m.T * m.D)), dim3(256), 0, s, o, expert, y, m.T, (int)m.K,
                       m.D);
  NSH_LAUNCHED();
  return 0;
}

int64_t sort_count_ints(int64_t N, int64_t E) { return round64(ceil_div(N, kSortBlock) * E); }

int launch_sort_slots(const int32_t* idx, const SlotTables& t, int* count, int64_t N, int K, int E, int pad, int bm,
                      int64_t fill, hipStream_t s) {
  const int nblk = (int)ceil_div(N, kSortBlock);
  hipLaunchKernelGGL(slots_count_kernel, dim3(nblk), dim3(kSortBlock), 0, s, idx, N, E, count, t.perm, t.tok, fill);
  NSH_LAUNCHED();
  hipLaunchKernelGGL(slots_scan_kernel, dim3(1), dim3(1024), 0, s, count, nblk, E, pad, bm, t.seg, t.tiles, t.ntiles,
                     t.blk);
  NSH_LAUNCHED();
  hipLaunchKernelGGL(slots_place_kernel, dim3(nblk), dim3(kSortBlock), 0, s, idx, N, E, K, count, t.perm, t.tok,
                     t.expert);
  NSH_LAUNCHED();
  return 0;
}

int launch_route(const RouteArgs& a, hipStream_t s) {
  if (a.T <= 0) return 0;
  if (rows_of_16(a.E, a.K)) {
    const bool vec = logits_float4(a.E, a.logits, nullptr);
    NSH_ROUTE_ROWS(route_row_kernel);
    NSH_LAUNCHED();
    return 0;
  }
  const dim3 g((unsigned)ceil_div(a.T, 4));
  if (a.E <= 256) hipLaunchKernelGGL(route_kernel<4>, g, dim3(256), 0, s, a);
  else if (a.E <= 512) hipLaunchKernelGGL(route_kernel<8>, g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(route_kernel<16>, g, dim3(256), 0, s, a);
  NSH_LAUNCHED();
  return 0;
}

int launch_route_grad(const RouteGradArgs& a, hipStream_t s) {
  if (a.T <= 0) return 0;
  if (rows_of_16(a.E, a.K)) {
    const bool vec = logits_float4(a.E, a.logits, a.dlogits);
    NSH_ROUTE_ROWS(route_grad_row_kernel);
    NSH_LAUNCHED();
    return 0;
  }
  const dim3 g((unsigned)ceil_div(a.T, 4));
  if (a.E <= 256) hipLaunchKernelGGL(route_grad_kernel<4>, g, dim3(256), 0, s, a);
  else if (a.E <= 512) hipLaunchKernelGGL(route_grad_kernel<8>, g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(route_grad_kernel<16>, g, dim3(256), 0, s, a);
  NSH_LAUNCHED();
  return 0;
}

// Whether the layer runs without a sort: up to 6 slots an expert on average.  64
// experts of 1024 x 1024, two slots a token, us, this and sorted: 1 token 12,
// 186; 32 tokens 87, 198; 128 137, 204; 200 184, 207; 256 217, 208.
// That is serving on a balanced router.  With gradients the sorted way is ahead
// sooner (192 tokens, 6 slots an expert: 731, 602), of 64 experts of 64 x 256 (both
// products in one kernel) from about 3 slots an expert: 94, 82, and 128, 82 at 6.
// Every 8 slots of one expert are a pass after the other, so tokens that agree on
// two experts wait for it: 192 of them 1006, 202, of 64 x 256 368, 26.
constexpr int kFewPerExpert = 6;
static bool few_slots(const MoeShape& m) { return m.T * m.K <= kFewSlots && m.T * m.K <= kFewPerExpert * m.E; }
// K chunks of a product [.., k] x [k, cols] over the experts that `slots` reach:
// about 256 workgroups, of 64 steps of K at least (64 experts of 1024 x 1024, 1
// and 8 tokens of 2 slots, us: 128 workgroups 11.1, 33.3; 256 11.6, 33.3; 512
// 15.3, 27.5; 1024 15.2, 30.1: the chunks' sums cost a round trip for each four).
static int few_chunks(int64_t k, int64_t cols, int64_t slots, int64_t E) {
  const int64_t wgs = ceil_div(cols, 64) * std::min(slots, E);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(16, ceil_div(256, wgs)), k / 64));
}

// state: the slots' experts, then u [N, H] by slot
static int launch_few(const float* x, const int32_t* idx, const float* weight, const float* W1, const float* W2,
                      float* y, const MoeShape& m, int act, void* state, void* workspace, hipStream_t s) {
  const int64_t N = m.T * m.K;
  FewArgs a;
  a.slots = (int)N; a.choices = (int)m.K; a.E = (int)m.E; a.idx = idx; a.act = act;
  a.by_slot = N < m.E;
  auto product = [&](auto first, int64_t k, int64_t cols, const float* W) {
    constexpr bool FIRST = decltype(first)::value;
    const int chunks = few_chunks(k, cols, N, m.E);
    a.W = W; a.k = (int)k; a.cols = (int)cols;
    a.chunk = (int)ceil_div(k, chunks);
    const dim3 g((unsigned)ceil_div(cols, 64), (unsigned)std::min(N, m.E), (unsigned)ceil_div(k, a.chunk));
    if (cols % 4 == 0 && (reinterpret_cast<uintptr_t>(W) & 15) == 0)
      hipLaunchKernelGGL((few_kernel<FIRST, 4>), g, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((few_kernel<FIRST, 1>), g, dim3(256), 0, s, a);
    return (int)g.z;
  };
  float* u = static_cast<float*>(workspace);
  float* o = u + round64(few_chunks(m.D, m.H, N, m.E) * N * m.H);
  a.in = x; a.out = u; a.keep = nullptr; a.parts = 1;
  a.parts = product(std::true_type{}, m.D, m.H, W1);
  NSH_LAUNCHED();
  int* expert = static_cast<int*>(state);
  a.in = u; a.out = o;
  a.keep = state ? reinterpret_cast<float*>(expert + round64(N)) : nullptr;
  const int parts = product(std::false_type{}, m.H, m.D, W2);
  NSH_LAUNCHED();
  hipLaunchKernelGGL(few_combine_kernel, dim3((unsigned)ceil_div(m.T * m.D, 256)), dim3(256), 0, s, o, idx, weight, y,
                     expert, m.T * m.D, (int)m.K, (int)m.D, (int)m.E, (int)N, parts);
  NSH_LAUNCHED();
  return 0;
}

static int launch_few_grad(const float* dy, const float* x, const float* weight, const float* W1, const float* W2,
                           const void* state, float* dx, float* dweight, float* dW1, float* dW2, const MoeShape& m,
                           int act, void* workspace, hipStream_t s) {
  const int64_t N = m.T * m.K;
  const int* expert = static_cast<const int*>(state);
  const float* u = reinterpret_cast<const float*>(expert + round64(N));
  float* dh = static_cast<float*>(workspace);
  float* hw = dh + round64(N * m.H);
  float* slots = hw + round64(N * m.H);
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  auto rows = [&](const float* in, int choices, const float* W, float* out, int64_t k, int64_t nrows) -> int {
    FewRowsArgs a;
    a.in = in; a.W = W; a.expert = expert; a.out = out;
    a.slots = (int)N; a.choices = choices; a.k = (int)k; a.rows = (int)nrows; a.E = (int)m.E;
    a.by_slot = N < m.E;
    const dim3 g((unsigned)ceil_div(nrows, 16), (unsigned)std::min(N, m.E));
    if (k % 4 == 0 && aligned(W)) hipLaunchKernelGGL(few_rows_kernel<true>, g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(few_rows_kernel<false>, g, dim3(256), 0, s, a);
    NSH_LAUNCHED();
    return 0;
  };
  auto outer = [&](const float* A, int ca, const float* B, int cb, float* C, int64_t M, int64_t Nc) -> int {
    FewOuterArgs a;
    a.A = A; a.B = B; a.expert = expert; a.C = C;
    a.slots = (int)N; a.ca = ca; a.cb = cb; a.M = (int)M; a.N = (int)Nc;
    const bool vec = Nc % 4 == 0 && aligned(B) && aligned(C);
    a.ctiles = (int)ceil_div(Nc, vec ? 1024 : 256);
    const dim3 g((unsigned)(a.ctiles * ceil_div(M, 16)), (unsigned)m.E);
    if (vec) hipLaunchKernelGGL(few_outer_kernel<true>, g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(few_outer_kernel<false>, g, dim3(256), 0, s, a);
    NSH_LAUNCHED();
    return 0;
  };
  if (rows(dy, (int)m.K, W2, dh, m.D, m.H) != 0) return -1;
  hipLaunchKernelGGL(few_back_kernel, dim3((unsigned)ceil_div(N, 4)), dim3(256), 0, s, u, dh, hw, weight, dweight,
                     expert, (int)N, (int)m.H, act);
  NSH_LAUNCHED();
  if (dx) {
    if (rows(dh, 0, W1, slots, m.H, m.D) != 0) return -1;
    if (launch_combine(slots, expert, dx, m, s) != 0) return -1;
  }
  if (dW1 && outer(x, (int)m.K, dh, 0, dW1, m.D, m.H) != 0) return -1;
  if (dW2 && outer(hw, 0, dy, (int)m.K, dW2, m.H, m.D) != 0) return -1;
  return 0;
}

// state: the sorted slots' tables, then the pre-activations [T K, H]
size_t experts_state_bytes(const MoeShape& m) {
  if (split_takes(m)) return split_state_bytes(m);
  if (few_slots(m)) return 4 * (size_t)(round64(m.T * m.K) + m.T * m.K * m.H);
  const int64_t N = m.T * m.K;
  return 4 * (size_t)(tables_ints(N, m.E) + N * m.H);
}
// workspace: the sort's counts, the tables (no state), then of the forward
// hidden [N, H] and slots [N, D]; of the backward dh, hw [N, H], x and dy
// sorted and the slots [N, D], and the weight gradients' items and partial sums
size_t experts_workspace_bytes(const MoeShape& m, bool grad) {
  if (split_takes(m)) return split_workspace_bytes(m, grad);
  const int64_t N = m.T * m.K;
  if (few_slots(m)) {
    const int64_t fwd = round64(few_chunks(m.D, m.H, N, m.E) * N * m.H) + few_chunks(m.H, m.D, N, m.E) * N * m.D;
    return 4 * (size_t)std::max(fwd, grad ? 2 * round64(N * m.H) + N * m.D : 0);
  }
  const int64_t fwd = sort_count_ints(N, m.E) + tables_ints(N, m.E) + round64(N * m.H) + N * m.D;
  const int64_t bwd = 2 * round64(N * m.H) + 3 * round64(N * m.D) + round64(moe_bwd_kpart_floats(N, m.D, m.H)) +
                      moe_bwd_kitem_ints(N, m.D, m.H, m.E);
  return 4 * (size_t)std::max(fwd, grad ? bwd : 0);
}

int launch_experts(const float* x, const int32_t* idx, const float* weight, const float* W1, const float* W2, float* y,
                   const MoeShape& m, int act, void* state, void* workspace, hipStream_t s) {
  const int64_t N = m.T * m.K;
  if (m.T <= 0 || m.D <= 0) return 0;
  if (split_takes(m)) return launch_experts_split(x, idx, weight, W1, W2, y, m, act, state, workspace, s);
  if (few_slots(m)) return launch_few(x, idx, weight, W1, W2, y, m, act, state, workspace, s);
  int* wi = static_cast<int*>(workspace);
  int* count = wi;
  wi += sort_count_ints(N, m.E);
  int* ti = state ? static_cast<int*>(state) : wi;
  if (!state) wi += tables_ints(N, m.E);
  float* hidden = reinterpret_cast<float*>(wi);
  float* slots = hidden + round64(N * m.H);
  const SlotTables t = tables_at(ti, N, m.E);
  if (launch_sort_slots(idx, t, count, N, (int)m.K, (int)m.E, 1, 128, 0, s) != 0) return -1;
  if (small_takes(m, x, W1, W2)) {
    float* pre = state ? reinterpret_cast<float*>(ti + tables_ints(N, m.E)) : nullptr;
    if (launch_small(x, weight, W1, W2, t, pre, slots, m, act, s) != 0) return -1;
    return launch_combine(slots, t.expert, y, m, s);
  }
  GemmArgs g = grouped(t, N, m.H, m.D, x, W1, hidden, m, false);
  g.a_rows = t.tok;
  g.act = act;
  if (state) {  // the pre-activation stays for the gradient
    g.C = reinterpret_cast<float*>(ti + tables_ints(N, m.E));
    g.C2 = hidden;
  }
  if (launch_gemm_ex(g, false, false, 1, s) != 0) return -1;
  GemmArgs g2 = grouped(t, N, m.D, m.H, hidden, W2, slots, m, false);
  g2.c_rows = t.perm;
  g2.row_scale = weight;
  if (launch_gemm_ex(g2, false, false, 1, s) != 0) return -1;
  return launch_combine(slots, t.expert, y, m, s);
}

int launch_experts_grad(const float* dy, const float* x, const float* weight, const float* W1, const float* W2,
                        const void* state, float* dx, float* dweight, float* dW1, float* dW2, const MoeShape& m,
                        int act, void* workspace, hipStream_t s) {
  const int64_t N = m.T * m.K;
  if (N <= 0 || m.D <= 0) {
    if (dW1 && launch_fill(dW1, m.E * m.D * m.H, 0.f, s) != 0) return -1;
    if (dW2 && launch_fill(dW2, m.E * m.D * m.H, 0.f, s) != 0) return -1;
    return dweight ? launch_fill(dweight, N, 0.f, s) : 0;
  }
  if (split_takes(m))
    return launch_experts_split_grad(dy, x, weight, W1, W2, state, dx, dweight, dW1, dW2, m, act, workspace, s);
  if (few_slots(m)) return launch_few_grad(dy, x, weight, W1, W2, state, dx, dweight, dW1, dW2, m, act, workspace, s);
  int* ti = const_cast<int*>(static_cast<const int*>(state));
  const SlotTables t = tables_at(ti, N, m.E);
  const float* pre = reinterpret_cast<const float*>(ti + tables_ints(N, m.E));
  float* dh = static_cast<float*>(workspace);
  float* hw = dh + round64(N * m.H);
  float* xs = hw + round64(N * m.H);
  float* dys = xs + round64(N * m.D);
  float* slots = dys + round64(N * m.D);
  float* kpart = slots + round64(N * m.D);
  int* kitems = reinterpret_cast<int*>(kpart + round64(moe_bwd_kpart_floats(N, m.D, m.H)));
  const int* nrows = t.seg + m.E;
  if (dweight && launch_fill(dweight, N, 0.f, s) != 0) return -1;
  // the two products of the weights' gradients, from rows by position
  auto weight_grads = [&]() -> int {
    if (!dW1 && !dW2) return 0;
    if (launch_moe_kitems(t.seg, kitems, nullptr, N, m.D, m.H, m.E, s) != 0) return -1;
    if (dW1 && launch_moe_weight_grad(xs, dh, dW1, m.D, m.H, kitems, kpart, N, m.D, m.H, m.E, s) != 0) return -1;
    return dW2 ? launch_moe_weight_grad(hw, dys, dW2, m.H, m.D, kitems, kpart, N, m.D, m.H, m.E, s) : 0;
  };
  if (small_takes(m, dy, W1, W2) && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
    const bool rows = dW1 || dW2;
    if (launch_small_grad(dy, x, weight, W1, W2, t, pre, dh, hw, rows ? xs : nullptr, rows ? dys : nullptr, dweight,
                          dx ? slots : nullptr, m, act, s) != 0)
      return -1;
    if (dx && launch_combine(slots, t.expert, dx, m, s) != 0) return -1;
    return weight_grads();
  }
  GemmArgs g = grouped(t, N, m.H, m.D, dy, W2, dh, m, true);
  g.a_rows = t.tok;
  if (launch_gemm_ex(g, false, true, 1, s) != 0) return -1;
  hipLaunchKernelGGL(bwd_rows_kernel, dim3((unsigned)ceil_div(N, 4)), dim3(256), 0, s, pre, dh, hw, weight, dweight,
                     t.perm, nrows, (int)m.H, act);
  NSH_LAUNCHED();
  if (dx) {
    GemmArgs h = grouped(t, N, m.D, m.H, dh, W1, slots, m, true);
    h.c_rows = t.perm;
    if (launch_gemm_ex(h, false, true, 1, s) != 0) return -1;
    if (launch_combine(slots, t.expert, dx, m, s) != 0) return -1;
  }
  if (!dW1 && !dW2) return 0;
  hipLaunchKernelGGL(gather_kernel, dim3(stream_blocks(N * m.D)), dim3(256), 0, s, x, dy, t.tok, nrows, xs, dys, m.D);
  NSH_LAUNCHED();
  return weight_grads();
}

}  // namespace nship
