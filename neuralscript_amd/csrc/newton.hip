// Newton-Schulz orthogonalisation of n matrices [r, c], and the Muon step that
// takes its update from it.
//
//   X = G / (|G|_F + 1e-7);  steps times: A = X X^T, X = a X + (b A + c A A) X
//
// with X held wide ([m, N], m = min(r, c) <= N): each product drives every
// singular value s in (0, 1] through a s + b s^3 + c s^5, which in five steps
// ends between about 0.7 and 1.2 for all but the smallest.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace nship {
namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr double kNsEps = 1e-7;
constexpr int kNormParts = 64;  // partial sums of a matrix's norm

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
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (int64_t)gridDim.x * 256) {
    float u = g[base + i];
    if (m) {
      const float mm = mu * m[base + i] + u;
      m[base + i] = mm;
      u = update_of(u, mm, mu, nesterov);
    }
    sum += (double)u * u;
  }
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)blockIdx.y * kNormParts + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// X [m, N] = the update over its norm, transposed where r > c.
__global__ __launch_bounds__(256) void ns_start_kernel(const float* __restrict__ g, const float* __restrict__ m,
                                                       float mu, int nesterov, int64_t r, int64_t c, int parts,
                                                       const double* __restrict__ part, float* __restrict__ X) {
  const int64_t elems = r * c, base = (int64_t)blockIdx.y * elems;
  double sq = 0.;
  for (int p = 0; p < parts; p++) sq += part[(int64_t)blockIdx.y * kNormParts + p];
  const double by = 1. / (sqrt(sq) + kNsEps);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (int64_t)gridDim.x * 256) {
    float u = g[base + i];
    if (m) u = update_of(u, m[base + i], mu, nesterov);
    const int64_t row = i / c, col = i - row * c;
    X[base + (r > c ? col * r + row : i)] = (float)(u * by);
  }
}

// P = a I + b A + c P
__global__ __launch_bounds__(256) void ns_poly_kernel(const float* __restrict__ A, float* __restrict__ P, int64_t m) {
  const int64_t elems = m * m, base = (int64_t)blockIdx.y * elems;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (int64_t)gridDim.x * 256)
    P[base + i] = (i / m == i % m ? kNsA : 0.f) + kNsB * A[base + i] + kNsC * P[base + i];
}

__global__ __launch_bounds__(256) void ns_end_kernel(const float* __restrict__ X, float* __restrict__ q,
                                                     float* __restrict__ w, float le, float decay, int64_t r,
                                                     int64_t c) {
  const int64_t elems = r * c, base = (int64_t)blockIdx.y * elems;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / c, col = i - row * c;
    const float x = X[base + (r > c ? col * r + row : i)];
    if (w) w[base + i] = w[base + i] - le * x - decay * w[base + i];
    else q[base + i] = x;
  }
}

constexpr int64_t round64(int64_t n) { return (n + 63) / 64 * 64; }

}  // namespace

// the norms' partial sums, X twice, A and P
size_t newton_schulz_bytes(int64_t n, int64_t r, int64_t c) {
  const int64_t m = std::min(r, c);
  return (size_t)n * kNormParts * 8 + 4 * (size_t)(2 * round64(n * r * c) + 2 * round64(n * m * m));
}

int launch_newton_schulz(const float* g, float* q, const MuonNs* step, int64_t n, int64_t r, int64_t c, int steps,
                         void* workspace, hipStream_t s) {
  const int64_t m = std::min(r, c), N = std::max(r, c), elems = r * c;
  if (n <= 0 || elems <= 0) return 0;
  double* part = static_cast<double*>(workspace);
  float* X = reinterpret_cast<float*>(part + n * kNormParts);
  float* Y = X + round64(n * elems);
  float* A = Y + round64(n * elems);
  float* P = A + round64(n * m * m);
  const int parts = (int)std::min<int64_t>(kNormParts, ceil_div(elems, 1024));
  float* mom = step ? step->m : nullptr;
  const float mu = step ? step->mu : 0.f;
  const int nesterov = step ? step->nesterov : 0;
  const dim3 all((unsigned)std::min<int64_t>(ceil_div(elems, 1024), 4096), (unsigned)n);
  hipLaunchKernelGGL(ns_norm_kernel, dim3(parts, (unsigned)n), dim3(256), 0, s, g, mom, mu, nesterov, elems, part);
  NSH_LAUNCHED();
  hipLaunchKernelGGL(ns_start_kernel, all, dim3(256), 0, s, g, mom, mu, nesterov, r, c, parts, part, X);
  NSH_LAUNCHED();
  for (int k = 0; k < steps; k++) {
    GemmArgs a;
    a.A = X; a.B = X; a.C = A;
    a.M = (int)m; a.N = (int)m; a.K = (int)N;
    a.lda = N; a.ldb = N; a.ldc = m;
    a.sA = elems; a.sB = elems; a.sC = m * m;
    if (launch_gemm_ex(a, false, true, (int)n, s) != 0) return -1;
    GemmArgs p;
    p.A = A; p.B = A; p.C = P;
    p.M = (int)m; p.N = (int)m; p.K = (int)m;
    p.lda = m; p.ldb = m; p.ldc = m;
    p.sA = m * m; p.sB = m * m; p.sC = m * m;
    if (launch_gemm_ex(p, false, false, (int)n, s) != 0) return -1;
    hipLaunchKernelGGL(ns_poly_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(m * m, 1024), 4096), (unsigned)n),
                       dim3(256), 0, s, A, P, m);
    NSH_LAUNCHED();
    GemmArgs x;
    x.A = P; x.B = X; x.C = Y;
    x.M = (int)m; x.N = (int)N; x.K = (int)m;
    x.lda = m; x.ldb = N; x.ldc = N;
    x.sA = m * m; x.sB = elems; x.sC = elems;
    if (launch_gemm_ex(x, false, false, (int)n, s) != 0) return -1;
    std::swap(X, Y);
  }
  hipLaunchKernelGGL(ns_end_kernel, all, dim3(256), 0, s, X, q, step ? step->w : nullptr, step ? step->le : 0.f,
                     step ? step->decay : 0.f, r, c);
  NSH_LAUNCHED();
  return 0;
}

}  // namespace nship
