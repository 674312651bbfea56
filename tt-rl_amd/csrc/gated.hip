// The gated projections of a feed-forward block,
//
//   h = act(x W_gate + b_gate) * (x W_up + b_up),
//
// both products, the activation and the product of the two in one kernel, and
// their gradients.  x is (M, K), the weights (K, N), the biases N or null.
//
//   du = dh * act(g),  dg = dh * u * act'(g)
//   dx = dg W_gate^T + du W_up^T,  dW = x^T d.,  db = column sums of d.
//
// k_gated: a workgroup of four wavefronts owns 64 rows by 64 columns of both
// products, so that one lane ends with the same elements of g and of u and the
// epilogue needs no exchange; FP32 MFMA, operands staged 32 deep through LDS
// with the next stage's loads in flight.
#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace ttrl {
namespace {

enum Act { kSilu, kGelu, kRelu, kSigmoid };

// act(g) and its derivative.
__device__ __forceinline__ float gate(int act, float g, float* slope) {
  if (act == kRelu) {
    *slope = g > 0.f ? 1.f : 0.f;
    return g > 0.f ? g : g * 0.f;  // NaN stays
  }
  if (act == kGelu) {
    const float half = 0.5f * (1.f + erff(g * 0.70710678f));
    *slope = half + g * expf(-0.5f * g * g) * 0.39894228f;
    return g * half;
  }
  const float s = 1.f / (1.f + expf(-g));
  if (act == kSigmoid) {
    *slope = s * (1.f - s);
    return s;
  }
  *slope = s * (1.f + g * (1.f - s));
  return g * s;
}

__device__ __forceinline__ f32x4 mfma4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

struct GatedArgs {
  const float *x, *wg, *wu, *bg, *bu;
  float *g, *u, *h;  // g and u null when nobody reads them
  int M, K, N, act;
};

constexpr int kBM = 64, kBN = 64, kBK = 32;

template <int W>
__device__ __forceinline__ void fetch(const float* p, bool in, float (&f)[W]) {
  if constexpr (W == 4) {
    const f32x4 v = in ? *reinterpret_cast<const f32x4*>(p) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = v[j];
  } else {
    f[0] = in ? *p : 0.f;
  }
}

// W: floats a load (4: K and N multiples of 4, operands on 16 bytes).
template <int W>
__global__ __launch_bounds__(256) void k_gated(GatedArgs a) {
  constexpr int PA = kBK + 4, PB = kBN + 4, NA = kBM * kBK / W / 256, NB = kBK * kBN / W / 256;
  __shared__ __attribute__((aligned(16))) float la[kBM * PA];
  __shared__ __attribute__((aligned(16))) float lb[2][kBK * PB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const long m0 = long(blockIdx.x) * kBM;
  const int n0 = int(blockIdx.y) * kBN;
  float fa[NA][W], fb[2][NB][W];
  auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < NA; ++u) {
      const int i = tid + u * 256, r = i / (kBK / W), c = i % (kBK / W) * W;
      fetch(a.x + (m0 + r) * a.K + k0 + c, m0 + r < a.M && k0 + c < a.K, fa[u]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int i = tid + u * 256, r = i / (kBN / W), c = i % (kBN / W) * W;
        fetch((q ? a.wu : a.wg) + long(k0 + r) * a.N + n0 + c, k0 + r < a.K && n0 + c < a.N, fb[q][u]);
      }
  };
  f32x4 acc[2][4];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  load(0);
  for (int k0 = 0; k0 < a.K; k0 += kBK) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NA; ++u) {
      const int i = tid + u * 256, r = i / (kBK / W), c = i % (kBK / W) * W;
#pragma unroll
      for (int j = 0; j < W; ++j) la[r * PA + c + j] = fa[u][j];
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int i = tid + u * 256, r = i / (kBN / W), c = i % (kBN / W) * W;
#pragma unroll
        for (int j = 0; j < W; ++j) lb[q][r * PB + c + j] = fb[q][u][j];
      }
    __syncthreads();
    if (k0 + kBK < a.K) load(k0 + kBK);
#pragma unroll
    for (int kb = 0; kb < kBK / 16; ++kb) {
      const f32x4 xa = *reinterpret_cast<const f32x4*>(la + (wave * 16 + lr) * PA + kb * 16 + 4 * lg);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[q][j] = mfma4(xa[r], lb[q][(kb * 16 + 4 * lg + r) * PB + j * 16 + lr], acc[q][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + j * 16 + lr;
    if (n >= a.N) continue;
    const float bg = a.bg ? a.bg[n] : 0.f, bu = a.bu ? a.bu[n] : 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long m = m0 + wave * 16 + 4 * lg + r;
      if (m >= a.M) continue;
      const float g = acc[0][j][r] + bg, u = acc[1][j][r] + bu;
      float slope;
      const long at = m * a.N + n;
      if (a.g) {
        a.g[at] = g;
        a.u[at] = u;
      }
      a.h[at] = gate(a.act, g, &slope) * u;
    }
  }
}

// dg and du from dh, g and u.
__global__ __launch_bounds__(256) void k_gated_slopes(const float* __restrict__ dh, const float* __restrict__ g,
                                                      const float* __restrict__ u, float* __restrict__ dg,
                                                      float* __restrict__ du, long n, int act) {
  for (long i = long(blockIdx.x) * 256 + threadIdx.x; i < n; i += long(gridDim.x) * 256) {
    float slope;
    const float d = dh[i], a = gate(act, g[i], &slope);
    dg[i] = d * u[i] * slope;
    du[i] = d * a;
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_gated(const ttrl_gated_desc* d, const char* name) {
  TTRL_REQUIRE(d, "%s: null description", name);
  TTRL_REQUIRE(d->M >= 0 && d->K > 0 && d->N > 0, "%s: bad extents M=%d, K=%d, N=%d", name, d->M, d->K, d->N);
  TTRL_REQUIRE(d->act >= 0 && d->act <= kSigmoid, "%s: unknown activation %d", name, d->act);
  TTRL_REQUIRE(d->M <= 64 * 0x7fffffL && d->N <= 64 * 65535, "%s: too large", name);
  return TTRL_OK;
}

}  // namespace
}  // namespace ttrl

using namespace ttrl;

extern "C" {

int ttrl_gated_forward(ttrl_ctx* ctx, const ttrl_gated_desc* d) {
  const char* name = "ttrl_gated_forward";
  if (int rc = check_gated(d, name)) return rc;
  TTRL_REQUIRE(ctx, "%s: null context", name);
  if (d->M == 0) return TTRL_OK;
  TTRL_REQUIRE(d->x && d->w_gate && d->w_up && d->h, "%s: null operand", name);
  TTRL_REQUIRE(!d->g == !d->u, "%s: g and u are kept together", name);
  const GatedArgs a{d->x, d->w_gate, d->w_up, d->b_gate, d->b_up, d->g, d->u, d->h, d->M, d->K, d->N, d->act};
  const dim3 grid(ceil_div(d->M, kBM), ceil_div(d->N, kBN));
  if (d->K % 4 == 0 && d->N % 4 == 0 && aligned16(d->x) && aligned16(d->w_gate) && aligned16(d->w_up))
    hipLaunchKernelGGL(k_gated<4>, grid, dim3(256), 0, stream_of(ctx), a);
  else
    hipLaunchKernelGGL(k_gated<1>, grid, dim3(256), 0, stream_of(ctx), a);
  return check_launch(name);
}

int ttrl_gated_slopes(ttrl_ctx* ctx, int M, int N, int act, const float* dh, const float* g, const float* u, float* dg,
                      float* du) {
  TTRL_REQUIRE(ctx, "ttrl_gated_slopes: null context");
  TTRL_REQUIRE(M >= 0 && N > 0 && act >= 0 && act <= kSigmoid, "ttrl_gated_slopes: bad extents or activation");
  if (M == 0) return TTRL_OK;
  TTRL_REQUIRE(dh && g && u && dg && du, "ttrl_gated_slopes: null operand");
  const long n = long(M) * N;
  hipLaunchKernelGGL(k_gated_slopes, dim3(unsigned(std::min(8192L, (n + 255) / 256))), dim3(256), 0, stream_of(ctx), dh,
                     g, u, dg, du, n, act);
  return check_launch("ttrl_gated_slopes");
}

}  // extern "C"
