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
// Two ways to the products, chosen by the rows (kFewRows):
//
// Few rows (an acting step) only read the weights once: k_few takes them
// straight from memory into FP32 MFMA.
//
// Otherwise the products run on the bf16 matrix cores as FP32 products: a
// float is exactly the sum of three bf16, and of the nine products of two
// floats' parts the six largest are kept (split_gemm.hpp has the bounds and
// the reference).  Unlike the convolutions' core there, which splits operands as it
// stages them, operands are split once, by k_pack, into the very order in
// which the matrix cores take them: 16 rows x 32 k of one part are 1 KiB,
//   [block of 16 rows][step of 32 k][part][k / 8][row][8 k],
// so k_mma moves whole fragments from memory to LDS without a register and
// reads them without conflicts, and every part is split once however many
// tiles read it.  Packing writes 6 bytes a value beside the 4 read; a product
// reads each value M / 128 or N / 128 times.
#include "split_gemm.hpp"

#include <algorithm>
#include <cmath>

namespace ttrl {
namespace {

enum Act { kSilu, kGelu, kRelu, kSigmoid };

// act(g) and its derivative.
__device__ __forceinline__ float gate(int act, float g, float* slope) {
  if (act == kRelu) {
    *slope = g > 0.f ? 1.f : 0.f;
    return g > 0.f || g != g ? g : 0.f;  // NaN stays
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

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// ------------------------------------------------------------- operands ---

// What a product's operands are made of, element by element (k_mma's second
// way, and k_pack's sources).
struct Source {
  const float *x, *wg, *wu;      // (M, K), (K, N)
  const float *dh, *g, *u;       // (M, N)
  int M, K, N, act;
  int N32;                       // N in whole steps of 32
  __device__ __forceinline__ float slope_of(long m, int n, int up) const {
    const long at = m * N + n;
    float s;
    const float a = gate(act, g[at], &s);
    return up ? dh[at] * a : dh[at] * u[at] * s;
  }
};
enum Product { kForward, kInput, kWeight };
// Columns of both projections lie in blocks of 16 in turn: 16 of gate, 16 of up.
__device__ __forceinline__ int column_of(int n, int* up) {
  *up = n >> 4 & 1;
  return (n >> 5) * 16 + (n & 15);
}
__device__ float element_a(const Source& s, int product, long m, int k) {
  if (product == kForward) return m < s.M && k < s.K ? s.x[m * s.K + k] : 0.f;
  if (product == kWeight) return m < s.K && k < s.M ? s.x[long(k) * s.K + m] : 0.f;
  const int up = k >= s.N32, n = k - up * s.N32;
  return m < s.M && n < s.N ? s.slope_of(m, n, up) : 0.f;
}
__device__ float element_b(const Source& s, int product, int n, int k) {
  int up;
  if (product == kInput) {
    up = k >= s.N32;
    const int c = k - up * s.N32;
    return n < s.K && c < s.N ? (up ? s.wu : s.wg)[long(n) * s.N + c] : 0.f;
  }
  const int c = column_of(n, &up);
  if (c >= s.N) return 0.f;
  if (product == kForward) return k < s.K ? (up ? s.wu : s.wg)[long(k) * s.N + c] : 0.f;
  return k < s.M ? s.slope_of(k, c, up) : 0.f;
}

constexpr int kPart = 1024, kFrag = 3 * kPart;  // bytes of 16 x 32 values: a part, all three

// A matrix packed by rows (k along its columns) and by columns (k along its
// rows), either or both.  Block b of 16 rows, step s of 32 k is fragment
// (b * mul + add) * steps + s + first.
struct Packed {
  char* p;
  int steps, first, mul, add;
};
struct PackJob {
  const float* src;  // plain matrix (R, C), or null: both slopes of the Source
  int R, C;
  Packed rows[2], cols[2];  // of the gate and of the up slopes; a plain matrix has the first
  float* sums;              // [R / 32][2][C] column sums of the slopes, or null
  int tiles_c, block0;
};
constexpr int kJobs = 3, kPackR = 32, kPackC = 64;
struct PackArgs {
  PackJob job[kJobs];
  int jobs;
  Source s;
};

// A lane's 8 values of a fragment, split.
__device__ __forceinline__ void put_fragment(const Packed& to, int block, int step, int lane, const float (&v)[8]) {
  Planes p;
  split8<false>(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]}, p);
  char* at = to.p + (long(block * to.mul + to.add) * to.steps + step + to.first) * kFrag + lane * 16;
  *reinterpret_cast<u32x4*>(at) = p.h;
  *reinterpret_cast<u32x4*>(at + kPart) = p.m;
  *reinterpret_cast<u32x4*>(at + 2 * kPart) = p.l;
}

// A workgroup takes 32 x 64 values through LDS and writes them in both orders.
__global__ __launch_bounds__(256) void k_pack(PackArgs a) {
  constexpr int P = kPackC + 4;
  __shared__ __attribute__((aligned(16))) float tile[2][kPackR * P];
  int q = 0;
#pragma unroll
  for (int i = 1; i < kJobs; ++i)
    if (i < a.jobs && int(blockIdx.x) >= a.job[i].block0) q = i;
  const PackJob& j = a.job[q];
  const int id = int(blockIdx.x) - j.block0, tr = id / j.tiles_c, tc = id - tr * j.tiles_c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const int parts = j.src ? 1 : 2;
  for (int i = tid; i < kPackR * kPackC; i += 256) {
    const int r = i / kPackC, c = i % kPackC;
    const long row = long(tr) * kPackR + r;
    const int col = tc * kPackC + c;
    const bool in = row < j.R && col < j.C;
    const long at = row * j.C + col;
    if (j.src) {
      tile[0][r * P + c] = in ? j.src[at] : 0.f;
    } else {
      float s = 0.f, d = 0.f, act = 0.f, u = 0.f;
      if (in) {
        act = gate(a.s.act, a.s.g[at], &s);
        d = a.s.dh[at];
        u = a.s.u[at];
      }
      tile[0][r * P + c] = d * u * s;
      tile[1][r * P + c] = d * act;
    }
  }
  __syncthreads();
  for (int part = 0; part < parts; ++part) {
    const float* T = tile[part];
    // Four fragments each way: two blocks of 16 rows by two steps of columns,
    // four blocks of 16 columns by one step of rows.
    if (j.rows[part].p) {
      const int b = wave >> 1, s = wave & 1;
      if (tr * 2 + b < (j.R + 15) / 16 && tc * 2 + s < (j.C + 31) / 32) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = T[(b * 16 + lr) * P + s * 32 + lg * 8 + i];
        put_fragment(j.rows[part], tr * 2 + b, tc * 2 + s, lane, v);
      }
    }
    if (j.cols[part].p && tc * 4 + wave < (j.C + 15) / 16) {
      float v[8], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = T[(lg * 8 + i) * P + wave * 16 + lr];
      put_fragment(j.cols[part], tc * 4 + wave, tr, lane, v);
      if (j.sums) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int c = tc * kPackC + wave * 16 + lr;
        if (lg == 0 && c < j.C) j.sums[(long(tr) * 2 + part) * j.C + c] = sum;
      }
    }
  }
}

// ------------------------------------------------------------ the product ---

struct MmaArgs {
  const char *a, *b;  // packed operands
  int product;
  int M, N;                  // rows of a and of b
  int steps, per;            // steps of 32 k, of a split
  int tiles_m, tiles_n;
  float* part;               // partial sums of the splits, [split][M][N], or null
  const float *bg, *bu;      // kForward
  float *o0, *o1, *o2;       // kForward h, g, u; kInput dx; kWeight dW_gate, dW_up
  Source s;
};

// Element (m, n) of a product goes where it belongs.
struct Gated {
  float g, u;
};
__device__ __forceinline__ void put_gated(const MmaArgs& a, long m, int c, float g, float u) {
  g += a.bg ? a.bg[c] : 0.f;
  u += a.bu ? a.bu[c] : 0.f;
  const long at = m * a.s.N + c;
  float slope;
  a.o0[at] = gate(a.s.act, g, &slope) * u;
  if (a.o1) {
    a.o1[at] = g;
    a.o2[at] = u;
  }
}

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

// Tile id of the workgroup: the workgroups of an XCD (every eighth) take
// neighbouring tiles, eight tile rows by the columns in turn, so that its L2
// serves the operands that they share.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int total = tiles_m * tiles_n, each = total / 8, over = total % 8;
  const int x = id % 8, i = id / 8;
  const int t = x < over ? x * (each + 1) + i : over * (each + 1) + (x - over) * each + i;
  const int band = t / (8 * tiles_n), first = band * 8, high = min(8, tiles_m - first), in = t - band * 8 * tiles_n;
  *tm = first + in % high;
  *tn = in / high;
}

// WM x WN wavefronts of FM x FN fragments of 16 x 16.
template <int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(64 * WM * WN) void k_mma(MmaArgs a) {
  constexpr int NW = WM * WN, TA = WM * FM, TB = WN * FN, LOADS = (TA + TB) * 3 / NW;
  static_assert((TA + TB) * 3 % NW == 0, "whole fragments for every wavefront");
  __shared__ __attribute__((aligned(16))) char lds[2][(TA + TB) * kFrag];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_of(int(blockIdx.x), a.tiles_m, a.tiles_n, &tm, &tn);
  const int s0 = int(blockIdx.y) * a.per, s1 = min(a.steps, s0 + a.per);
  const long pitch = long(a.steps) * kFrag;
  // Part c of the tile's fragments: a's blocks first, then b's.
  auto load = [&](int buf, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = wave * LOADS + i, f = c / 3;
      const char* src = f < TA ? a.a + (long(tm) * TA + f) * pitch : a.b + (long(tn) * TB + f - TA) * pitch;
      src += long(s) * kFrag + (c - f * 3) * kPart + lane * 16;
      __builtin_amdgcn_global_load_lds((gvoid*)src, (lvoid*)(lds[buf] + c * kPart), 16, 0, 0);
    }
  };
  f32x4 acc[FM][FN], low[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = low[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  load(0, s0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the barrier alone does not wait for loads into LDS
  __syncthreads();
  for (int s = s0, buf = 0; s < s1; ++s, buf ^= 1) {
    const char* A = lds[buf] + wm * FM * kFrag + lane * 16;
    const char* B = lds[buf] + (TA + wn * FN) * kFrag + lane * 16;
    u32x4 pa[3][FM], pb[3][FN];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
      for (int i = 0; i < FM; ++i) pa[p][i] = *reinterpret_cast<const u32x4*>(A + i * kFrag + p * kPart);
#pragma unroll
      for (int j = 0; j < FN; ++j) pb[p][j] = *reinterpret_cast<const u32x4*>(B + j * kFrag + p * kPart);
    }
    if (s + 1 < s1) load(buf ^ 1, s + 1);  // after the reads, which need not wait for it
    // The products of the lower parts have sums of their own, so the main sum
    // is rounded once per 32 k.
    auto mul = [&](f32x4 (&d)[FM][FN], int x, int y) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) d[i][j] = mfma_bf16(pa[x][i], pb[y][j], d[i][j]);
    };
    mul(acc, 0, 0);
    mul(low, 0, 1);
    mul(low, 1, 0);
    mul(low, 1, 1);
    mul(low, 0, 2);
    mul(low, 2, 0);
    __builtin_amdgcn_sched_barrier(0);  // the products first: they cover the loads
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

  // Infinities, NaN and operands near the ends of the range do not survive
  // the split (see split_gemm.hpp): such elements, and rows with no sum of
  // kSplitTiny among the wavefront's columns, are formed again in FP32.  Each
  // goes by its own row, so no row's bits depend on another row.
  const long mw = (long(tm) * TA + wm * FM) * 16;
  const int nw = (tn * TB + wn * FN) * 16;
  bool again = false;
  uint32_t tiny = 0;  // bit 4 i + r: row r of fragments i
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        float v = acc[i][j][r] += low[i][j][r];
        if (mw + i * 16 + 4 * lg + r >= a.M || nw + j * 16 + lr >= a.N) v = 0.f;  // rows nobody packed
        again = again || !__builtin_isfinite(v);
        top = fmaxf(top, fabsf(v));
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
      tiny |= uint32_t(top > 0.f && top < kSplitTiny) << (4 * i + r);
    }
  if (__any(again || tiny)) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) low[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int k = s0 * 32; k < s1 * 32; k += 4) {
      float ea[FM], eb[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) ea[i] = element_a(a.s, a.product, mw + i * 16 + lr, k + lg);
#pragma unroll
      for (int j = 0; j < FN; ++j) eb[j] = element_b(a.s, a.product, nw + j * 16 + lr, k + lg);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) low[i][j] = mfma_f32(ea[i], eb[j], low[i][j]);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!__builtin_isfinite(acc[i][j][r]) || (tiny >> (4 * i + r) & 1)) acc[i][j][r] = low[i][j][r];
  }

#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long m = mw + i * 16 + 4 * lg + r;
      if (m >= a.M) continue;
      if (a.part) {
        float* to = a.part + (long(blockIdx.y) * a.M + m) * a.N;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int n = nw + j * 16 + lr;
          if (n < a.N) to[n] = acc[i][j][r];
        }
      } else if (a.product == kInput) {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int n = nw + j * 16 + lr;
          if (n < a.N) a.o0[m * a.N + n] = acc[i][j][r];
        }
      } else {
#pragma unroll
        for (int j = 0; j < FN; j += 2) {
          const int c = (nw + j * 16) / 2 + lr;
          if (c >= a.s.N) continue;
          if (a.product == kForward) {
            put_gated(a, m, c, acc[i][j][r], acc[i][j + 1][r]);
          } else {
            if (a.o0) a.o0[m * a.s.N + c] = acc[i][j][r];
            if (a.o1) a.o1[m * a.s.N + c] = acc[i][j + 1][r];
          }
        }
      }
    }
}

// The splits' sums, in order, and what follows them.
__global__ __launch_bounds__(256) void k_splits(MmaArgs a, int splits) {
  const long total = long(a.M) * a.N, half = long(a.M) * a.s.N;
  const long count = a.product == kInput ? total : half;
  for (long i = long(blockIdx.x) * 256 + threadIdx.x; i < count; i += long(gridDim.x) * 256) {
    if (a.product == kInput) {
      float t = 0.f;
      for (int s = 0; s < splits; ++s) t += a.part[s * total + i];
      a.o0[i] = t;
      continue;
    }
    const long m = i / a.s.N;
    const int c = int(i - m * a.s.N);
    const long at = m * a.N + (c >> 4) * 32 + (c & 15);
    float g = 0.f, u = 0.f;
    for (int s = 0; s < splits; ++s) {
      g += a.part[s * total + at];
      u += a.part[s * total + at + 16];
    }
    if (a.product == kForward) {
      put_gated(a, m, c, g, u);
    } else {
      if (a.o0) a.o0[i] = g;
      if (a.o1) a.o1[i] = u;
    }
  }
}

// Bias gradients: the column sums of every 32 rows, in order.
__global__ __launch_bounds__(256) void k_bias(const float* __restrict__ sums, int tiles, int N, float* __restrict__ db_gate,
                                              float* __restrict__ db_up) {
  __shared__ double red[256];
  const int c = int(blockIdx.x) * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
  double t = 0.0;
  if (c < 2 * N)
    for (int i = q; i < tiles; i += 16) t += double(sums[long(i) * 2 * N + c]);
  red[threadIdx.x] = t;
  __syncthreads();
  if (q || c >= 2 * N) return;
  for (int i = 1; i < 16; ++i) t += red[i * 16 + threadIdx.x];
  float* to = c < N ? db_gate : db_up;
  if (to) to[c < N ? c : c - N] = float(t);
}

// ------------------------------------------------------------- few rows ---

// 16 columns of both projections and up to 16 RB rows: the weights go from
// memory into the products' registers, the wavefronts share K and their sums
// meet in LDS, in order.  XV: x in whole 16-byte rows.
struct FewArgs {
  const float *x, *wg, *wu;
  MmaArgs out;
};
constexpr int kFewWaves = 8;
__device__ __forceinline__ float at_or_zero(__amdgpu_buffer_rsrc_t r, uint32_t off) { return ld_f1(r, off); }

template <int RB, bool XV>
__global__ __launch_bounds__(64 * kFewWaves) void k_few(FewArgs a) {
  __shared__ float part[kFewWaves][2 * RB * 256];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = a.out.s.M, K = a.out.s.K, N = a.out.s.N, n = int(blockIdx.x) * 16 + lr;
  const __amdgpu_buffer_rsrc_t rx = make_res(a.x, uint32_t(M) * uint32_t(K) * 4u);
  const uint32_t bytes = uint32_t(K) * uint32_t(N) * 4u;
  const __amdgpu_buffer_rsrc_t rg = make_res(a.wg, bytes), ru = make_res(a.wu, bytes);
  const int blocks = (K + 15) / 16, per = (blocks + kFewWaves - 1) / kFewWaves;
  f32x4 acc[2][RB];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int DEEP = 4;  // blocks of 16 k in flight
  const int first = wave * per, last = min(blocks, first + per);
  for (int k0 = first; k0 < last; k0 += DEEP) {
    float w[2][DEEP][4];
    f32x4 x[DEEP][RB];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int k = (k0 + d) * 16 + 4 * lg;
      const bool in = k0 + d < last;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t off = in && k + r < K && n < N ? (uint32_t(k + r) * uint32_t(N) + uint32_t(n)) * 4u : ~0u;
        w[0][d][r] = at_or_zero(rg, off);
        w[1][d][r] = at_or_zero(ru, off);
      }
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const int m = b * 16 + lr;
        if constexpr (XV) {
          x[d][b] = ld_f4(rx, in && m < M && k < K ? (uint32_t(m) * uint32_t(K) + uint32_t(k)) * 4u : ~0u - 15u);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[d][b][r] = at_or_zero(rx, in && m < M && k + r < K ? (uint32_t(m) * uint32_t(K) + uint32_t(k + r)) * 4u : ~0u);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
          for (int q = 0; q < 2; ++q) acc[q][b] = mfma_f32(x[d][b][r], w[q][d][r], acc[q][b]);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[wave][(q * RB + b) * 256 + (4 * lg + r) * 16 + lr] = acc[q][b][r];
  __syncthreads();
  for (int i = tid; i < RB * 256; i += 64 * kFewWaves) {
    const int m = i >> 4, c = int(blockIdx.x) * 16 + (i & 15);
    if (m >= M || c >= N) continue;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      g += part[w][i];
      u += part[w][RB * 256 + i];
    }
    put_gated(a.out, m, c, g, u);
  }
}

// ------------------------------------------------------------------ host ---

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
long up_to(long n, long q) { return (n + q - 1) / q * q; }

// Rows that read the weights as they are: beyond, packing them pays.
constexpr int kFewRows = 32;

// A product's tiles and splits: 128 x 128 where they fill the compute units
// (or nearly), else 64 x 64, and k in splits while there are fewer workgroups
// than two a compute unit and a split keeps kMinSteps steps.
constexpr int kMinSteps = 6;
struct MmaPlan {
  bool big;
  int tiles_m, tiles_n, splits, per;
};
MmaPlan plan_mma(long M, long N, long steps) {
  MmaPlan p{};
  p.big = ((M + 127) / 128) * ((N + 127) / 128) >= 192;
  const int t = p.big ? 128 : 64;
  p.tiles_m = int((M + t - 1) / t);
  p.tiles_n = int((N + t - 1) / t);
  const long tiles = long(p.tiles_m) * p.tiles_n, want = p.big ? 256 : 512;
  long splits = tiles >= want / 2 ? 1 : std::min((want + tiles - 1) / tiles, std::max(1L, steps / kMinSteps));
  splits = std::min(splits, 64L);
  p.per = int((steps + splits - 1) / splits);
  p.splits = int((steps + p.per - 1) / p.per);
  return p;
}

// One product: its packed operands and partial sums in the workspace.
struct Layout {
  long a, b, part;  // bytes
  MmaPlan plan;
  long rows_a, rows_b;
  int steps;
};
Layout layout_of(long M, long N, long steps) {
  Layout l{};
  l.plan = plan_mma(M, N, steps);
  l.rows_a = M;
  l.rows_b = N;
  l.steps = int(steps);
  l.a = up_to(M, 128) / 16 * steps * kFrag;
  l.b = up_to(N, 128) / 16 * steps * kFrag;
  l.part = l.plan.splits > 1 ? up_to(long(l.plan.splits) * M * N * 4, 256) : 0;
  return l;
}
struct Layouts {
  Layout fwd, dx, dw;
  long sums;
};
Layouts layouts_of(const ttrl_gated_desc* d) {
  const long rows = std::max(1, d->M), both = up_to(d->N, 16) * 2, n32 = (d->N + 31) / 32;
  Layouts l;
  l.fwd = layout_of(rows, both, (d->K + 31) / 32);
  l.dx = layout_of(rows, d->K, 2 * n32);
  l.dw = layout_of(d->K, both, (rows + 31) / 32);
  l.sums = up_to((rows + 31) / 32 * 2 * d->N * 4, 256);
  return l;
}

Source source_of(const ttrl_gated_desc* d) {
  return Source{d->x, d->w_gate, d->w_up, d->dh, d->g, d->u, d->M, d->K, d->N, d->act, int(up_to(d->N, 32))};
}

int check_gated(const ttrl_gated_desc* d, const char* name) {
  TTRL_REQUIRE(d, "%s: null description", name);
  TTRL_REQUIRE(d->M >= 0 && d->K > 0 && d->N > 0, "%s: bad extents M=%d, K=%d, N=%d", name, d->M, d->K, d->N);
  TTRL_REQUIRE(d->act >= 0 && d->act <= kSigmoid, "%s: unknown activation %d", name, d->act);
  const long most = 1L << 29;
  TTRL_REQUIRE(long(d->M) * d->K < most && long(d->K) * d->N < most && long(d->M) * d->N < most,
               "%s: operands of 2^29 values or more (M=%d, K=%d, N=%d)", name, d->M, d->K, d->N);
  return TTRL_OK;
}

int launch_pack(ttrl_ctx* ctx, PackArgs& a, const char* name) {
  long blocks = 0;
  for (int i = 0; i < a.jobs; ++i) {
    PackJob& j = a.job[i];
    j.tiles_c = int((j.C + kPackC - 1) / kPackC);
    j.block0 = int(blocks);
    blocks += long(j.tiles_c) * ((j.R + kPackR - 1) / kPackR);
  }
  hipLaunchKernelGGL(k_pack, dim3(unsigned(blocks)), dim3(256), 0, stream_of(ctx), a);
  return check_launch(name);
}

int launch_mma(ttrl_ctx* ctx, MmaArgs& a, const Layout& l, float* part, const char* name) {
  a.M = int(l.rows_a);
  a.N = int(l.rows_b);
  a.steps = l.steps;
  a.per = l.plan.per;
  a.tiles_m = l.plan.tiles_m;
  a.tiles_n = l.plan.tiles_n;
  a.part = l.plan.splits > 1 ? part : nullptr;
  const dim3 grid(unsigned(a.tiles_m) * unsigned(a.tiles_n), unsigned(l.plan.splits));
  if (l.plan.big) hipLaunchKernelGGL((k_mma<2, 2, 4, 4>), grid, dim3(256), 0, stream_of(ctx), a);
  else hipLaunchKernelGGL((k_mma<2, 2, 2, 2>), grid, dim3(256), 0, stream_of(ctx), a);
  if (int rc = check_launch(name)) return rc;
  if (!a.part) return TTRL_OK;
  const long count = long(a.M) * (a.product == kInput ? a.N : a.s.N);
  hipLaunchKernelGGL(k_splits, dim3(unsigned(std::min(2048L, (count + 255) / 256))), dim3(256), 0, stream_of(ctx), a,
                     l.plan.splits);
  return check_launch(name);
}

}  // namespace
}  // namespace ttrl

using namespace ttrl;

extern "C" {

int ttrl_gated_space(const ttrl_gated_desc* d, long* forward_bytes, long* backward_bytes) {
  if (int rc = check_gated(d, "ttrl_gated_space")) return rc;
  TTRL_REQUIRE(forward_bytes && backward_bytes, "ttrl_gated_space: null output");
  const Layouts l = layouts_of(d);
  *forward_bytes = d->M <= kFewRows ? 0 : l.fwd.a + l.fwd.b + l.fwd.part;
  *backward_bytes = l.dx.a + l.dx.b + l.dw.a + l.dw.b + std::max(l.dx.part, l.dw.part) + l.sums;
  return TTRL_OK;
}

int ttrl_gated_forward(ttrl_ctx* ctx, const ttrl_gated_desc* d) {
  const char* name = "ttrl_gated_forward";
  if (int rc = check_gated(d, name)) return rc;
  TTRL_REQUIRE(ctx, "%s: null context", name);
  if (d->M == 0) return TTRL_OK;
  TTRL_REQUIRE(d->x && d->w_gate && d->w_up && d->h, "%s: null operand", name);
  TTRL_REQUIRE(!d->g == !d->u, "%s: g and u are kept together", name);
  MmaArgs m{};
  m.product = kForward;
  m.bg = d->b_gate;
  m.bu = d->b_up;
  m.o0 = d->h;
  m.o1 = d->g;
  m.o2 = d->u;
  m.s = source_of(d);
  if (d->M <= kFewRows) {
    const FewArgs f{d->x, d->w_gate, d->w_up, m};
    const dim3 grid(ceil_div(d->N, 16)), block(64 * kFewWaves);
    const bool xv = d->K % 4 == 0 && aligned16(d->x);
    auto go = [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      if (xv) hipLaunchKernelGGL((k_few<RB, true>), grid, block, 0, stream_of(ctx), f);
      else hipLaunchKernelGGL((k_few<RB, false>), grid, block, 0, stream_of(ctx), f);
    };
    if (d->M <= 16) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
    return check_launch(name);
  }
  TTRL_REQUIRE(d->work && aligned16(d->work), "%s: null or unaligned workspace", name);
  const Layout l = layouts_of(d).fwd;
  char *pa = static_cast<char*>(d->work), *pb = pa + l.a;
  PackArgs p{};
  p.s = m.s;
  p.jobs = 3;
  p.job[0] = PackJob{d->x, d->M, d->K};
  p.job[0].rows[0] = Packed{pa, l.steps, 0, 1, 0};
  for (int q = 0; q < 2; ++q) {
    p.job[1 + q] = PackJob{q ? d->w_up : d->w_gate, d->K, d->N};
    p.job[1 + q].cols[0] = Packed{pb, l.steps, 0, 2, q};
  }
  if (int rc = launch_pack(ctx, p, name)) return rc;
  m.a = pa;
  m.b = pb;
  return launch_mma(ctx, m, l, reinterpret_cast<float*>(pb + l.b), name);
}

int ttrl_gated_backward(ttrl_ctx* ctx, const ttrl_gated_desc* d) {
  const char* name = "ttrl_gated_backward";
  if (int rc = check_gated(d, name)) return rc;
  TTRL_REQUIRE(ctx, "%s: null context", name);
  if (d->M == 0) {
    const long n = d->N, w = long(d->K) * n;
    if (d->dw_gate)
      if (int rc = ttrl_fill_f32(ctx, d->dw_gate, 0.f, w)) return rc;
    if (d->dw_up)
      if (int rc = ttrl_fill_f32(ctx, d->dw_up, 0.f, w)) return rc;
    if (d->db_gate)
      if (int rc = ttrl_fill_f32(ctx, d->db_gate, 0.f, n)) return rc;
    if (d->db_up)
      if (int rc = ttrl_fill_f32(ctx, d->db_up, 0.f, n)) return rc;
    return TTRL_OK;
  }
  TTRL_REQUIRE(d->x && d->w_gate && d->w_up && d->g && d->u && d->dh, "%s: null operand", name);
  TTRL_REQUIRE(d->work && aligned16(d->work), "%s: null or unaligned workspace", name);
  const Layouts l = layouts_of(d);
  const bool dw = d->dw_gate || d->dw_up, db = d->db_gate || d->db_up;
  char *dxa = static_cast<char*>(d->work), *dxb = dxa + l.dx.a, *dwa = dxb + l.dx.b, *dwb = dwa + l.dw.a;
  float* part = reinterpret_cast<float*>(dwb + l.dw.b);
  float* sums = reinterpret_cast<float*>(dwb + l.dw.b + std::max(l.dx.part, l.dw.part));
  const int n32 = (d->N + 31) / 32;
  const Source s = source_of(d);
  PackArgs p{};
  p.s = s;
  PackJob& slopes = p.job[p.jobs++];
  slopes = PackJob{nullptr, d->M, d->N};
  for (int q = 0; q < 2; ++q) {
    if (d->dx) slopes.rows[q] = Packed{dxa, l.dx.steps, q * n32, 1, 0};
    if (dw || db) slopes.cols[q] = Packed{dwb, l.dw.steps, 0, 2, q};
  }
  slopes.sums = db ? sums : nullptr;
  if (dw) {
    PackJob& x = p.job[p.jobs++];
    x = PackJob{d->x, d->M, d->K};
    x.cols[0] = Packed{dwa, l.dw.steps, 0, 1, 0};
  }
  if (int rc = launch_pack(ctx, p, name)) return rc;
  if (d->dx) {
    PackArgs w{};
    w.s = s;
    w.jobs = 2;
    for (int q = 0; q < 2; ++q) {
      w.job[q] = PackJob{q ? d->w_up : d->w_gate, d->K, d->N};
      w.job[q].rows[0] = Packed{dxb, l.dx.steps, q * n32, 1, 0};
    }
    if (int rc = launch_pack(ctx, w, name)) return rc;
    MmaArgs m{};
    m.a = dxa;
    m.b = dxb;
    m.product = kInput;
    m.o0 = d->dx;
    m.s = s;
    if (int rc = launch_mma(ctx, m, l.dx, part, name)) return rc;
  }
  if (dw) {
    MmaArgs m{};
    m.a = dwa;
    m.b = dwb;
    m.product = kWeight;
    m.o0 = d->dw_gate;
    m.o1 = d->dw_up;
    m.s = s;
    if (int rc = launch_mma(ctx, m, l.dw, part, name)) return rc;
  }
  if (db) {
    hipLaunchKernelGGL(k_bias, dim3(ceil_div(2L * d->N, 16)), dim3(256), 0, stream_of(ctx), sums, (d->M + 31) / 32, d->N,
                       d->db_gate, d->db_up);
    if (int rc = check_launch(name)) return rc;
  }
  return TTRL_OK;
}

}  // extern "C"
