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
// Two ways to the forward products, chosen by their work (kFewWork):
//
// Small ones (an acting step) read the weights straight from memory into FP32
// MFMA, in one launch (k_few).
//
// Otherwise the products run on the fp16 matrix cores.  Every row of an operand
// (the values that one output sums over) is scaled by a power of two, so that
// its largest value lies in [2^14, 2^15), and each value v is split into
//
//   h = v to the nearest fp16,  l = v - h to the nearest fp16,
//
// 11 significant bits each, of either sign: v - h - l is at most 2^-23 of v's
// power of two.  Of the four products of two values' parts hh, hl and lh are
// kept; ll is at most 2^-22 of the product, of either sign.  Together a product
// is off by 2^-21 at worst and 2^-24 in the mean, as one rounding of FP32 is;
// every partial product is exact in FP32 and added in FP32, the sum rounded
// three times per 32 k.  (Error against float64 at 8192 x 1024 x 4096: 1.1e-6 of
// a gradient's norm, a library's FP32 products 1.7e-6.)  fp16 ends at 2^-24, so a
// value under 2^-2 (2^-16 of its row's largest) is off by up to 2^-25 instead;
// such values are counted by row, and every sum in which they could show (doubt()
// and lossy_sums() below), or that is not finite, is formed again in FP32.  So a
// sum is off by 2^-21 + 2^-22 of its terms' absolute values at most, beside FP32's
// own rounding.
//
// (Three bf16 parts, 24 bits at any exponent, need six products and no scale:
// the forward and backward pass of 8192 x 1024 x 4096 took 2651 us so, 1546
// with two fp16 parts in the same tiles, and 1424 to 1441 as it stands, 30 of
// them for the guard against small values.)
//
// Operands are split once, by k_pack, into the very order in which the matrix
// cores take them: 16 rows x 32 k of one part are 1 KiB,
//   [block of 16 rows][step of 32 k][part][k / 8][row][8 k],
// so k_mma moves whole fragments from memory to LDS without a register and
// reads them without conflicts, and every value is split once however many
// tiles read it.  The scales cost one more pass over what is packed (k_scan);
// packing writes 4 bytes a value beside the 4 read.  Where the time of that pass
// goes (us): forward scan 13, pack 25, product 439; backward scan 117, pack 268
// (1.1 GB, 4 TB/s), both products 603.
#include "tile_gemm.hpp"

#include <algorithm>
#include <cmath>

namespace ttrl {
namespace {

enum Act { kSilu, kGelu, kRelu, kSigmoid, kNone };

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

// What a product's operands are made of (k_pack's sources, and those of sums
// that are formed again).
struct Source {
  const float *x, *wg, *wu;      // (M, K), (K, N)
  const float *dh, *g, *u;       // (M, N)
  int M, K, N, act;
  int N32;                       // N in whole steps of 32
};
enum Product { kForward, kInput, kWeight };
// Columns of both projections lie in blocks of 16 in turn: 16 of gate, 16 of up.
__device__ __forceinline__ int column_of(int n, int* up) {
  *up = n >> 4 & 1;
  return (n >> 5) * 16 + (n & 15);
}

constexpr int kParts = 2, kPart = 1024, kFrag = kParts * kPart;  // bytes of 16 x 32 values: a part, both

// What is known of a packed row.
struct __attribute__((aligned(16))) Row {
  int scale;  // the exponent of the largest value less 14
  int small;  // values that fp16 ends above: not zero and, scaled, under 2^-2
  int solid;  // values that are 2^8 and more, scaled, in every `sample`-th step
  int unused;
};
// A matrix packed by rows (k along its columns) and by columns (k along its
// rows), either or both.  Block b of 16 rows, step s of 32 k is fragment
// (b * mul + add) * steps + s + first.
struct Packed {
  char* p;
  int steps, first, mul, add;
  Row* rows;
  int sample;  // a power of two
};
struct PackJob {
  const float* src;  // plain matrix (R, C), or null: both slopes of the Source
  int R, C;
  Packed rows[2], cols[2];        // of the gate and of the up slopes; a plain matrix has the first
  uint32_t *row_max, *col_max;    // largest magnitudes (bits) of the scan's tiles: [tile column][R], [part][tile row][C]
  float* sums;                    // [R / 32][2][C] column sums of the slopes, or null
  int tiles_c, block0, scan_c, scan0;
};
constexpr int kJobs = 4, kPackR = 32, kPackC = 64, kScanR = 32, kScanC = 128;
struct PackArgs {
  PackJob job[kJobs];
  int jobs;
  Source s;
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest magnitudes of 32 x 128 values by row and by column.  NaN and
// infinity count as the largest.  A wavefront has 8 rows, all (of slopes 4) in
// flight.  Bound: memory (the backward's 470 MB 117 us, 4.0 TB/s), at 777 x 1333
// the activations, 10 us (64 rows a tile: 21).
template <int ACT>  // of slopes; kNone: a plain matrix
__device__ __forceinline__ void scan_tile(const PackJob& j, const Source& s, int tr, int tc, uint32_t (*top)[4][kScanC]) {
  constexpr bool SLOPES = ACT != kNone;
  constexpr int NC = kScanC / 64, PARTS = SLOPES ? 2 : 1, DEEP = SLOPES ? 4 : 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = j.R, C = j.C, c0 = tc * kScanC, r0 = tr * kScanR + wave * (kScanR / 4);
  uint32_t col[PARTS][NC] = {};
#pragma unroll 1
  for (int d = 0; d < kScanR / 4; d += DEEP) {
    float v[SLOPES ? 3 : 1][DEEP][NC];
    uint32_t row[DEEP] = {}, m[DEEP][NC][PARTS];
#pragma unroll
    for (int y = 0; y < DEEP; ++y)
#pragma unroll
      for (int x = 0; x < NC; ++x) {  // the last row and column again where the matrix ends
        const long at = long(min(r0 + d + y, R - 1)) * C + min(c0 + x * 64 + lane, C - 1);
        if constexpr (SLOPES) {
          v[0][y][x] = s.g[at];
          v[1][y][x] = s.u[at];
          v[2][y][x] = s.dh[at];
        } else {
          v[0][y][x] = j.src[at];
        }
      }
#pragma unroll
    for (int y = 0; y < DEEP; ++y)
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        if constexpr (SLOPES) {
          float slope;
          const float act = gate(ACT, v[0][y][x], &slope);
          m[y][x][0] = magnitude(v[2][y][x] * v[1][y][x] * slope);
          m[y][x][1] = magnitude(v[2][y][x] * act);
        } else {
          m[y][x][0] = magnitude(v[0][y][x]);
        }
      }
#pragma unroll
    for (int y = 0; y < DEEP; ++y)
#pragma unroll
      for (int x = 0; x < NC; ++x)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          row[y] = max(row[y], m[y][x][p]);
          col[p][x] = max(col[p][x], m[y][x][p]);
        }
    if (j.row_max) {
#pragma unroll
      for (int y = 0; y < DEEP; ++y) {
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) row[y] = max(row[y], uint32_t(__shfl_xor(int(row[y]), x, 64)));
        if (lane == 0 && r0 + d + y < R) j.row_max[long(tc) * R + r0 + d + y] = row[y];
      }
    }
  }
  if (!j.col_max) return;
#pragma unroll
  for (int p = 0; p < PARTS; ++p)
#pragma unroll
    for (int x = 0; x < NC; ++x) top[p][wave][x * 64 + lane] = col[p][x];
  __syncthreads();
  const int c = c0 + (tid & (kScanC - 1)), p = tid / kScanC, x = tid & (kScanC - 1);
  if (c < C && p < PARTS)
    j.col_max[(long(p) * ((R + kScanR - 1) / kScanR) + tr) * C + c] =
        max(max(top[p][0][x], top[p][1][x]), max(top[p][2][x], top[p][3][x]));
}

__global__ __launch_bounds__(256) void k_scan(PackArgs a) {
  __shared__ uint32_t top[2][4][kScanC];
  int q = 0;
#pragma unroll
  for (int i = 1; i < kJobs; ++i)
    if (i < a.jobs && int(blockIdx.x) >= a.job[i].scan0) q = i;
  const PackJob& j = a.job[q];
  const int id = int(blockIdx.x) - j.scan0, tr = id / j.scan_c, tc = id - tr * j.scan_c;
  if (j.src) scan_tile<kNone>(j, a.s, tr, tc, top);
  else if (a.s.act == kSilu) scan_tile<kSilu>(j, a.s, tr, tc, top);
  else if (a.s.act == kGelu) scan_tile<kGelu>(j, a.s, tr, tc, top);
  else if (a.s.act == kRelu) scan_tile<kRelu>(j, a.s, tr, tc, top);
  else scan_tile<kSigmoid>(j, a.s, tr, tc, top);
}

// What the scan's tiles say together: the scale of every packed row, and its
// count of small values from 0.  64 rows a workgroup, four shares of the tiles.
struct ScaleJob {
  const uint32_t* part;  // [parts][rows]
  int parts, rows, block0;
  Packed to;
};
constexpr int kScales = 6;
struct ScaleArgs {
  ScaleJob job[kScales];
  int jobs;
};
constexpr int kNothing = -100000;      // the scale of a row of zeros
constexpr int kUnbounded = 128 - 14;  // and of one that is not finite
__global__ __launch_bounds__(256) void k_scales(ScaleArgs a) {
  __shared__ uint32_t top[256];
  int q = 0;
#pragma unroll
  for (int i = 1; i < kScales; ++i)
    if (i < a.jobs && int(blockIdx.x) >= a.job[i].block0) q = i;
  const ScaleJob& j = a.job[q];
  const int tid = threadIdx.x, r = (int(blockIdx.x) - j.block0) * 64 + (tid & 63), share = tid >> 6;
  uint32_t m = 0;
  if (r < j.rows)
#pragma unroll 4
    for (int p = share; p < j.parts; p += 4) m = max(m, j.part[long(p) * j.rows + r]);
  top[tid] = m;
  __syncthreads();
  if (share || r >= (j.rows + 15) / 16 * 16) return;  // whole blocks: packed rows beyond the matrix are zeros
  m = max(max(m, top[tid + 64]), max(top[tid + 128], top[tid + 192]));
  const int at = ((r >> 4) * j.to.mul + j.to.add) * 16 + (r & 15);
  const int e = m >> 23 ? int(m >> 23) - 127 : 31 - __clz(int(m)) - 149;
  j.to.rows[at] = Row{m ? e - 14 : kNothing, 0, 0, 0};
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// h of a value that is not zero and too small for fp16; zeros are 0.
#define kTiny (-_Float16(0))

// A lane's 8 values of a fragment, scaled and split.
__device__ __forceinline__ void put_fragment(const Packed& to, int block, int step, int lane, int scale, const float (&v)[8]) {
  f16x8 h, l;
  int small = 0, solid = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = scale == kNothing ? 0.f : __builtin_ldexpf(v[i], -scale);
    h[i] = _Float16(x);
    l[i] = _Float16(x - float(h[i]));
    if (h[i] == _Float16(0)) h[i] = x == 0.f ? _Float16(0) : kTiny;
    small += fabsf(x) < 0.25f && v[i] != 0.f;
    solid += fabsf(x) >= 256.f;
  }
  char* at = to.p + (long(block * to.mul + to.add) * to.steps + step + to.first) * kFrag + lane * 16;
  *reinterpret_cast<f16x8*>(at) = h;
  *reinterpret_cast<f16x8*>(at + kPart) = l;
  const bool sampled = ((step + to.first) & (to.sample - 1)) == 0;  // uniform
  if (!sampled && !__any(small)) return;
  int both = small << 16 | solid;
  both += __shfl_xor(both, 16, 64);
  both += __shfl_xor(both, 32, 64);
  if (lane < 16) {  // counts: any order gives the same
    Row* row = to.rows + (block * to.mul + to.add) * 16 + lane;
    if (sampled && (both & 0xffff)) atomicAdd(&row->solid, both & 0xffff);
    if (both >> 16) atomicAdd(&row->small, both >> 16);
  }
}

// A workgroup takes 32 x 64 values through LDS and writes them in both orders.
// Bound: memory, 12 bytes read and 16 written for each pair of slopes (8192 x
// 4096 with x and both weights: 268 us, 4.0 TB/s; a large copy 4.7).
constexpr int kPackP = kPackC + 4;
template <int ACT>
__device__ __forceinline__ void pack_tile(const PackJob& j, const Source& s, int tr, int tc, float (*tile)[kPackR * kPackP]) {
  constexpr bool SLOPES = ACT != kNone;
  constexpr int P = kPackP, PARTS = SLOPES ? 2 : 1, EACH = kPackR * kPackC / 256;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = tc * kPackC + lane;
  // Four fragments each way: two blocks of 16 rows by two steps of columns,
  // four blocks of 16 columns by one step of rows.
  const int rb = tr * 2 + (wave >> 1), rs = tc * 2 + (wave & 1), cb = tc * 4 + wave;
  const bool in_r = rb < (j.R + 15) / 16 && rs < (j.C + 31) / 32, in_c = cb < (j.C + 15) / 16;
  int scale_r[PARTS] = {}, scale_c[PARTS] = {};
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    const Packed &r = j.rows[p], &k = j.cols[p];
    if (r.p && in_r) scale_r[p] = r.rows[(rb * r.mul + r.add) * 16 + lr].scale;
    if (k.p && in_c) scale_c[p] = k.rows[(cb * k.mul + k.add) * 16 + lr].scale;
  }
  float v[SLOPES ? 3 : 1][EACH];  // a thread's values, 4 rows apart, in flight together
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const long at = long(min(tr * kPackR + i * 4 + wave, j.R - 1)) * j.C + min(c, j.C - 1);
    if constexpr (SLOPES) {
      v[0][i] = s.g[at];
      v[1][i] = s.u[at];
      v[2][i] = s.dh[at];
    } else {
      v[0][i] = j.src[at];
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int r = i * 4 + wave;
    const bool in = tr * kPackR + r < j.R && c < j.C;
    if constexpr (SLOPES) {
      float slope;
      const float act = gate(ACT, v[0][i], &slope);
      tile[0][r * P + lane] = in ? v[2][i] * v[1][i] * slope : 0.f;
      tile[1][r * P + lane] = in ? v[2][i] * act : 0.f;
    } else {
      tile[0][r * P + lane] = in ? v[0][i] : 0.f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    const float* T = tile[part];
    if (j.rows[part].p && in_r) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = T[((wave >> 1) * 16 + lr) * P + (wave & 1) * 32 + lg * 8 + i];
      put_fragment(j.rows[part], rb, rs, lane, scale_r[part], w);
    }
    if (j.cols[part].p && in_c) {
      float w[8], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = T[(lg * 8 + i) * P + wave * 16 + lr];
      put_fragment(j.cols[part], cb, tr, lane, scale_c[part], w);
      if (SLOPES && j.sums) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += w[i];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const int col = tc * kPackC + wave * 16 + lr;
        if (lg == 0 && col < j.C) j.sums[(long(tr) * 2 + part) * j.C + col] = sum;
      }
    }
  }
}

__global__ __launch_bounds__(256) void k_pack(PackArgs a) {
  __shared__ __attribute__((aligned(16))) float tile[2][kPackR * kPackP];
  int q = 0;
#pragma unroll
  for (int i = 1; i < kJobs; ++i)
    if (i < a.jobs && int(blockIdx.x) >= a.job[i].block0) q = i;
  const PackJob& j = a.job[q];
  const int id = int(blockIdx.x) - j.block0, tr = id / j.tiles_c, tc = id - tr * j.tiles_c;
  if (j.src) pack_tile<kNone>(j, a.s, tr, tc, tile);
  else if (a.s.act == kSilu) pack_tile<kSilu>(j, a.s, tr, tc, tile);
  else if (a.s.act == kGelu) pack_tile<kGelu>(j, a.s, tr, tc, tile);
  else if (a.s.act == kRelu) pack_tile<kRelu>(j, a.s, tr, tc, tile);
  else pack_tile<kSigmoid>(j, a.s, tr, tc, tile);
}

// ------------------------------------------------------------ the product ---

struct MmaArgs {
  const char *a, *b;  // packed operands
  const Row *rows_a, *rows_b;
  int product;
  int places;                // of the sampled steps
  int M, N;                  // rows of a and of b
  int steps, per;            // steps of 32 k, of a split
  int tiles_m, tiles_n, splits;
  bool wide;                 // results' rows start on 16 bytes
  float* part;               // partial sums of the splits, [split][M][N], or null
  const float *bg, *bu;      // kForward
  float *o0, *o1, *o2;       // kForward h, g, u; kInput dx; kWeight dW_gate, dW_up
  Source s;
};

// Products of one launch: the second's workgroups start at a multiple of 8, so
// that both go to the XCDs alike.
struct MmaPair {
  MmaArgs job[2];
  int first;  // the second's first workgroup
};

// Projections (biases added) of element (m, c) of h.
__device__ __forceinline__ void put_gated(const MmaArgs& a, long m, int c, float g, float u) {
  const long at = m * a.s.N + c;
  float slope;
  a.o0[at] = gate(a.s.act, g, &slope) * u;
  if (a.o1) {
    a.o1[at] = g;
    a.o2[at] = u;
  }
}

__device__ __forceinline__ float bias_of(const float* b, int c) { return b ? b[c] : 0.f; }

// W columns of a row, on 16 bytes where W is 4.
template <int W>
__device__ __forceinline__ void put(float* to, const float (&v)[W]) {
  if constexpr (W == 4) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
  else *to = v[0];
}
template <int W>
__device__ __forceinline__ void get(const float* from, float (&v)[W]) {
  if constexpr (W == 4) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e];
  } else {
    v[0] = *from;
  }
}

// A wavefront's results go from LDS where they belong, neighbouring lanes to
// neighbouring columns, W at a time.
template <int W, int ROWS, int COLS, int PITCH>
__device__ __forceinline__ void put_tile(const MmaArgs& a, int split, const float* mine, long m0, int n0, int lane) {
  if (a.part || a.product == kInput) {
    constexpr int L = COLS / W;  // lanes of a row
    float* to = a.part ? a.part + long(split) * a.M * a.N : a.o0;
    const int x = lane % L * W, n = n0 + x;
    if (n >= a.N) return;
#pragma unroll 2
    for (int y = lane / L; y < ROWS; y += 64 / L) {
      if (m0 + y >= a.M) break;
      float v[W];
      get(mine + y * PITCH + x, v);
      put(to + (m0 + y) * a.N + n, v);
    }
    return;
  }
  constexpr int L = COLS / 2 / W;
  const int x = lane % L * W, at = (x >> 4) * 32 + (x & 15), c = n0 / 2 + x, N = a.s.N;
  if (c >= N) return;
  float bg[W], bu[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    bg[e] = bias_of(a.bg, c + e);
    bu[e] = bias_of(a.bu, c + e);
  }
#pragma unroll 1
  for (int y = lane / L; y < ROWS; y += 64 / L) {
    if (m0 + y >= a.M) break;
    float g[W], u[W], h[W];
    get(mine + y * PITCH + at, g);
    get(mine + y * PITCH + at + 16, u);
    const long to = (m0 + y) * N + c;
    if (a.product == kWeight) {
      if (a.o0) put(a.o0 + to, g);
      if (a.o1) put(a.o1 + to, u);
      continue;
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
      g[e] += bg[e];
      u[e] += bu[e];
      float slope;
      h[e] = gate(a.s.act, g[e], &slope) * u[e];
    }
    put(a.o0 + to, h);
    if (a.o1) {
      put(a.o1 + to, g);
      put(a.o2 + to, u);
    }
  }
}

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

// Waits until at most N of this wavefront's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

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

__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Whether values that fp16 ends above could show in a sum at 2^-22 of its terms'
// absolute values, or it is not finite.  Each of them is off by up to 2^-25 and
// multiplied by up to 2^15, 2^-10 together; the terms amount to |sum| at least, and
// to 2^16 for every place where row and column are both solid: among the sampled
// places as many as both have solid ones beyond the number of places.  The
// second holds nearly everywhere in dense operands; the first decides where
// zeros meet large values.  It is asked of every sum, since the sums of other
// columns say nothing about it.  (Counting in every step kept packing 100 us
// longer at 8192 x 1024 x 4096.)
struct Guard {
  float spare, least;  // of a row's and a column's: solid places beyond what the small ones need; the sum that hides them
  __device__ __forceinline__ Guard(const Row& r, int places)
      : spare(float(r.solid - places) * 16.f - float(r.small)), least(float(r.small) * 4096.f) {}
};
__device__ __forceinline__ bool doubt(const Guard& a, const Guard& b, float sum) {
  const float size = fabsf(sum);
  return !((a.spare + b.spare >= 0.f || size >= a.least + b.least) && size < __builtin_inff());
}

// Magnitudes of a fragment's values, and 1 where fp16 ends above them.
__device__ __forceinline__ void magnitudes(f16x8 h, f16x8* size, f16x8* small) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  const u16x8 v = __builtin_bit_cast(u16x8, h);
  u16x8 m, one;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = v[i] == 0x8000 ? 1 : v[i] & 0x7fff;  // kTiny: the least there is
    one[i] = v[i] && m[i] < 0x3400 ? 0x3c00 : 0;
  }
  *size = __builtin_bit_cast(f16x8, m);
  *small = __builtin_bit_cast(f16x8, one);
}

// Where counts leave a doubt about 16 rows, pairs decide: the terms' absolute
// values and, in units of 2^-25, what the small values among them may be off by
// are formed from the h parts.  Sums in which that could show become infinite
// in the wavefront's results.  The factor leaves h's rounding to what the counts
// have passed.
template <int FH, int PITCH>
__device__ __forceinline__ void lossy_sums(const char* a, const char* b, long pitch, int s0, int s1, float* at) {
  f32x4 terms[FH], off[FH];
#pragma unroll
  for (int j = 0; j < FH; ++j) terms[j] = off[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int s = s0; s < s1; ++s) {
    f16x8 ha, hb[FH], size_a, small_a;
    ha = *reinterpret_cast<const f16x8*>(a + long(s) * kFrag);
#pragma unroll
    for (int j = 0; j < FH; ++j) hb[j] = *reinterpret_cast<const f16x8*>(b + j * pitch + long(s) * kFrag);
    magnitudes(ha, &size_a, &small_a);
#pragma unroll
    for (int j = 0; j < FH; ++j) {
      f16x8 size_b, small_b;
      magnitudes(hb[j], &size_b, &small_b);
      terms[j] = mfma_f16(size_a, size_b, terms[j]);
      off[j] = mfma_f16(small_a, size_b, off[j]);
      off[j] = mfma_f16(size_a, small_b, off[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < FH; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (!(off[j][r] <= 8.03125f * terms[j][r])) at[r * PITCH + j * 16] = __builtin_inff();
}

// A fragment's sums in FP32 from the plain operands, steps s0 to s1.  Addresses
// past the ends stay on the last element, so that nothing branches and a step's
// loads are in flight together.
template <int PRODUCT>
__device__ __forceinline__ f32x4 plain_sums(const Source& s, long m, int n, int s0, int s1, int lg) {
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
  int up = 0;
  const int c = PRODUCT == kInput ? n : column_of(n, &up);  // its column (of dx: weight row)
  const bool in_n = c < (PRODUCT == kInput ? s.K : s.N), in_m = m < (PRODUCT == kWeight ? s.K : s.M);
  const long mc = min(m, long(PRODUCT == kWeight ? s.K : s.M) - 1);
  const int nc = min(c, (PRODUCT == kInput ? s.K : s.N) - 1);
#pragma unroll 1
  for (int step = s0; step < s1; ++step) {
    float a[8], b[8], d[PRODUCT == kForward ? 1 : 3][8];
    const bool second = PRODUCT == kInput && step * 32 >= s.N32;  // of both projections' columns
    const bool of_up = PRODUCT == kInput ? second : up != 0;
    const float* w = of_up ? s.wu : s.wg;
    const int k0 = step * 32 - (second ? s.N32 : 0) + lg, K = PRODUCT == kForward ? s.K : PRODUCT == kInput ? s.N : s.M;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const long k = min(k0 + 4 * q, K - 1), at = PRODUCT == kInput ? mc * s.N + k : k * s.N + nc;
      if constexpr (PRODUCT == kForward) {
        a[q] = s.x[mc * s.K + k];
        b[q] = w[at];
      } else {
        if constexpr (PRODUCT == kInput) b[q] = w[long(nc) * s.N + k];
        else a[q] = s.x[k * s.K + mc];
        d[0][q] = s.g[at];
        d[1][q] = s.u[at];
        d[2][q] = s.dh[at];
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if constexpr (PRODUCT != kForward) {
        float slope;
        const float act = gate(s.act, d[0][q], &slope);
        (PRODUCT == kInput ? a[q] : b[q]) = of_up ? d[2][q] * act : d[2][q] * d[1][q] * slope;
      }
      const bool in_k = k0 + 4 * q < K;
      sum = mfma_f32(in_m && in_k ? a[q] : 0.f, in_n && in_k ? b[q] : 0.f, sum);
    }
  }
  return sum;
}

// WM x WN wavefronts of FM x FN fragments of 16 x 16, BUFS steps of operands in
// LDS.  256 x 256 tiles run at 0.94 (forward, with the activation and three
// outputs) and 1.37 PFLOP/s of fp16 (both gradients) at 8192 x 1024 x 4096; a
// large bf16 product of the library 1.15.  Tiles of 256 x 128 were bound by the
// L2s, which gave 9.7 TB/s (450 and 680 us where 256 x 256 took 404 and 604, both
// before sums were guarded one by one); reading the next step's fragments while
// this one's products run took as long.
// 64 x 64 tiles, three workgroups a compute unit, are as near the L2s' rate (9.4
// TB/s at 777 x 500 x 1333); there a workgroup's 16 steps take 6 of 12 us, the
// scales 2 and the results 2.5.
template <int WM, int WN, int FM, int FN, int BUFS>
__global__ __launch_bounds__(64 * WM * WN) void k_mma(MmaPair pair) {
  const int second = int(blockIdx.x) >= pair.first, id = int(blockIdx.x) - (second ? pair.first : 0);
  const MmaArgs& a = pair.job[second];
  const int tiles = a.tiles_m * a.tiles_n, split = id / tiles;
  if (split >= a.splits) return;  // fills up to a multiple of 8
  constexpr int NW = WM * WN, TA = WM * FM, TB = WN * FN, LOADS = (TA + TB) * kParts / NW;
  static_assert((TA + TB) * kParts % NW == 0, "whole fragments for every wavefront");
  // The results leave through LDS, 64 columns of a wavefront at a time.
  constexpr int ROWS = FM * 16, FH = FN < 4 ? FN : 4, COLS = FH * 16, PITCH = COLS + 4, L = COLS / 4;
  constexpr int BUF = (TA + TB) * kFrag, OUT = NW * ROWS * PITCH * 4;
  __shared__ __attribute__((aligned(16))) char lds[BUFS * BUF > OUT ? BUFS * BUF : OUT];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_of(id - split * tiles, a.tiles_m, a.tiles_n, &tm, &tn);
  const int s0 = split * a.per, s1 = min(a.steps, s0 + a.per);
  const long pitch = long(a.steps) * kFrag;
  // Part c of the tile's fragments: a's blocks first, then b's.
  const char* from[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int c = wave * LOADS + i, f = c / kParts;
    from[i] = (f < TA ? a.a + (long(tm) * TA + f) * pitch : a.b + (long(tn) * TB + f - TA) * pitch) +
              long(s0) * kFrag + (c - f * kParts) * kPart;
  }
  auto load = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      __builtin_amdgcn_global_load_lds((gvoid*)(from[i] + lane * 16), (lvoid*)(lds + buf * BUF + (wave * LOADS + i) * kPart), 16, 0, 0);
      from[i] += kFrag;
    }
  };
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // One step of loads in flight for every buffer but one.  A barrier alone does
  // not wait for loads into LDS: each wavefront waits for its own of the step
  // at hand, and the barrier for everybody's; behind it the buffer of the step
  // before is free.
  constexpr int AHEAD = BUFS - 1;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (s0 + i < s1) load(i);
  for (int s = s0, buf = 0; s < s1; ++s, buf = buf == AHEAD ? 0 : buf + 1) {
    if (s + AHEAD - 1 < s1) wait_loads<LOADS*(AHEAD - 1)>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const char* A = lds + buf * BUF + wm * FM * kFrag + lane * 16;
    const char* B = lds + buf * BUF + (TA + wn * FN) * kFrag + lane * 16;
    f16x8 pa[kParts][FM], pb[kParts][FN];
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
#pragma unroll
      for (int i = 0; i < FM; ++i) pa[p][i] = *reinterpret_cast<const f16x8*>(A + i * kFrag + p * kPart);
#pragma unroll
      for (int j = 0; j < FN; ++j) pb[p][j] = *reinterpret_cast<const f16x8*>(B + j * kFrag + p * kPart);
    }
    if (s + AHEAD < s1) load(buf == 0 ? AHEAD : buf - 1);  // after the reads, which need not wait for it
    auto mul = [&](int x, int y) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma_f16(pa[x][i], pb[y][j], acc[i][j]);
    };
    mul(1, 0);
    mul(0, 0);
    mul(0, 1);
    __builtin_amdgcn_sched_barrier(0);  // the products before the next wait: they cover the loads
  }

  // The rest by rows, through LDS, in loops that stay rolled: unrolled over the
  // fragments it is more code than the instruction cache holds, and every
  // workgroup waits for it (15 us and more).  Memory is written in whole lines.
  const long mw = (long(tm) * TA + wm * FM) * 16;
  __syncthreads();  // the buffers are read
  float* mine = reinterpret_cast<float*>(lds) + wave * ROWS * PITCH;
#pragma unroll 1
  for (int part = 0; part < FN / FH; ++part) {
    const int nw = (tn * TB + wn * FN + part * FH) * 16;
#pragma unroll
    for (int x = 0; x < FN / FH; ++x)
      if (part == x)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FH; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) mine[(i * 16 + 4 * lg + r) * PITCH + j * 16 + lr] = acc[i][x * FH + j][r];

    // Scales taken out, sums in doubt looked into and formed again.
    const int x4 = lane % L * 4, y0 = lane / L;
    int scale_b[4];
    Guard guard_b[4] = {{Row{}, 0}, {Row{}, 0}, {Row{}, 0}, {Row{}, 0}};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      scale_b[e] = kNothing;
      if (nw + x4 + e < a.N) {
        const Row r = a.rows_b[nw + x4 + e];
        scale_b[e] = r.scale;
        guard_b[e] = Guard(r, a.places);
      }
    }
    uint32_t again = 0;  // bit i: in 16 rows
#pragma unroll 2
    for (int i = 0; i < ROWS * L / 64; ++i) {
      const int y = i * (64 / L) + y0;
      Row ra{kNothing, 0, 0, 0};
      if (mw + y < a.M) ra = a.rows_a[mw + y];
      const Guard guard_a(ra, 0);
      f32x4* at = reinterpret_cast<f32x4*>(mine + y * PITCH + x4);
      f32x4 v = *at;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool none = ra.scale == kNothing || scale_b[e] == kNothing;  // zeros, and rows nobody packed
        bad = bad || (none ? ra.scale == kUnbounded || scale_b[e] == kUnbounded : doubt(guard_a, guard_b[e], v[e]));
        v[e] = none ? 0.f : __builtin_ldexpf(v[e], ra.scale + scale_b[e]);
      }
      *at = v;
      again |= uint32_t(bad) << (i * (64 / L) / 16);
    }
    if (__any(again)) {
#pragma unroll 1
      for (int i = 0; i < FM; ++i) {
        const long m = mw + i * 16;
        if (!__any(again >> i & 1) || m >= a.M) continue;
        float* at = mine + (i * 16 + 4 * lg) * PITCH + lr;
        lossy_sums<FH, PITCH>(a.a + (m / 16) * pitch + lane * 16, a.b + long(nw / 16) * pitch + lane * 16, pitch, s0, s1, at);
#pragma unroll 1
        for (int j = 0; j < FH; ++j, at += 16) {
          const int n = nw + j * 16;
          bool bad = false;
#pragma unroll
          for (int r = 0; r < 4; ++r) bad = bad || !__builtin_isfinite(at[r * PITCH]);
          if (!__any(bad) || n >= a.N) continue;
          const f32x4 exact = a.product == kForward ? plain_sums<kForward>(a.s, m + lr, n + lr, s0, s1, lg)
                              : a.product == kInput ? plain_sums<kInput>(a.s, m + lr, n + lr, s0, s1, lg)
                                                    : plain_sums<kWeight>(a.s, m + lr, n + lr, s0, s1, lg);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!__builtin_isfinite(at[r * PITCH])) at[r * PITCH] = exact[r];
        }
      }
    }

    if (a.wide) put_tile<4, ROWS, COLS, PITCH>(a, split, mine, mw, nw, lane);
    else put_tile<1, ROWS, COLS, PITCH>(a, split, mine, mw, nw, lane);
  }
}

// What follows the products: the splits' sums, in order, and the bias
// gradients, the column sums of every 32 rows in order.
struct FinishArgs {
  MmaArgs job[2];
  int blocks[2];  // workgroups of the products' splits
  int columns;    // and of the column sums, 16 columns each in turn
  const float* sums;
  int tiles, N;
  float *db_gate, *db_up;
};
__device__ __forceinline__ void add_splits(const MmaArgs& a, int block, int blocks) {
  const long total = long(a.M) * a.N, half = long(a.M) * a.s.N;
  const long count = a.product == kInput ? total : half;
  for (long i = long(block) * 256 + threadIdx.x; i < count; i += long(blocks) * 256) {
    if (a.product == kInput) {
      float t = 0.f;
      for (int s = 0; s < a.splits; ++s) t += a.part[s * total + i];
      a.o0[i] = t;
      continue;
    }
    const long m = i / a.s.N;
    const int c = int(i - m * a.s.N);
    const long at = m * a.N + (c >> 4) * 32 + (c & 15);
    float g = 0.f, u = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      g += a.part[s * total + at];
      u += a.part[s * total + at + 16];
    }
    if (a.product == kForward) {
      put_gated(a, m, c, g + bias_of(a.bg, c), u + bias_of(a.bu, c));
    } else {
      if (a.o0) a.o0[i] = g;
      if (a.o1) a.o1[i] = u;
    }
  }
}
__global__ __launch_bounds__(256) void k_finish(FinishArgs a) {
  __shared__ double red[256];
  int block = int(blockIdx.x);
  for (int j = 0; j < 2; ++j) {
    if (block < a.blocks[j]) {
      add_splits(a.job[j], block, a.blocks[j]);
      return;
    }
    block -= a.blocks[j];
  }
  const long N = a.N;
  const int q = threadIdx.x >> 4;
  for (long c = long(block) * 16 + (threadIdx.x & 15); c - (threadIdx.x & 15) < 2 * N; c += a.columns * 16L) {
    double t = 0.0;
    if (c < 2 * N)
      for (int i = q; i < a.tiles; i += 16) t += double(a.sums[i * 2 * N + c]);
    red[threadIdx.x] = t;
    __syncthreads();
    if (q == 0 && c < 2 * N) {
      for (int i = 1; i < 16; ++i) t += red[i * 16 + threadIdx.x];
      float* to = c < N ? a.db_gate : a.db_up;
      if (to) to[c < N ? c : c - N] = float(t);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------- small products ---

// 16 columns of both projections and 16 RB rows: the weights go from memory
// into the products' registers, the wavefronts share K and their sums meet in
// LDS, in order.  XV: x in whole 16-byte rows.  Bound: at one row the launch and
// two memory round trips (512 x 2048, 8.4 MB of weights: 5.0 us, 1.7 TB/s); with
// more the weights' loads, 64 bytes of a row for each of 16 columns, dword by dword
// (1024 x 4096 with 64 rows 18 us: 1.8 TB/s of weights, 59 TFLOP/s where a large
// FP32 product runs at 153).
struct FewArgs {
  const float *x, *wg, *wu;
  MmaArgs out;
  int first;  // column that the launch begins with
};
constexpr int kFewWaves = 8;
// Workgroups in x of one launch: its threads are counted in 32 bits, and a count
// that passes them starts what is left of it without an error.
constexpr int kFewGroups = 1 << 22;

template <int RB, bool XV>
__global__ __launch_bounds__(64 * kFewWaves) void k_few(FewArgs a) {
  __shared__ float part[kFewWaves][2 * RB * 256];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = a.out.s.M, K = a.out.s.K, N = a.out.s.N, n0 = a.first + int(blockIdx.x) * 16, n = n0 + lr;
  const __amdgpu_buffer_rsrc_t rx = make_res(a.x, uint32_t(M) * uint32_t(K) * 4u);
  const uint32_t bytes = uint32_t(K) * uint32_t(N) * 4u;
  const __amdgpu_buffer_rsrc_t rg = make_res(a.wg, bytes), ru = make_res(a.wu, bytes);
  const int blocks = (K + 15) / 16, per = (blocks + kFewWaves - 1) / kFewWaves;
  const int m0 = int(blockIdx.y) * 16 * RB;
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
        w[0][d][r] = ld_f1(rg, off);
        w[1][d][r] = ld_f1(ru, off);
      }
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const int m = m0 + b * 16 + lr;
        if constexpr (XV) {
          x[d][b] = ld_f4(rx, in && m < M && k < K ? (uint32_t(m) * uint32_t(K) + uint32_t(k)) * 4u : ~0u - 15u);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[d][b][r] = ld_f1(rx, in && m < M && k + r < K ? (uint32_t(m) * uint32_t(K) + uint32_t(k + r)) * 4u : ~0u);
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
    const int m = m0 + (i >> 4), c = n0 + (i & 15);
    if (m >= M || c >= N) continue;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      g += part[w][i];
      u += part[w][RB * 256 + i];
    }
    put_gated(a.out, m, c, g + bias_of(a.out.bg, c), u + bias_of(a.out.bu, c));
  }
}

// ------------------------------------------------------------------ host ---

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
long up_to(long n, long q) { return (n + q - 1) / q * q; }

// Products that read their operands as they are: beyond, packing pays.  Forward
// alone, calls one after another, this way and packed, us: K 512, N 2048 with 128
// rows 9.4 / 27, 256 17 / 27, 512 32 / 30; 1024, 4096 with 32 13 / 38, 64 18 / 39, 192
// 49 / 43; 2048, 1024 with 256 28 / 35, 300 53 / 38; 777 x 500 x 1333 43 / 34.  The line
// is at 256 rows of the first, 64 of the second and 128 of the third.
constexpr long kFewWork = 1L << 28;
bool few_products(const ttrl_gated_desc* d) {
  return long(d->M) * d->K <= kFewWork / d->N && d->M <= 64 * 65535;  // 64 rows to each of a grid's y
}

// A product's tiles and splits: 256 x 256 where they fill three quarters of the
// compute units, counting what shares the launch, else 64 x 64, and k in splits
// while there are fewer workgroups than two a compute unit and a split keeps
// kMinSteps steps.  Forward alone in tiles of 256 x 256 and of 64 x 64, us: 128 tiles
// (2048 x 512 x 2048) 81 / 57; 256 tiles 73 / 73 (8192 x 256 x 1024), 87 / 92 (4096 x 512
// x 2048), 127 / 146 (4096 x 1024 x 2048); 512 tiles 159 / 163 (8192 x 512 x 2048); 1024
// tiles 446 / 507 (8192 x 1024 x 4096).
constexpr int kMinSteps = 6;
struct MmaPlan {
  bool big;
  int tiles_m, tiles_n, splits, per;
};
MmaPlan plan_mma(long M, long N, long steps, int together) {
  MmaPlan p{};
  p.big = ((M + 255) / 256) * ((N + 255) / 256) * together >= 192;
  const int t = p.big ? 256 : 64;
  p.tiles_m = int((M + t - 1) / t);
  p.tiles_n = int((N + t - 1) / t);
  const long tiles = long(p.tiles_m) * p.tiles_n, want = p.big ? 256 / together : 512;
  long splits = tiles >= want / 2 ? 1 : std::min((want + tiles - 1) / tiles, std::max(1L, steps / kMinSteps));
  splits = std::min(splits, 64L);
  p.per = int((steps + splits - 1) / splits);
  p.splits = int((steps + p.per - 1) / p.per);
  return p;
}

// One product: its packed operands with their scales, and its partial sums, in
// the workspace.
struct Layout {
  long a, b, rows, part;  // bytes
  MmaPlan plan;
  long rows_a, rows_b;
  int steps, sample, places;
};
constexpr int kSampled = 8;  // steps whose solid values are counted, at most
// `terms` of a sum lie in whole steps of 32, twice over where there are two `halves`.
Layout layout_of(long M, long N, long terms, int halves, int together) {
  Layout l{};
  const long steps = (terms + 31) / 32;
  l.steps = int(steps * halves);
  for (l.sample = 1; l.sample * kSampled < l.steps;) l.sample *= 2;
  for (long s = 0; s < l.steps; s += l.sample) l.places += int(std::min(32L, terms - s % steps * 32));
  l.plan = plan_mma(M, N, l.steps, together);
  l.rows_a = M;
  l.rows_b = N;
  l.a = up_to(M, 256) / 16 * l.steps * kFrag;  // whole tiles are read, whatever lies there
  l.b = up_to(N, 256) / 16 * l.steps * kFrag;
  l.rows = up_to((up_to(M, 16) + up_to(N, 16)) * long(sizeof(Row)), 256);
  l.part = l.plan.splits > 1 ? up_to(long(l.plan.splits) * M * N * 4, 256) : 0;
  return l;
}
// The operands of a product laid out from `at`.
struct Operands {
  Packed a, b;
};
Operands operands_at(const Layout& l, char* at) {
  Row* rows = reinterpret_cast<Row*>(at + l.a + l.b);
  return Operands{Packed{at, l.steps, 0, 1, 0, rows, l.sample}, Packed{at + l.a, l.steps, 0, 1, 0, rows + up_to(l.rows_a, 16), l.sample}};
}
Packed moved(Packed p, int first, int mul, int add) {
  p.first = first;
  p.mul = mul;
  p.add = add;
  return p;
}
long scan_rows(long R) { return (R + kScanR - 1) / kScanR; }
long scan_cols(long C) { return (C + kScanC - 1) / kScanC; }

struct Layouts {
  Layout fwd, dx, dw;
  long fwd_max, bwd_max, sums;  // bytes of the scans' results and of the column sums
};
Layouts layouts_of(const ttrl_gated_desc* d) {
  const long rows = std::max(1, d->M), both = up_to(d->N, 16) * 2;
  Layouts l;
  l.fwd = layout_of(rows, both, d->K, 1, 1);
  l.dx = layout_of(rows, d->K, d->N, 2, 2);
  l.dw = layout_of(d->K, both, rows, 1, 2);
  l.fwd_max = up_to((scan_cols(d->K) * rows + 2 * scan_rows(d->K) * d->N) * 4, 256);
  l.bwd_max = up_to((scan_cols(d->N) * (rows + 2L * d->K) + scan_rows(rows) * (2L * d->N + d->K)) * 4, 256);
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

int launch_pack(ttrl_ctx* ctx, PackArgs& a, ScaleArgs& c, const char* name) {
  long blocks = 0, scans = 0, scales = 0;
  for (int i = 0; i < a.jobs; ++i) {
    PackJob& j = a.job[i];
    j.tiles_c = int((j.C + kPackC - 1) / kPackC);
    j.block0 = int(blocks);
    blocks += long(j.tiles_c) * ((j.R + kPackR - 1) / kPackR);
    j.scan_c = int(scan_cols(j.C));
    j.scan0 = int(scans);
    scans += scan_cols(j.C) * scan_rows(j.R);
  }
  for (int i = 0; i < c.jobs; ++i) {
    c.job[i].block0 = int(scales);
    scales += (c.job[i].rows + 63) / 64;
  }
  hipLaunchKernelGGL(k_scan, dim3(unsigned(scans)), dim3(256), 0, stream_of(ctx), a);
  if (int rc = check_launch(name)) return rc;
  hipLaunchKernelGGL(k_scales, dim3(unsigned(scales)), dim3(256), 0, stream_of(ctx), c);
  if (int rc = check_launch(name)) return rc;
  hipLaunchKernelGGL(k_pack, dim3(unsigned(blocks)), dim3(256), 0, stream_of(ctx), a);
  return check_launch(name);
}

void fill_in(MmaArgs& a, const Layout& l, const Operands& o, float* part) {
  a.a = o.a.p;
  a.b = o.b.p;
  a.rows_a = o.a.rows;
  a.rows_b = o.b.rows;
  a.M = int(l.rows_a);
  a.N = int(l.rows_b);
  a.steps = l.steps;
  a.places = l.places;
  a.per = l.plan.per;
  a.tiles_m = l.plan.tiles_m;
  a.tiles_n = l.plan.tiles_n;
  a.splits = l.plan.splits;
  a.part = l.plan.splits > 1 ? part : nullptr;
  const int width = a.product == kInput || a.part ? a.N : a.s.N;
  a.wide = width % 4 == 0 && (a.part || (aligned16(a.o0) && aligned16(a.o1) && aligned16(a.o2)));
}

// One or two products of one plan's tiles.
int launch_mma(ttrl_ctx* ctx, const MmaArgs* const* jobs, int count, bool big, const char* name) {
  MmaPair p{};
  long blocks = 0;
  for (int i = 0; i < count; ++i) {
    if (i) p.first = int(blocks = up_to(blocks, 8));
    p.job[i] = *jobs[i];
    blocks += long(jobs[i]->tiles_m) * jobs[i]->tiles_n * jobs[i]->splits;
  }
  if (count == 1) p.first = int(blocks);
  const dim3 grid{unsigned(blocks)};
  if (big) hipLaunchKernelGGL((k_mma<4, 2, 4, 8, 2>), grid, dim3(512), 0, stream_of(ctx), p);
  else hipLaunchKernelGGL((k_mma<2, 2, 2, 2, 3>), grid, dim3(256), 0, stream_of(ctx), p);
  return check_launch(name);
}

// Splits of the products that have any, and the bias gradients.
int launch_finish(ttrl_ctx* ctx, const MmaArgs* const* jobs, int count, FinishArgs& a, const char* name) {
  long blocks = a.columns = a.sums ? int(std::min(4096L, (2L * a.N + 15) / 16)) : 0;
  for (int i = 0; i < count; ++i) {
    const MmaArgs& m = *jobs[i];
    if (!m.part) continue;
    a.job[i] = m;
    const long n = long(m.M) * (m.product == kInput ? m.N : m.s.N);
    a.blocks[i] = int(std::min(2048L, (n + 255) / 256));
    blocks += a.blocks[i];
  }
  if (!blocks) return TTRL_OK;
  hipLaunchKernelGGL(k_finish, dim3(unsigned(blocks)), dim3(256), 0, stream_of(ctx), a);
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
  *forward_bytes = few_products(d) ? 0 : l.fwd.a + l.fwd.b + l.fwd.rows + l.fwd_max + l.fwd.part;
  *backward_bytes = l.dx.a + l.dx.b + l.dx.rows + l.dw.a + l.dw.b + l.dw.rows + l.bwd_max +
                    l.dx.part + l.dw.part + l.sums;
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
  if (few_products(d)) {
    FewArgs f{d->x, d->w_gate, d->w_up, m, 0};
    const int rb = d->M <= 16 ? 1 : d->M <= 32 ? 2 : 4;
    const int groups = ceil_div(d->N, 16);
    const dim3 block(64 * kFewWaves);
    const bool xv = d->K % 4 == 0 && aligned16(d->x);
    for (int from = 0; from < groups; from += kFewGroups) {
      const dim3 grid(std::min(kFewGroups, groups - from), ceil_div(d->M, 16 * rb));
      f.first = from * 16;
      auto go = [&](auto rb) {
        constexpr int RB = decltype(rb)::value;
        if (xv) hipLaunchKernelGGL((k_few<RB, true>), grid, block, 0, stream_of(ctx), f);
        else hipLaunchKernelGGL((k_few<RB, false>), grid, block, 0, stream_of(ctx), f);
      };
      if (rb == 1) go(std::integral_constant<int, 1>{});
      else if (rb == 2) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 4>{});
      if (int rc = check_launch(name)) return rc;
    }
    return TTRL_OK;
  }
  TTRL_REQUIRE(d->work && aligned16(d->work), "%s: null or unaligned workspace", name);
  const Layouts ls = layouts_of(d);
  const Layout& l = ls.fwd;
  char* at = static_cast<char*>(d->work);
  const Operands o = operands_at(l, at);
  uint32_t* tops = reinterpret_cast<uint32_t*>(at + l.a + l.b + l.rows);
  PackArgs p{};
  ScaleArgs c{};
  p.s = m.s;
  p.jobs = c.jobs = 3;
  p.job[0] = PackJob{d->x, d->M, d->K};
  p.job[0].rows[0] = o.a;
  p.job[0].row_max = tops;
  c.job[0] = ScaleJob{tops, int(scan_cols(d->K)), d->M, 0, o.a};
  tops += scan_cols(d->K) * d->M;
  for (int q = 0; q < 2; ++q, tops += scan_rows(d->K) * d->N) {
    PackJob& w = p.job[1 + q];
    w = PackJob{q ? d->w_up : d->w_gate, d->K, d->N};
    w.cols[0] = moved(o.b, 0, 2, q);
    w.col_max = tops;
    c.job[1 + q] = ScaleJob{tops, int(scan_rows(d->K)), d->N, 0, w.cols[0]};
  }
  if (int rc = launch_pack(ctx, p, c, name)) return rc;
  fill_in(m, l, o, reinterpret_cast<float*>(at + l.a + l.b + l.rows + ls.fwd_max));
  const MmaArgs* jobs[] = {&m};
  if (int rc = launch_mma(ctx, jobs, 1, l.plan.big, name)) return rc;
  FinishArgs f{};
  return launch_finish(ctx, jobs, 1, f, name);
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
  if (!d->dx && !dw && !db) return TTRL_OK;
  char *at_dx = static_cast<char*>(d->work), *at_dw = at_dx + l.dx.a + l.dx.b + l.dx.rows;
  char* rest = at_dw + l.dw.a + l.dw.b + l.dw.rows;
  const Operands odx = operands_at(l.dx, at_dx), odw = operands_at(l.dw, at_dw);
  uint32_t* tops = reinterpret_cast<uint32_t*>(rest);
  float* part = reinterpret_cast<float*>(rest + l.bwd_max);
  float* sums = reinterpret_cast<float*>(rest + l.bwd_max + l.dx.part + l.dw.part);
  const int n32 = (d->N + 31) / 32;
  const Source s = source_of(d);
  PackArgs p{};
  ScaleArgs c{};
  p.s = s;
  auto scaled = [&](long parts, int rows, const Packed& to) {
    c.job[c.jobs++] = ScaleJob{tops, int(parts), rows, 0, to};
    uint32_t* at = tops;
    tops += parts * rows;
    return at;
  };
  PackJob& slopes = p.job[p.jobs++];
  slopes = PackJob{nullptr, d->M, d->N};
  for (int q = 0; q < 2; ++q) {
    if (d->dx) slopes.rows[q] = moved(odx.a, q * n32, 1, 0);
    if (dw || db) slopes.cols[q] = moved(odw.b, 0, 2, q);
  }
  if (d->dx) slopes.row_max = scaled(scan_cols(d->N), d->M, odx.a);  // both slopes are one row there
  if (dw || db) {
    slopes.col_max = scaled(scan_rows(d->M), d->N, slopes.cols[0]);
    scaled(scan_rows(d->M), d->N, slopes.cols[1]);
  }
  slopes.sums = db ? sums : nullptr;
  if (dw) {
    PackJob& x = p.job[p.jobs++];
    x = PackJob{d->x, d->M, d->K};
    x.cols[0] = odw.a;
    x.col_max = scaled(scan_rows(d->M), d->K, odw.a);
  }
  if (d->dx) {
    uint32_t* at = scaled(2 * scan_cols(d->N), d->K, odx.b);  // as are both weights
    for (int q = 0; q < 2; ++q) {
      PackJob& w = p.job[p.jobs++];
      w = PackJob{q ? d->w_up : d->w_gate, d->K, d->N};
      w.rows[0] = moved(odx.b, q * n32, 1, 0);
      w.row_max = at + q * scan_cols(d->N) * d->K;
    }
  }
  if (int rc = launch_pack(ctx, p, c, name)) return rc;
  MmaArgs mx{}, mw{};
  mx.product = kInput;
  mx.o0 = d->dx;
  mw.product = kWeight;
  mw.o0 = d->dw_gate;
  mw.o1 = d->dw_up;
  mx.s = mw.s = s;
  fill_in(mx, l.dx, odx, part);
  fill_in(mw, l.dw, odw, part + l.dx.part / 4);
  const MmaArgs* jobs[2];
  int count = 0;
  if (d->dx) jobs[count++] = &mx;
  if (dw) jobs[count++] = &mw;
  if (count == 2 && l.dx.plan.big != l.dw.plan.big) {
    if (int rc = launch_mma(ctx, jobs, 1, l.dx.plan.big, name)) return rc;
    if (int rc = launch_mma(ctx, jobs + 1, 1, l.dw.plan.big, name)) return rc;
  } else if (count) {
    if (int rc = launch_mma(ctx, jobs, count, (d->dx ? l.dx : l.dw).plan.big, name)) return rc;
  }
  FinishArgs f{};
  f.sums = db ? sums : nullptr;
  f.tiles = (d->M + 31) / 32;
  f.N = d->N;
  f.db_gate = d->db_gate;
  f.db_up = d->db_up;
  return launch_finish(ctx, jobs, count, f, name);
}

}  // extern "C"
