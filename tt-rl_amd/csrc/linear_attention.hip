// Linear attention with a decay for each head: a recurrent memory whose state
// is a matrix per head,
//
//   S_t = a_t S_{t-1} + k_t v_t^T,   o_t = s q_t^T S_t,   a_t = exp(g_t),
//
// with a_t = 0 where an episode starts (`done`), so that nothing of one episode
// reaches another.  s is the scale.  One head's q and k have K values, v and o
// have V, the state K x V; kv_heads < H heads share their k and v.
//
// Every output is one kind of sweep.  With the gradient state
// G_t = s q_t do_t^T + a_{t+1} G_{t+1} (G_T the final state's gradient),
//
//   o_t  = s S_t^T q_t        sweep (x, y, z) = (q, k, v)
//   dq_t = s S_t do_t         sweep (do, v, k), its state S^T
//   dv_t = G_t^T k_t          sweep backwards in time (k, q, do)
//   dk_t = G_t v_t            sweep backwards in time (v, do, q), its state G^T
//
// where a sweep forms out_i = sum over j <= i of w(i, j) (x_i . y_j) z_j, and
// w(i, j) is the product of the decays between steps j and i.  In time order a
// step's decay is its own a_t; backwards it is a_{t+1}, the step's after it.
// For the decay, X_t = a_t <S_{t-1}, G_t> = dL/dg_t satisfies
// X_t = X_{t+1} + q_t . dq_t - k_t . dk_t, and is 0 where an episode starts.
//
// A sweep takes chunks of 32 steps.  Inside a chunk the sums are products of
// 32 x 32 weights (P = (X Y^T) * w, out += P Z), and the chunks are joined by
// the state (out += w X S, S = a S + (w Y)^T Z).  Each wavefront owns 16 columns of
// the state and keeps them in registers for its whole sweep: an accumulator of
// v_mfma_f32_16x16x4f32 holds row 4 * (lane / 16) + r, which is the k that the
// same lane's B operand needs when the r-th of four products takes
// k = 4 * (lane / 16) + r, so the state is product, sum and operand without
// a move.  x and y go through LDS, z straight into registers.
//
// Where there are few heads and sequences, the sequence is cut into segments
// that run side by side: a first launch forms what each segment adds to the
// state, a second joins them in order (start[s + 1] = decay[s] start[s] +
// added[s]), and the sweeps then start from the joined states.
//
// Precision: products, sums and states are FP32; the sums of log decays are in
// double, and each weight is the exponential of a difference of two of them, so
// a strong decay in a chunk takes nothing from the weights after it.
//
// Values that are not finite stay in their episode and behind their step: a
// masked weight is selected, never multiplied, and a chunk whose z holds such
// values forms its inner sums over the allowed steps alone.
#include "common.hpp"

#include <cmath>

namespace ttrl {
namespace {

constexpr int kChunk = 32;
// Below this exp() is zero in float32: such a step forgets as a start does.
constexpr float kForget = -104.f;
constexpr int kMaxHead = 128;

struct Operand {
  const float* p;
  int heads, dim, share;  // row (t, b, h) at ((t * B + b) * heads + h / share) * dim
};

struct Sweep {
  Operand x, y, z;
  float* out;  // (T, B, H, E)
  Operand dot;  // rows to multiply the output's rows with, or null
  float* dots;  // [E / 16][B * H][T] partial sums of those products, 16 columns each
  const float* start;  // state on entering a segment: [segment][B * H][D * E], or of the first one only
  int start_all;       // one for every segment
  float* end;          // the last segment's state, [B * H][D * E]
  int end_decay;       // end is the state entering step 0: one more decay
  int sk, se;          // strides of a state's element (d, e)
  int back;            // backwards in time
  float alpha_out;     // factor of the outputs
  float alpha_pair;    // factor of every product x . y z
};

struct SweepArgs {
  Sweep s[3];
  const float* g;
  const float* done;
  int g_rows;  // g is (T, B, H), else (1, H)
  int T, B, H, seg, nseg;
  float* added;   // first launch: [segment][B * H][D * E]
  float* decays;  // first launch: [segment][B * H]
};

__device__ __forceinline__ f32x4 mfma4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// One chunk's decays, step i of the chunk in lane i of every wavefront.
struct Decays {
  double c;      // sum of the log decays since the chunk's or the episode's start
  int lo;        // the episode's first step in the chunk, -1: before it
  float into;    // weight of the state on entering the chunk (0: none)
  float left;    // weight of the step in the state on leaving it (0: none)
  float keep;    // weight of the entering state in the leaving one (uniform)
  int first;     // first step that the leaving state holds (uniform)
  __device__ __forceinline__ void form(float g, bool reset, int lane) {
    const int i = lane & 31;
    const uint32_t starts = uint32_t(__ballot(reset));
    const uint32_t m = starts & (0xffffffffu >> (31 - i));
    lo = m ? 31 - __clz(m) : -1;
    c = reset ? 0.0 : double(g);
#pragma unroll
    for (int d = 1; d < kChunk; d <<= 1) {
      const double t = __shfl_up(c, d, 32);
      if (i - d >= max(lo, 0)) c += t;
    }
    const double ce = __shfl(c, 31, 32);
    const int le = starts ? 31 - __clz(starts) : -1;
    first = max(le, 0);
    into = lo < 0 ? expf(float(c)) : 0.f;
    left = i >= first ? expf(float(ce - c)) : 0.f;
    keep = le < 0 ? expf(float(ce)) : 0.f;
  }
};

// The log decay of step t and whether it forgets what was before it.
__device__ __forceinline__ void step_decay(const SweepArgs& a, int t, int b, int h, float& g, bool& reset) {
  g = 0.f;
  reset = false;
  if (t < a.T) {
    g = a.g_rows ? a.g[(long(t) * a.B + b) * a.H + h] : a.g[h];
    const float d = a.done ? a.done[long(t) * a.B + b] : 0.f;
    reset = d > 0.f || g < kForget;
  }
}

// 32 rows of an operand on their way into LDS.
template <int KP, int NT, bool VEC>
struct Rows {
  static constexpr int W = VEC ? 4 : 1, CH = KP / W, PER = (kChunk * CH + NT - 1) / NT;
  static constexpr bool WHOLE = kChunk * CH % NT == 0;
  float f[PER][W];
  __device__ __forceinline__ void issue(const Operand& o, long base, long pitch, int s0, int n, int dir, int tid) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + u * NT, r = i / CH, c = i % CH * W;
      const bool in = (WHOLE || r < kChunk) && s0 + r < n && c < o.dim;
      const float* p = o.p + base + long(dir) * (s0 + r) * pitch + c;
      if constexpr (VEC) {
        const f32x4 v = in ? *reinterpret_cast<const f32x4*>(p) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) f[u][j] = v[j];
      } else {
        f[u][0] = in ? *p : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(float* lds, int tid) const {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + u * NT, r = i / CH, c = i % CH * W;
      if (!WHOLE && r >= kChunk) continue;
      float* d = lds + r * (KP + 4) + c;
      if constexpr (VEC) *reinterpret_cast<f32x4*>(d) = f32x4{f[u][0], f[u][1], f[u][2], f[u][3]};
      else *d = f[u][0];
    }
  }
};

// LOCAL: the first launch, what a segment adds to the state.
template <int KP, int NW, bool VEC, bool LOCAL>
__global__ __launch_bounds__(64 * NW) void k_sweep(SweepArgs a) {
  constexpr int NT = 64 * NW, KB = KP / 16, PX = KP + 4, PP = kChunk + 4;
  __shared__ __attribute__((aligned(16))) float lx[LOCAL ? 1 : 2][LOCAL ? 4 : kChunk * PX];
  __shared__ __attribute__((aligned(16))) float ly[2][kChunk * PX];
  __shared__ __attribute__((aligned(16))) float lp[LOCAL ? 1 : 2][LOCAL ? 4 : kChunk * PP];
  const Sweep& w = a.s[blockIdx.z];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const int bh = int(blockIdx.x), b = bh / a.H, h = bh - b * a.H, seg = int(blockIdx.y);
  const int t0 = seg * a.seg, n = min(a.seg, a.T - t0);
  const int D = w.x.dim, E = w.z.dim, nkb = (D + 15) / 16;
  const int dir = w.back ? -1 : 1, tb = w.back ? t0 + n - 1 : t0;  // time of step s: tb + dir * s
  const int td = w.back ? tb + 1 : tb;                             // of its decay
  const int e = wave * 16 + lr;

  auto base = [&](const Operand& o) { return ((long(tb) * a.B + b) * o.heads + h / o.share) * long(o.dim); };
  auto pitch = [&](const Operand& o) { return long(a.B) * o.heads * o.dim; };
  const long bx = LOCAL ? 0 : base(w.x), px = LOCAL ? 0 : pitch(w.x);
  const long by = base(w.y), py = pitch(w.y), bz = base(w.z), pz = pitch(w.z);
  const long po = long(a.B) * a.H * E, bo = ((long(tb) * a.B + b) * a.H + h) * long(E);

  f32x4 S[KB];
  {
    const float* st = LOCAL ? nullptr : w.start;
    const bool any = st && (w.start_all || (w.back ? seg + 1 == a.nseg : seg == 0));
    if (any) st += (w.start_all ? long(seg) * a.B * a.H + bh : long(bh)) * D * E;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = k * 16 + 4 * lg + r;
        S[k][r] = any && d < D && e < E ? st[long(d) * w.sk + long(e) * w.se] : 0.f;
      }
  }

  Rows<KP, NT, VEC> rx, ry;
  float zn[2][4];
  float gn;
  bool fn;
  auto fetch = [&](int s0) {
    if constexpr (!LOCAL) rx.issue(w.x, bx, px, s0, n, dir, tid);
    ry.issue(w.y, by, py, s0, n, dir, tid);
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int s = s0 + jb * 16 + 4 * lg + r;
        zn[jb][r] = s < n && e < E ? w.z.p[bz + long(dir) * s * pz + e] : 0.f;
      }
    const int s = s0 + (lane & 31);
    gn = 0.f;
    fn = false;
    if (s < n) step_decay(a, td + dir * s, b, h, gn, fn);
  };
  fetch(0);
  float total = 1.f;
  int buf = 0;
  for (int s0 = 0; s0 < n; s0 += kChunk, buf ^= 1) {
    float* X = lx[LOCAL ? 0 : buf];
    float* Y = ly[buf];
    float* P = lp[LOCAL ? 0 : buf];
    if constexpr (!LOCAL) rx.store(X, tid);
    ry.store(Y, tid);
    float z[2][4];
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) z[jb][r] = zn[jb][r];
    Decays dc;
    dc.form(gn, fn, lane);
    if (s0 + kChunk < n) fetch(s0 + kChunk);
    __syncthreads();

    if constexpr (!LOCAL) {
      // Weights of the chunk's own steps: the three 16 x 16 blocks that have any.
      for (int f = wave; f < 3; f += NW) {
        const int ri = f > 0, cj = f > 1;
        f32x4 p = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          if (k >= nkb) break;
          const f32x4 xa = *reinterpret_cast<const f32x4*>(X + (ri * 16 + lr) * PX + k * 16 + 4 * lg);
          const f32x4 yb = *reinterpret_cast<const f32x4*>(Y + (cj * 16 + lr) * PX + k * 16 + 4 * lg);
#pragma unroll
          for (int r = 0; r < 4; ++r) p = mfma4(xa[r], yb[r], p);
        }
        const int j = cj * 16 + lr;
        const double cjv = __shfl(dc.c, j, 32);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = ri * 16 + 4 * lg + r;
          const double ci = __shfl(dc.c, i, 32);
          const int lo = __shfl(dc.lo, i, 32);
          P[i * PP + j] = j <= i && j >= lo ? p[r] * (expf(float(ci - cjv)) * w.alpha_out * w.alpha_pair) : 0.f;
        }
      }
      // What the entering state gives each row.
      f32x4 o[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) o[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        if (k >= nkb) break;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const f32x4 xa = *reinterpret_cast<const f32x4*>(X + (f * 16 + lr) * PX + k * 16 + 4 * lg);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[f] = mfma4(xa[r], S[k][r], o[f]);
        }
      }
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = f * 16 + 4 * lg + r;
          const float in = __shfl(dc.into, i, 32);
          const int lo = __shfl(dc.lo, i, 32);
          o[f][r] = lo < 0 ? o[f][r] * (in * w.alpha_out) : 0.f;
        }
      __syncthreads();
      bool odd = false;
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd = odd || !finite(z[jb][r]);
      if (!__any(odd)) {
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int f = jb; f < 2; ++f) {
            const f32x4 pa = *reinterpret_cast<const f32x4*>(P + (f * 16 + lr) * PP + jb * 16 + 4 * lg);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[f] = mfma4(pa[r], z[jb][r], o[f]);
          }
      } else {
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll 1
            for (int m = 0; m < 4; ++m) {
              const int j = jb * 16 + 4 * m + r;
              const float zj = __shfl(z[jb][r], lr + 16 * m, 64);
#pragma unroll
              for (int f = jb; f < 2; ++f)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const int i = f * 16 + 4 * lg + q, lo = __shfl(dc.lo, i, 32);
                  if (j <= i && j >= lo) o[f][q] += P[i * PP + j] * zj;
                }
            }
      }
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int s = s0 + f * 16 + 4 * lg + r;
          if (s < n && e < E) w.out[bo + long(dir) * s * po + e] = o[f][r];
        }
      if (w.dot.p) {
        const long bd = base(w.dot), pd = pitch(w.dot);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int s = s0 + f * 16 + 4 * lg + r;
            float d = s < n && e < E ? w.dot.p[bd + long(dir) * s * pd + e] * o[f][r] : 0.f;
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) d += __shfl_xor(d, m, 64);
            if (lr == 0 && s < n && wave * 16 < E)
              w.dots[(long(wave) * a.B * a.H + bh) * a.T + tb + dir * s] = d;
          }
      }
    }

    // The state on leaving the chunk.
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[k][r] = dc.first > 0 || dc.keep == 0.f ? 0.f : S[k][r] * dc.keep;
    total *= dc.keep;
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = jb * 16 + 4 * lg + r;
        const float lf = __shfl(dc.left, j, 32);
        z[jb][r] = j >= dc.first ? z[jb][r] * (lf * w.alpha_pair) : 0.f;
      }
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      if (k >= nkb) break;
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = jb * 16 + 4 * lg + r;
          float y = Y[j * PX + k * 16 + lr];
          if (dc.first > 0) y = j >= dc.first ? y : 0.f;
          S[k] = mfma4(y, z[jb][r], S[k]);
        }
    }
  }

  float* end = nullptr;
  float scale = 1.f;
  bool none = false;
  if constexpr (LOCAL) {
    end = a.added + (long(seg) * a.B * a.H + bh) * D * E;
    if (tid == 0) a.decays[long(seg) * a.B * a.H + bh] = total;
  } else if (w.end && (w.back ? seg == 0 : seg + 1 == a.nseg)) {
    end = w.end + long(bh) * D * E;
    if (w.end_decay) {
      float g;
      step_decay(a, 0, b, h, g, none);
      scale = expf(g);
    }
  }
  if (end) {
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = k * 16 + 4 * lg + r;
        if (d < D && e < E) end[long(d) * w.sk + long(e) * w.se] = none ? 0.f : S[k][r] * scale;
      }
  }
}

constexpr int kJoinThreads = 256;

// added[s] becomes the state on entering segment s, in the order of the sweep.
__global__ __launch_bounds__(kJoinThreads) void k_join(float* __restrict__ added, const float* __restrict__ decays,
                                                       const float* __restrict__ start, long BH, int DE, int nseg,
                                                       int back) {
  const long i = long(blockIdx.x) * kJoinThreads + threadIdx.x;
  if (i >= BH * DE) return;
  const long bh = i / DE;
  float run = start ? start[i] : 0.f;
  for (int q = 0; q < nseg; ++q) {
    const int s = back ? nseg - 1 - q : q;
    const float u = added[s * BH * DE + i], d = decays[s * BH + bh];
    added[s * BH * DE + i] = run;
    run = (d == 0.f ? 0.f : run * d) + u;
  }
}

// cross[s][bh] = <state before, gradient state after> at the end of segment s:
// the gradient of the log decays up to there from what lies beyond.
__global__ __launch_bounds__(kJoinThreads) void k_cross(SweepArgs a, const float* __restrict__ states,
                                                        const float* __restrict__ grads,
                                                        const float* __restrict__ final_state,
                                                        const float* __restrict__ final_grad, int DE,
                                                        float* __restrict__ cross) {
  __shared__ float red[kJoinThreads / 64];
  const long BH = long(a.B) * a.H, bh = blockIdx.x;
  const int s = int(blockIdx.y), b = int(bh / a.H), h = int(bh - long(b) * a.H);
  const bool last = s + 1 == a.nseg;
  const float* x = last ? final_state + bh * DE : states + ((s + 1) * BH + bh) * DE;
  const float* y = last ? final_grad : grads + s * BH * DE;
  float d = 0.f;
  if (y) {
    y += bh * DE;
    for (int i = threadIdx.x; i < DE; i += kJoinThreads) d += x[i] * y[i];
  }
  d = block_sum<kJoinThreads>(d, red);
  if (threadIdx.x) return;
  float g;
  bool reset;
  step_decay(a, (s + 1) * a.seg, b, h, g, reset);  // past the last step: no decay
  cross[s * BH + bh] = reset || !y ? 0.f : (last ? d : d * expf(g));
}

// dL/dg from the rows' products: a wavefront walks one head's segment back.
__global__ __launch_bounds__(64) void k_decay_grad(SweepArgs a, const float* __restrict__ qd, int nq,
                                                   const float* __restrict__ kd, int nk,
                                                   const float* __restrict__ cross, float* __restrict__ dg,
                                                   double* __restrict__ sums) {
  const long BH = long(a.B) * a.H, bh = blockIdx.x;
  const int s = int(blockIdx.y), lane = threadIdx.x, b = int(bh / a.H), h = int(bh - long(b) * a.H);
  const int t0 = s * a.seg, n = min(a.seg, a.T - t0);
  double carry = cross ? double(cross[s * BH + bh]) : 0.0, sum = 0.0;
  for (int e = n; e > 0; e -= 64) {
    const int t = t0 + e - 1 - lane;  // lane 0 the latest step
    const bool in = lane < e;
    double x = 0.0;
    float g = 0.f;
    bool reset = false;
    if (in) {
      for (int i = 0; i < nq; ++i) x += double(qd[(i * BH + bh) * a.T + t]);
      for (int i = 0; i < nk; ++i) x -= double(kd[(i * BH + bh) * a.T + t]);
      step_decay(a, t, b, h, g, reset);
    }
    // X of a step sums the terms from it to the end of its episode: those of
    // the lanes before it, down to the one after the last start among them.
    const uint64_t starts = __ballot(reset);
    const uint64_t before = lane ? starts & (~0ull >> (64 - lane)) : 0ull;
    const int lo = before ? 64 - __clzll(before) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(x, d, 64);
      if (lane - d >= lo) x += y;
    }
    if (!before) x += carry;
    if (reset) x = 0.0;
    if (in && dg) dg[(long(t) * a.B + b) * a.H + h] = float(x);
    if (in) sum += x;
    carry = __shfl(x, min(e, 64) - 1, 64);
  }
  if (sums) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m, 64);
    if (lane == 0) sums[s * BH + bh] = sum;
  }
}

// The gradient of a decay that all steps share: the sums of its head, in order.
__global__ __launch_bounds__(64) void k_decay_total(const double* __restrict__ sums, int H, long rows,
                                                    float* __restrict__ dg) {
  const int h = int(blockIdx.x), lane = threadIdx.x;
  double x = 0.0;
  for (long i = lane; i < rows; i += 64) x += sums[i * H + h];
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m, 64);
  if (lane == 0) dg[h] = float(x);
}

// Gradients of shared heads: the sum over the heads that share one, in order.
__global__ __launch_bounds__(256) void k_share_sum(const float* __restrict__ x, float* __restrict__ y, long n, int share,
                                                   int dim) {
  for (long i = long(blockIdx.x) * 256 + threadIdx.x; i < n; i += long(gridDim.x) * 256) {
    const long row = i / dim;
    const float* p = x + row * share * dim + (i - row * dim);
    float t = p[0];
    for (int s = 1; s < share; ++s) t += p[long(s) * dim];
    y[i] = t;
  }
}

// A single token: the state read, stepped and written once.  A workgroup takes
// one head of one lane; a thread W columns of every KG-th row.
struct StepArgs {
  const float *q, *k, *v, *g, *done;
  float *state, *out;
  int g_rows, B, H, share, K, V;
  float scale;
};
constexpr int kStepThreads = 256;

template <int W>
__global__ __launch_bounds__(kStepThreads) void k_token(StepArgs a) {
  __shared__ float part[kStepThreads * W];
  const int bh = int(blockIdx.x), b = bh / a.H, h = bh - b * a.H, G = a.H / a.share;
  const int cols = (a.V + W - 1) / W, groups = kStepThreads / cols;
  const int c = int(threadIdx.x) % cols, kg = int(threadIdx.x) / cols;
  const float g = a.g_rows ? a.g[long(b) * a.H + h] : a.g[h];
  const bool reset = (a.done && a.done[b] > 0.f) || g < kForget;
  const float keep = expf(g);
  const float* q = a.q + (long(b) * a.H + h) * a.K;
  const float* k = a.k + (long(b) * G + h / a.share) * a.K;
  const float* v = a.v + (long(b) * G + h / a.share) * a.V + c * W;
  float* S = a.state + long(bh) * a.K * a.V + c * W;
  float o[W], vv[W];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    o[j] = 0.f;
    vv[j] = kg < groups ? v[j] : 0.f;
  }
  if (kg < groups) {
    for (int d = kg; d < a.K; d += groups) {
      float* p = S + long(d) * a.V;
      const float kd = k[d], qd = q[d];
      float s[W];
      if constexpr (W == 4) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = t[j];
      } else {
        s[0] = *p;
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        s[j] = (reset ? 0.f : s[j] * keep) + kd * vv[j];
        o[j] += qd * s[j];
      }
      if constexpr (W == 4) *reinterpret_cast<f32x4*>(p) = f32x4{s[0], s[1], s[2], s[3]};
      else *p = s[0];
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) part[threadIdx.x * W + j] = o[j];
  __syncthreads();
  for (int e = threadIdx.x; e < a.V; e += kStepThreads) {
    float t = 0.f;
    for (int i = 0; i < groups; ++i) t += part[(i * cols + e / W) * W + e % W];
    a.out[long(bh) * a.V + e] = t * a.scale;
  }
}

// ------------------------------------------------------------------ host ---

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Every row of the operand starts on 16 bytes.
bool wide(const Operand& o) { return !o.p || (o.dim % 4 == 0 && aligned16(o.p)); }

template <bool LOCAL>
int launch_sweeps(ttrl_ctx* ctx, const SweepArgs& a, int count, const char* name) {
  int D = 0, E = 0;
  bool vec = true;
  for (int i = 0; i < count; ++i) {
    D = std::max(D, a.s[i].x.dim);
    E = std::max(E, a.s[i].z.dim);
    vec = vec && wide(a.s[i].y) && (LOCAL || wide(a.s[i].x));
  }
  const dim3 grid(unsigned(a.B) * unsigned(a.H), unsigned(a.nseg), unsigned(count));
  auto go = [&](auto kp, auto nw) {
    constexpr int KP = decltype(kp)::value, NW = decltype(nw)::value;
    if (vec) hipLaunchKernelGGL((k_sweep<KP, NW, true, LOCAL>), grid, dim3(64 * NW), 0, stream_of(ctx), a);
    else hipLaunchKernelGGL((k_sweep<KP, NW, false, LOCAL>), grid, dim3(64 * NW), 0, stream_of(ctx), a);
  };
  auto width = [&](auto kp) {
    if (E <= 32) go(kp, std::integral_constant<int, 2>{});
    else if (E <= 64) go(kp, std::integral_constant<int, 4>{});
    else go(kp, std::integral_constant<int, 8>{});
  };
  if (D <= 32) width(std::integral_constant<int, 32>{});
  else if (D <= 64) width(std::integral_constant<int, 64>{});
  else width(std::integral_constant<int, 128>{});
  return check_launch(name);
}

// Segments of a sequence: enough workgroups for the 256 compute units, and
// whole chunks.
struct Plan {
  int seg, nseg;
};
Plan plan_of(int T, long BH) {
  const long want = std::max(1L, (1024 + BH - 1) / std::max(1L, BH));
  const long chunks = std::max(1L, long(T + kChunk - 1) / kChunk);
  const long per = (chunks + want - 1) / want;
  const int seg = int(per * kChunk);
  return {seg, std::max(1, (T + seg - 1) / seg)};
}

struct Space {  // floats of the caller's buffers, in order
  long states, decays, grads, gdecays, cross, qdots, kdots, dk, dv, sums;
};

int check_desc(const ttrl_linear_attention_desc* d, const char* name) {
  TTRL_REQUIRE(d, "%s: null description", name);
  TTRL_REQUIRE(d->T >= 0 && d->B >= 0 && d->H > 0 && d->kv_heads > 0 && d->H % d->kv_heads == 0,
               "%s: %d heads do not share %d key/value heads evenly (T=%d, B=%d)", name, d->H, d->kv_heads, d->T, d->B);
  TTRL_REQUIRE(d->K > 0 && d->V > 0 && d->K <= kMaxHead && d->V <= kMaxHead,
               "%s: head widths of 1 to %d are supported, got K=%d, V=%d", name, kMaxHead, d->K, d->V);
  TTRL_REQUIRE(long(d->B) * d->H <= 0x7fffffffL / 2, "%s: %d sequences of %d heads are too many", name, d->B, d->H);
  TTRL_REQUIRE(plan_of(d->T, long(d->B) * d->H).nseg <= 65535, "%s: %d steps are too many", name, d->T);
  return TTRL_OK;
}

SweepArgs args_of(const ttrl_linear_attention_desc* d) {
  SweepArgs a{};
  const Plan p = plan_of(d->T, long(d->B) * d->H);
  a.g = d->log_decay;
  a.done = d->done;
  a.g_rows = d->decay_steps;
  a.T = d->T;
  a.B = d->B;
  a.H = d->H;
  a.seg = p.seg;
  a.nseg = p.nseg;
  return a;
}

Space space_of(const ttrl_linear_attention_desc* d, int nseg) {
  const long BH = long(d->B) * d->H, DE = long(d->K) * d->V, S = nseg, rows = long(d->T) * d->B;
  const bool shared = d->H != d->kv_heads;
  auto even = [](long n) { return (n + 63) / 64 * 64; };
  Space s{};
  s.states = S > 1 ? even(S * BH * DE) : 0;
  s.decays = S > 1 ? even(S * BH) : 0;
  s.grads = s.states;
  s.gdecays = s.decays;
  s.cross = even(S * BH);
  s.qdots = even(long((d->K + 15) / 16) * BH * d->T);
  s.kdots = s.qdots;
  s.dk = shared ? even(rows * d->H * d->K) : 0;
  s.dv = shared ? even(rows * d->H * d->V) : 0;
  s.sums = even(2 * S * BH);
  return s;
}

}  // namespace
}  // namespace ttrl

using namespace ttrl;

extern "C" {

int ttrl_linear_attention_space(const ttrl_linear_attention_desc* d, long* saved_floats, long* work_floats) {
  if (int rc = check_desc(d, "ttrl_linear_attention_space")) return rc;
  TTRL_REQUIRE(saved_floats && work_floats, "ttrl_linear_attention_space: null output");
  const Space s = space_of(d, plan_of(d->T, long(d->B) * d->H).nseg);
  *saved_floats = s.states + s.decays;
  *work_floats = s.grads + s.gdecays + s.cross + s.qdots + s.kdots + s.dk + s.dv + s.sums;
  return TTRL_OK;
}

int ttrl_linear_attention_forward(ttrl_ctx* ctx, const ttrl_linear_attention_desc* d) {
  const char* name = "ttrl_linear_attention_forward";
  if (int rc = check_desc(d, name)) return rc;
  TTRL_REQUIRE(ctx, "%s: null context", name);
  if (d->B == 0) return TTRL_OK;
  const long BH = long(d->B) * d->H, DE = long(d->K) * d->V;
  TTRL_REQUIRE(d->final_state, "%s: null final state", name);
  if (d->T == 0) {
    const size_t bytes = size_t(BH) * size_t(DE) * sizeof(float);
    return d->state ? ttrl_d2d(ctx, d->final_state, d->state, bytes) : ttrl_fill_f32(ctx, d->final_state, 0.f, BH * DE);
  }
  TTRL_REQUIRE(d->q && d->k && d->v && d->log_decay && d->out, "%s: null operand", name);
  SweepArgs a = args_of(d);
  const int share = d->H / d->kv_heads;
  Sweep& s = a.s[0];
  s.x = {d->q, d->H, d->K, 1};
  s.y = {d->k, d->kv_heads, d->K, share};
  s.z = {d->v, d->kv_heads, d->V, share};
  s.out = d->out;
  s.start = d->state;
  s.end = d->final_state;
  s.sk = d->V;
  s.se = 1;
  s.alpha_out = d->scale;
  s.alpha_pair = 1.f;
  if (a.nseg > 1) {
    TTRL_REQUIRE(d->saved, "%s: null saved states", name);
    const Space sp = space_of(d, a.nseg);
    a.added = d->saved;
    a.decays = d->saved + sp.states;
    if (int rc = launch_sweeps<true>(ctx, a, 1, name)) return rc;
    hipLaunchKernelGGL(k_join, dim3(ceil_div(BH * DE, kJoinThreads)), dim3(kJoinThreads), 0, stream_of(ctx), a.added,
                       a.decays, d->state, BH, int(DE), a.nseg, 0);
    if (int rc = check_launch(name)) return rc;
    s.start = a.added;
    s.start_all = 1;
  }
  return launch_sweeps<false>(ctx, a, 1, name);
}

int ttrl_linear_attention_backward(ttrl_ctx* ctx, const ttrl_linear_attention_desc* d) {
  const char* name = "ttrl_linear_attention_backward";
  if (int rc = check_desc(d, name)) return rc;
  TTRL_REQUIRE(ctx, "%s: null context", name);
  const long BH = long(d->B) * d->H, DE = long(d->K) * d->V;
  if (d->T == 0 || d->B == 0) {
    if (d->dlog_decay && !d->decay_steps)
      if (int rc = ttrl_fill_f32(ctx, d->dlog_decay, 0.f, d->H)) return rc;
    if (!d->dstate || d->B == 0) return TTRL_OK;
    return d->dfinal ? ttrl_d2d(ctx, d->dstate, d->dfinal, size_t(BH) * size_t(DE) * sizeof(float))
                     : ttrl_fill_f32(ctx, d->dstate, 0.f, BH * DE);
  }
  TTRL_REQUIRE(d->q && d->k && d->v && d->log_decay && d->dout && d->work, "%s: null operand", name);
  TTRL_REQUIRE(d->dq && d->dk && d->dv, "%s: dq, dk and dv are all written", name);
  SweepArgs a = args_of(d);
  const Space sp = space_of(d, a.nseg);
  const int share = d->H / d->kv_heads;
  float* at = d->work;
  auto take = [&](long n) {
    float* p = at;
    at += n;
    return p;
  };
  float *grads = take(sp.grads), *gdecays = take(sp.gdecays), *cross = take(sp.cross), *qdots = take(sp.qdots),
        *kdots = take(sp.kdots), *dkh = take(sp.dk), *dvh = take(sp.dv), *sums = take(sp.sums);
  const Operand q{d->q, d->H, d->K, 1}, k{d->k, d->kv_heads, d->K, share}, v{d->v, d->kv_heads, d->V, share},
      go{d->dout, d->H, d->V, 1};
  const bool cut = a.nseg > 1;
  TTRL_REQUIRE(!cut || d->saved, "%s: null saved states", name);

  Sweep dv{};  // state G, (K, V)
  dv.x = k;
  dv.y = q;
  dv.z = go;
  dv.out = share > 1 ? dvh : d->dv;
  dv.start = d->dfinal;
  dv.end = d->dstate;
  dv.end_decay = 1;
  dv.sk = d->V;
  dv.se = 1;
  dv.back = 1;
  dv.alpha_out = 1.f;
  dv.alpha_pair = d->scale;
  if (cut) {
    a.s[0] = dv;
    a.added = grads;
    a.decays = gdecays;
    if (int rc = launch_sweeps<true>(ctx, a, 1, name)) return rc;
    hipLaunchKernelGGL(k_join, dim3(ceil_div(BH * DE, kJoinThreads)), dim3(kJoinThreads), 0, stream_of(ctx), grads,
                       gdecays, d->dfinal, BH, int(DE), a.nseg, 1);
    if (int rc = check_launch(name)) return rc;
    dv.start = grads;
    dv.start_all = 1;
  }
  Sweep dk = dv;  // state G^T, (V, K)
  dk.x = v;
  dk.y = go;
  dk.z = q;
  dk.out = share > 1 ? dkh : d->dk;
  dk.end = nullptr;
  dk.sk = 1;
  dk.se = d->V;
  Sweep dq{};  // state S^T, (V, K)
  dq.x = go;
  dq.y = v;
  dq.z = k;
  dq.out = d->dq;
  dq.start = cut ? d->saved : d->state;
  dq.start_all = cut;
  dq.sk = 1;
  dq.se = d->V;
  dq.alpha_out = d->scale;
  dq.alpha_pair = 1.f;
  if (d->dlog_decay) {
    dq.dot = q;
    dq.dots = qdots;
    dk.dot = k;
    dk.dots = kdots;
  }
  a.s[0] = dq;
  a.s[1] = dk;
  a.s[2] = dv;
  if (int rc = launch_sweeps<false>(ctx, a, 3, name)) return rc;

  if (d->dlog_decay) {
    const dim3 each(unsigned(BH), unsigned(a.nseg));
    const bool crossing = cut || d->dfinal;
    if (crossing) {
      TTRL_REQUIRE(!d->dfinal || d->final_state, "%s: the final state's gradient needs the final state", name);
      hipLaunchKernelGGL(k_cross, each, dim3(kJoinThreads), 0, stream_of(ctx), a, d->saved, grads, d->final_state,
                         d->dfinal, int(DE), cross);
      if (int rc = check_launch(name)) return rc;
    }
    double* total = d->decay_steps ? nullptr : reinterpret_cast<double*>(sums);
    const int parts = (d->K + 15) / 16;
    hipLaunchKernelGGL(k_decay_grad, each, dim3(64), 0, stream_of(ctx), a, qdots, parts, kdots, parts,
                       crossing ? cross : nullptr, d->decay_steps ? d->dlog_decay : nullptr, total);
    if (int rc = check_launch(name)) return rc;
    if (total) {
      hipLaunchKernelGGL(k_decay_total, dim3(unsigned(d->H)), dim3(64), 0, stream_of(ctx), total, d->H,
                         long(a.nseg) * d->B, d->dlog_decay);
      if (int rc = check_launch(name)) return rc;
    }
  }
  if (share > 1) {
    const long rows = long(d->T) * d->B * d->kv_heads;
    auto sum = [&](const float* x, float* y, int dim) {
      const long n = rows * dim;
      hipLaunchKernelGGL(k_share_sum, dim3(unsigned(std::min(4096L, (n + 255) / 256))), dim3(256), 0, stream_of(ctx), x,
                         y, n, share, dim);
      return check_launch(name);
    };
    if (int rc = sum(dkh, d->dk, d->K)) return rc;
    if (int rc = sum(dvh, d->dv, d->V)) return rc;
  }
  return TTRL_OK;
}

int ttrl_linear_attention_token(ttrl_ctx* ctx, int B, int H, int kv_heads, int K, int V, const float* q, const float* k,
                                const float* v, const float* log_decay, int decay_rows, const float* done, float scale,
                                float* state, float* out) {
  const char* name = "ttrl_linear_attention_token";
  TTRL_REQUIRE(ctx, "%s: null context", name);
  TTRL_REQUIRE(B >= 0 && H > 0 && kv_heads > 0 && H % kv_heads == 0,
               "%s: %d heads do not share %d key/value heads evenly (B=%d)", name, H, kv_heads, B);
  TTRL_REQUIRE(K > 0 && V > 0 && K <= kMaxHead && V <= kMaxHead,
               "%s: head widths of 1 to %d are supported, got K=%d, V=%d", name, kMaxHead, K, V);
  TTRL_REQUIRE(long(B) * H <= 0x7fffffffL / 2, "%s: %d lanes of %d heads are too many", name, B, H);
  if (B == 0) return TTRL_OK;
  TTRL_REQUIRE(q && k && v && log_decay && state && out, "%s: null operand", name);
  const StepArgs a{q, k, v, log_decay, done, state, out, decay_rows, B, H, H / kv_heads, K, V, scale};
  const dim3 grid(unsigned(B) * unsigned(H));
  if (V % 4 == 0 && aligned16(state) && aligned16(v))
    hipLaunchKernelGGL(k_token<4>, grid, dim3(kStepThreads), 0, stream_of(ctx), a);
  else
    hipLaunchKernelGGL(k_token<1>, grid, dim3(kStepThreads), 0, stream_of(ctx), a);
  return check_launch(name);
}

}  // extern "C"
