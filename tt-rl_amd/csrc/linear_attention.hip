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
// For the decay, X_t = a_t <S_{t-1}, G_t> = dL/dg_t is the sum over pairs of steps
// i >= t > j of what step j's key and value give step i's output, and 0 where an
// episode starts (k_decay_grad).
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
// added[s]), and the sweeps then start from the joined states.  Otherwise a
// sweep runs through and leaves the state at every segment's start.  Either
// way the backward has S and G at the ends of every segment, and the sum for
// dL/dg starts again there from <S, G>.
//
// What it measured (forward and backward where not said; us, and every operand
// read and every result written once at a large copy's 4.7 TB/s): 1024 steps of 32
// sequences, 8 heads of 64 x 64: 373 (116), its sweeps 122 and 258, bound by the
// wavefronts' chain of LDS reads and FP32 products of 32 cycles, one after another
// at one or three wavefronts a SIMD: a chunk issues 1.4 times the products of the
// recurrence forward and 2.1 times backward, and they run at 48 and 69 TFLOP/s where
// a large FP32 product reaches 153.  4001 x 2 x 6 of 40 x 72: 181 (14), 21 segments
// that each walk six chunks one after another, ten launches; 32 x 16 x 8 of 64 x 64:
// 31 (3), four launches; 2048 x 8 x 8 of 128 x 128 forward 206 (59), a third of it the
// first launch; one token of 1000 lanes 51 (57: part of the states stays in the
// last-level cache), of one lane 3.4, a launch.
//
// Precision: products, sums and states are FP32; the sums of log decays are in
// double, and each weight is the exponential of a difference of two of them, so
// a strong decay in a chunk takes nothing from the weights after it.  Errors
// against float64, of the norm: outputs and gradients of q, k, v and the state 1.3e-7
// to 2.7e-7; of log decays 3e-7 to 6e-7 where every step has its own, and 3e-7 to 2e-6
// in the median where all steps share one, whose terms cancel by as much as chance
// has it (a formula of chunked products by a library and its autograd: 1.2e-7 to
// 1e-6).
//
// Values that are not finite stay in their episode and behind their step: a
// masked weight is selected, never multiplied, and a chunk whose z holds such
// values forms its inner sums over the allowed steps alone.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

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
  float* out;          // (T, B, H, E)
  Operand dot;         // rows to multiply the output's rows with, or null
  float* dots;         // [E / 16][B * H][2][T] partial sums of those products, 16 columns each: whole, and of
                       // what the entering state gave
  const float* start;  // state on entering a segment: [segment][B * H][D * E], or of the first one only
  int start_all;       // one for every segment
  float* marks;        // where a sweep that runs through leaves the state at the segments' starts, or null
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
  int run;        // steps a sweep takes: seg, or T where it runs through
  float* added;   // first launch: [segment][B * H][D * E]
  float* decays;  // first launch: [segment][B * H]
};

__device__ __forceinline__ f32x4 mfma4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Memory goes through buffer resources, whose range check replaces branches:
// an offset past the range loads zeros and drops a store.  A chunk's resource
// starts at its earliest step and ends with the last step there is, so rows
// past the end are out of range by themselves; columns past the width get kOut.
constexpr uint32_t kOut = 0x80000000u;
constexpr int kFlags = 0x00020000;  // raw 32-bit dwords
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(a));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(hi) << 32 | lo), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), kFlags);
}
__device__ __forceinline__ float load1(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 load4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ void store1(__amdgpu_buffer_rsrc_t r, uint32_t off, float v) {
  __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, off, 0, 0);
}

// The sum over a row of 16 lanes, in every one of them.
__device__ __forceinline__ float row_sum(float x) {
#define TTRL_ROW_ROR(n) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + n, 0xf, 0xf, true))
  TTRL_ROW_ROR(8);
  TTRL_ROW_ROR(4);
  TTRL_ROW_ROR(2);
  TTRL_ROW_ROR(1);
#undef TTRL_ROW_ROR
  return x;
}

// One head's rows of an operand: chunk c's resource.
struct Rows {
  const float* p;  // step 0
  uint32_t pitch;  // bytes from one step to the next
  uint32_t width;  // bytes of a row
  __device__ __forceinline__ Rows(const Operand& o, int B, int b, int h) {
    p = o.p + (long(b) * o.heads + h / o.share) * o.dim;
    pitch = uint32_t(B) * uint32_t(o.heads) * uint32_t(o.dim) * 4u;
    width = uint32_t(o.dim) * 4u;
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk(int t, int n) const {  // n steps from t on
    return resource(reinterpret_cast<const char*>(p) + long(t) * pitch, n > 0 ? uint32_t(n - 1) * pitch + width : 0u);
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

// x of the lane N before or after, within 16 lanes; 0 where there is none.
template <int CONTROL>
__device__ __forceinline__ double of_row(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u)), CONTROL, 0xf, 0xf, true));
  const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u >> 32)), CONTROL, 0xf, 0xf, true));
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
template <int N>
__device__ __forceinline__ double before(double x) { return of_row<0x110 + N>(x); }
template <int N>
__device__ __forceinline__ double after(double x) { return of_row<0x100 + N>(x); }
__device__ __forceinline__ double of_lane(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(uint32_t(u), lane), hi = __builtin_amdgcn_readlane(uint32_t(u >> 32), lane);
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// 2^x, zero below float32's normal range.
__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }

// A chunk's decays, formed by one wavefront, row i of the sweep's order in lane i.
struct Decays {
  double c[kChunk];    // sum of the decays' logarithms (to base 2) since the chunk's or the episode's start
  float into[kChunk];  // weight of the state on entering the chunk (where lo < 0)
  float left[kChunk];  // weight of the row in the state on leaving it (from `first` on)
  int lo[kChunk];      // the episode's first row in the chunk, -1: before it
  float keep;          // weight of the entering state in the leaving one (0: none)
  int first;           // first row that the leaving state holds
  __device__ __forceinline__ void form(float g, bool reset, int lane) {
    const int i = lane & 31;
    const uint32_t starts = uint32_t(__ballot(reset));
    const uint32_t m = starts & (0xffffffffu >> (31 - i));
    const int l = m ? 31 - __clz(m) : -1, from = max(l, 0);
    double s = reset ? 0.0 : double(g) * 1.4426950408889634074, t;
    // Sums over 1, 2, 4, 8 and 16 lanes that end here, down to the episode's start.
    t = before<1>(s);
    s = i - 1 >= from ? s + t : s;
    t = before<2>(s);
    s = i - 2 >= from ? s + t : s;
    t = before<4>(s);
    s = i - 4 >= from ? s + t : s;
    t = before<8>(s);
    s = i - 8 >= from ? s + t : s;
    t = of_lane(s, 15);
    s = i >= 16 && from < 16 ? s + t : s;
    const double e = of_lane(s, 31);
    const int le = starts ? 31 - __clz(starts) : -1;
    const float in = power(float(s)), out = power(float(e - s)), all = power(float(e));
    if (lane < kChunk) {
      c[i] = s;
      lo[i] = l;
      into[i] = in;
      left[i] = out;
    }
    if (lane == 0) {
      keep = le < 0 ? all : 0.f;
      first = max(le, 0);
    }
  }
};
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
template <class V>
__device__ __forceinline__ V lds_at(const void* p) { return *reinterpret_cast<const V*>(p); }

// 32 rows of an operand on their way into LDS, row r of the sweep's order.
template <int KP, int NT, bool VEC>
struct Stage {
  static constexpr int W = VEC ? 4 : 1, CH = KP / W, PER = (kChunk * CH + NT - 1) / NT;
  static constexpr bool WHOLE = kChunk * CH % NT == 0;
  uint32_t off[PER];
  f32x4 v4[VEC ? PER : 1];
  float v1[VEC ? 1 : PER];
  __device__ __forceinline__ void init(const Rows& o, int back, int tid) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + u * NT, r = i / CH, c = i % CH * W;
      off[u] = (WHOLE || r < kChunk) && uint32_t(c) * 4u < o.width ? uint32_t(back ? kChunk - 1 - r : r) * o.pitch + uint32_t(c) * 4u : kOut;
    }
  }
  __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t r) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if constexpr (VEC) v4[u] = load4(r, off[u]);
      else v1[u] = load1(r, off[u]);
    }
  }
  __device__ __forceinline__ void store(float* lds, int tid) const {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + u * NT, r = i / CH, c = i % CH * W;
      if (!WHOLE && r >= kChunk) continue;
      if constexpr (VEC) *reinterpret_cast<f32x4*>(lds + r * (KP + 4) + c) = v4[u];
      else lds[r * (KP + 4) + c] = v1[u];
    }
  }
};

// A scalar that stays in registers: without this the compiler reads kernel
// arguments again where it needs them, a wait each time.
template <class T>
__device__ __forceinline__ void pin(T& x) {
  asm volatile("" : "+s"(x));
}

// LOCAL: the first launch, what a segment adds to the state.
template <int KP, int NW, bool VEC, bool LOCAL>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(KP >= 96 ? 2 : 3))) void k_sweep(
    SweepArgs a) {
  constexpr int NT = 64 * NW, KB = KP / 16, PX = KP + 4, PP = kChunk + 4;
  __shared__ __attribute__((aligned(16))) float lx[LOCAL ? 1 : 2][LOCAL ? 4 : kChunk * PX];
  __shared__ __attribute__((aligned(16))) float ly[2][kChunk * PX];
  __shared__ __attribute__((aligned(16))) float lp[LOCAL ? 1 : 2][LOCAL ? 4 : kChunk * PP];
  __shared__ __attribute__((aligned(16))) Decays ld[2];
  const Sweep& w = a.s[blockIdx.z];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = int(blockIdx.x), b = bh / a.H, h = bh - b * a.H, run = int(blockIdx.y);
  const int t0 = run * a.run, n = min(a.run, a.T - t0);
  int back = w.back, D = w.x.dim, E = w.z.dim, sk = w.sk, se = w.se;
  float alpha_out = w.alpha_out, alpha_pair = w.alpha_pair;
  float* marks = w.marks;
  const float* done = a.done;
  int g_rows = a.g_rows;
  pin(done), pin(g_rows), pin(back), pin(D), pin(E), pin(sk), pin(se), pin(alpha_out), pin(alpha_pair), pin(marks);
  const int nch = (n + kChunk - 1) / kChunk;
  const int e = wave * 16 + lr;
  const bool cols = wave * 16 < E;  // uniform: this wavefront has columns of the state
  const long BH = long(a.B) * a.H;

  const Rows rx(w.x, a.B, b, h), ry(w.y, a.B, b, h), rz(w.z, a.B, b, h);
  const Rows ro(Operand{w.out, a.H, E, 1}, a.B, b, h);
  const bool dotted = !LOCAL && w.dot.p;
  const Rows rd(dotted ? w.dot : w.z, a.B, b, h);
  Stage<KP, NT, VEC> sx, sy;
  if constexpr (!LOCAL) sx.init(rx, back, tid);
  sy.init(ry, back, tid);
  // Rows jb * 16 + 4 * lg + r of the sweep's order, this lane's column; formed
  // where they are used (kept over the loop they would take more registers
  // than the state), from the first by steps of one row.
  struct Offsets {
    uint32_t at[2][4];
  };
  auto offsets = [&](uint32_t pitch) __attribute__((always_inline)) {
    int q = lg;
    asm volatile("" : "+v"(q));
    const uint32_t by = back ? 0u - pitch : pitch, top = back ? uint32_t(kChunk - 1) * pitch : 0u;
    Offsets f;
    f.at[0][0] = top + (e < E ? uint32_t(4 * q) * by + uint32_t(e) * 4u : kOut);
    f.at[1][0] = f.at[0][0] + 16u * by;
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 1; r < 4; ++r) f.at[jb][r] = f.at[jb][r - 1] + by;
    return f;
  };
  auto element = [&](int q, int k, int r) __attribute__((always_inline)) {
    const int d = k * 16 + 4 * q + r;
    return (d < D) & (e < E) ? uint32_t(d * sk + e * se) * 4u : kOut;
  };
  auto chunk_at = [&](int i) __attribute__((always_inline)) { return back ? nch - 1 - i : i; };  // i-th of the sweep
  // A chunk's loads on their way; every wavefront takes the same ones, the
  // decays' a chunk earlier than the rows', so that none is waited for early.
  float zn[2][4], gn, dn;
  const uint32_t gp = g_rows ? uint32_t(a.B) * uint32_t(a.H) * 4u : 0u, dp = uint32_t(a.B) * 4u;
  const int shift = lane & 31, step = back ? kChunk - shift : shift;  // backwards a step's decay is that of the step after it
  auto fetch_decays = [&](int i) __attribute__((always_inline)) {
    const int t = t0 + (i < nch ? chunk_at(i) * kChunk : 0), left = i < nch ? min(a.T - t, kChunk + 1) : 0;
    const float* g = a.g + (g_rows ? (long(t) * a.B + b) * a.H + h : long(h));
    gn = load1(resource(g, left > 0 ? uint32_t(left - 1) * gp + 4u : 0u), uint32_t(step) * gp);
    dn = load1(resource(done ? done + long(t) * a.B + b : g, done && left > 0 ? uint32_t(left - 1) * dp + 4u : 0u),
               uint32_t(step) * dp);
  };
  auto form = [&](Decays& d, int i, float g, float ended) __attribute__((always_inline)) {
    const int s = chunk_at(i) * kChunk + step;
    const bool in = (i < nch) & (s < n + back) & (t0 + s < a.T);
    d.form(in ? g : 0.f, in & ((ended > 0.f) | (g < kForget)), lane);
  };
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int s0 = i < nch ? chunk_at(i) * kChunk : 0, t = t0 + s0, m = i < nch ? min(n - s0, kChunk) : 0;
    if constexpr (!LOCAL) sx.issue(rx.chunk(t, m));
    sy.issue(ry.chunk(t, m));
    const __amdgpu_buffer_rsrc_t r2 = rz.chunk(t, m);
    const Offsets f = offsets(rz.pitch);
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) zn[jb][r] = load1(r2, f.at[jb][r]);
    fetch_decays(i + 1);
  };
  f32x4 S[KB];
  fetch_decays(0);
  float gc = gn, ec = dn;
  fetch(0);
  {
    const bool any = !LOCAL && w.start && (w.start_all || (back ? t0 + n == a.T : t0 == 0));
    const __amdgpu_buffer_rsrc_t r0 =
        resource(any ? w.start + (w.start_all ? run * BH + bh : long(bh)) * D * E : w.y.p, any ? uint32_t(D) * E * 4u : 0);
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[k][r] = load1(r0, element(lg, k, r));
  }
  auto leave = [&](float* to, float scale, bool none) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r0 = resource(to, uint32_t(D) * E * 4u);
    int q = lg;
    asm volatile("" : "+v"(q));
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) store1(r0, element(q, k, r), none ? 0.f : S[k][r] * scale);
  };
  if (wave == 0) form(ld[0], 0, gc, ec);

  float total = 1.f;
  for (int i = 0; i < nch; ++i) {
    const int c = chunk_at(i), buf = i & 1;
    float* X = lx[LOCAL ? 0 : buf];
    float* Y = ly[buf];
    float* P = lp[LOCAL ? 0 : buf];
    const Decays& dc = ld[buf];
    if constexpr (!LOCAL) {
      sx.store(X, tid);
      if (marks && (back ? i == 0 || (c + 1) * kChunk % a.seg == 0 : c * kChunk % a.seg == 0))
        leave(marks + (c * kChunk / a.seg * BH + bh) * D * E, 1.f, false);
    }
    sy.store(Y, tid);
    float z[2][4];
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        z[jb][r] = zn[jb][r];
        asm volatile("" : "+v"(z[jb][r]));
      }
    gc = gn;
    ec = dn;
    asm volatile("" : "+v"(gc), "+v"(ec));  // moved before the loads below
    fetch(i + 1);
    __syncthreads();
    if (wave == 0) form(ld[buf ^ 1], i + 1, gc, ec);

    const int t = t0 + c * kChunk, m = min(n - c * kChunk, kChunk);
    float d[2][4];
    if (dotted) {
      const __amdgpu_buffer_rsrc_t r3 = rd.chunk(t, m);
      const Offsets at = offsets(rd.pitch);
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) d[f][r] = load1(r3, at.at[f][r]);
    }
    // The rows' products with d, each in one lane: lane `from` + 4 f + r of a row
    // of 16 has that of row f * 16 + 4 * lg + r.
    float dots = 0.f;
    auto form_dots = [&](int from, const f32x4(&o)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float sum = row_sum(e < E ? d[f][r] * o[f][r] : 0.f);
          dots = lr == from + 4 * f + r ? sum : dots;
        }
    };

    if constexpr (!LOCAL) {
      // Weights of the chunk's own rows: the three 16 x 16 blocks that have
      // any, by the last wavefronts (the ones without columns, if there are).
      for (int f = NW - 1 - wave; f < 3; f += NW) {
        const int ri = f > 0, cj = f > 1, j = cj * 16 + lr, row = ri * 16 + 4 * lg;
        const f64x2 c01 = lds_at<f64x2>(dc.c + row), c23 = lds_at<f64x2>(dc.c + row + 2);
        const double cj0 = dc.c[j];
        const i32x4 lo = lds_at<i32x4>(dc.lo + row);
        f32x4 p[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          const f32x4 xa = lds_at<f32x4>(X + (ri * 16 + lr) * PX + k * 16 + 4 * lg);
          const f32x4 yb = lds_at<f32x4>(Y + (cj * 16 + lr) * PX + k * 16 + 4 * lg);
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r & 1] = mfma4(xa[r], yb[r], p[r & 1]);
        }
        const double cr[4] = {c01.x, c01.y, c23.x, c23.y};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = (p[0][r] + p[1][r]) * (power(float(cr[r] - cj0)) * (alpha_out * alpha_pair));
          asm volatile("" : "+v"(x));  // a select, not a branch round the exponential
          P[(row + r) * PP + j] = (j <= row + r) & (j >= lo[r]) ? x : 0.f;
        }
      }
      // What the entering state gives each row.
      f32x4 o[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) o[f] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (cols) {
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          f32x4 xa[2];
#pragma unroll
          for (int f = 0; f < 2; ++f) xa[f] = lds_at<f32x4>(X + (f * 16 + lr) * PX + k * 16 + 4 * lg);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int f = 0; f < 2; ++f) o[f] = mfma4(xa[f][r], S[k][r], o[f]);
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const i32x4 lo = lds_at<i32x4>(dc.lo + f * 16 + 4 * lg);
          const f32x4 in = lds_at<f32x4>(dc.into + f * 16 + 4 * lg);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = o[f][r] * (in[r] * alpha_out);
            o[f][r] = lo[r] < 0 ? x : 0.f;
          }
        }
        if (dotted) form_dots(8, o);
      }
      __syncthreads();
      if (cols) {
        bool odd = false;
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int r = 0; r < 4; ++r) odd |= !finite(z[jb][r]);
        if (!__any(odd)) {
          f32x4 pa[3];
#pragma unroll
          for (int f = 0; f < 3; ++f) pa[f] = lds_at<f32x4>(P + ((f > 0) * 16 + lr) * PP + (f > 1) * 16 + 4 * lg);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            o[0] = mfma4(pa[0][r], z[0][r], o[0]);
            o[1] = mfma4(pa[1][r], z[0][r], o[1]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) o[1] = mfma4(pa[2][r], z[1][r], o[1]);
        } else {
          // z again, row by row, for the rows that see it
          const __amdgpu_buffer_rsrc_t r2 = rz.chunk(t, m);
#pragma unroll 1
          for (int j = 0; j < kChunk; ++j) {
            const float zj = load1(r2, e < E ? uint32_t(back ? kChunk - 1 - j : j) * rz.pitch + uint32_t(e) * 4u : kOut);
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const i32x4 lo = lds_at<i32x4>(dc.lo + f * 16 + 4 * lg);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int row = f * 16 + 4 * lg + r;
                const bool sees = (j <= row) & (j >= lo[r]);
                const float x = o[f][r] + (sees ? P[row * PP + j] : 0.f) * zj;
                o[f][r] = sees ? x : o[f][r];
              }
            }
          }
        }
        if (dotted) {
          form_dots(0, o);
          const __amdgpu_buffer_rsrc_t r4 = resource(w.dots + (long(wave) * BH + bh) * 2 * a.T + t, uint32_t(a.T + m) * 4u);
          const int row = (lr >> 2 & 1) * 16 + 4 * lg + (lr & 3), s = back ? kChunk - 1 - row : row;
          store1(r4, s < m ? uint32_t((lr >> 3) * a.T + s) * 4u : kOut, dots);
        }
        const __amdgpu_buffer_rsrc_t r2 = ro.chunk(t, m);
        const Offsets at = offsets(ro.pitch);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) store1(r2, at.at[f][r], o[f][r]);
      }
    }

    // The state on leaving the chunk.
    const float keep = dc.keep;
    const int first = __builtin_amdgcn_readfirstlane(dc.first);
    if constexpr (LOCAL) total *= keep;
    if (cols) {
#pragma unroll
      for (int jb = 0; jb < 2; ++jb) {
        const f32x4 left = lds_at<f32x4>(dc.left + jb * 16 + 4 * lg);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = jb * 16 + 4 * lg + r;
          const float x = z[jb][r] * (left[r] * alpha_pair);
          z[jb][r] = j >= first ? x : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = S[k][r] * keep;
          S[k][r] = keep == 0.f ? 0.f : x;
        }
#pragma unroll
      for (int jb = 0; jb < 2; ++jb) {
        float y[KB][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < KB; ++k) y[k][r] = Y[(jb * 16 + 4 * lg + r) * PX + k * 16 + lr];
        if (first > 0) {  // rows before `first` are another episode's
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int k = 0; k < KB; ++k) y[k][r] = jb * 16 + 4 * lg + r >= first ? y[k][r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < KB; ++k) S[k] = mfma4(y[k][r], z[jb][r], S[k]);
      }
    }
  }

  if constexpr (LOCAL) {
    leave(a.added + (run * BH + bh) * D * E, 1.f, false);
    if (tid == 0) a.decays[run * BH + bh] = total;
  } else if (w.end && (back ? t0 == 0 : t0 + n == a.T)) {
    float g = 0.f;
    bool none = false;
    if (w.end_decay) step_decay(a, 0, b, h, g, none);
    leave(w.end + long(bh) * D * E, expf(g), none);
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
  constexpr int DEEP = 16;  // segments in flight: one at a time each waits for memory (63 segments 19.6 us, with 16 11.7)
  for (int q0 = 0; q0 < nseg; q0 += DEEP) {
    float u[DEEP], d[DEEP];
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int q = min(q0 + j, nseg - 1), s = back ? nseg - 1 - q : q;
      u[j] = added[s * BH * DE + i];
      d[j] = decays[s * BH + bh];
    }
#pragma unroll
    for (int j = 0; j < DEEP; ++j) {
      const int q = q0 + j, s = back ? nseg - 1 - q : q;
      if (q >= nseg) break;
      added[s * BH * DE + i] = run;
      run = (d[j] == 0.f ? 0.f : run * d[j]) + u[j];
    }
  }
}

// dL/dg of one head's segment.  X_t is the sum over pairs i >= t > j.  Of the pairs
// that end or begin in t's chunk, those with the other step before the chunk are
// in q_i . dq_i of the entering state alone, those with the other step after it in
// k_j . dk_j: sums from t on and up to t, in which nothing cancels.  Pairs inside
// the chunk are in the rest of both products, once in either, so their sum is
// that of the differences from t on, or less those before t: the nearer end of
// the episode's steps here.  Pairs around the chunk follow from one chunk's
// first X to the one before it, and start again from <S, G> at the segment's end.
// (As one running sum of q . dq - k . dk every step's rounding went on to all steps
// before it, and a decay that all steps share collected it: the gradient of 90
// steps of 228 sequences was off by 5.9e-6 in the median of 8 inputs, 1.6e-6 so.
// It takes 5 us more here and 5 in the sweeps of 1024 steps of 256 heads.)
constexpr int kGradThreads = 256, kMark = kGradThreads;  // a segment's steps at most
__global__ __launch_bounds__(kGradThreads) void k_decay_grad(SweepArgs a, const float* __restrict__ states,
                                                             const float* __restrict__ grads,
                                                             const float* __restrict__ final_state,
                                                             const float* __restrict__ final_grad, int DE,
                                                             const float* __restrict__ qd, const float* __restrict__ kd,
                                                             int parts, float* __restrict__ dg,
                                                             double* __restrict__ sums, int first_bh) {
  constexpr int NWV = kGradThreads / 64, NC = kGradThreads / kChunk;
  __shared__ float red[NWV];
  __shared__ double first[NC], last[NC], part[NWV];
  __shared__ int whole[NC];
  const long BH = long(a.B) * a.H, bh = first_bh + long(blockIdx.x);
  const int s = int(blockIdx.y), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = tid / kChunk, i = tid % kChunk;
  const int b = int(bh / a.H), h = int(bh - long(b) * a.H);
  const int t0 = s * a.seg, n = min(a.seg, a.T - t0), t = t0 + tid;
  const bool in = tid < n;
  float v[4][kMaxHead / 16], g = 0.f;
  bool reset = false;
  if (in) {
    for (int p = 0; p < parts; ++p) {
      const long at = (p * BH + bh) * 2 * a.T + t;
      v[0][p] = qd[at];
      v[1][p] = kd[at];
      v[2][p] = qd[at + a.T];
      v[3][p] = kd[at + a.T];
    }
    step_decay(a, t, b, h, g, reset);
  }
  const bool end = s + 1 == a.nseg;
  const float* sx = end ? final_state + bh * DE : states + ((s + 1) * BH + bh) * DE;
  const float* sy = end ? (final_grad ? final_grad + bh * DE : nullptr) : grads + (s * BH + bh) * DE;
  double beyond = 0.0;  // X of the step after the segment
  if (sy) {  // uniform
    float d = 0.f;
    for (int e = tid; e < DE; e += kGradThreads) d += sx[e] * sy[e];
    d = block_sum<kGradThreads>(d, red);
    float ge;
    bool re;
    step_decay(a, t0 + n, b, h, ge, re);  // past the last step: no decay
    beyond = re ? 0.0 : double(d) * double(expf(ge));
  }
  double net = 0.0, left = 0.0, right = 0.0;  // pairs inside the chunk, with steps before it, with steps after it
  if (in)
    for (int p = 0; p < parts; ++p) {
      left += double(v[2][p]);
      right += double(v[3][p]);
      net += (double(v[0][p]) - double(v[2][p])) - (double(v[1][p]) - double(v[3][p]));
    }
  const uint32_t starts = uint32_t(__ballot(reset) >> (lane & 32));  // of this chunk
  const uint32_t upto = starts & (0xffffffffu >> (31 - i)), later = starts & ~(0xffffffffu >> (31 - i));
  const int lo = upto ? 31 - __clz(upto) : 0, hi = later ? __ffs(later) - 2 : kChunk - 1;  // the episode's steps here
  // Sums over a chunk's 32 lanes, of the episode's steps up to this one and from it on.
  auto up_to = [&](double x) __attribute__((always_inline)) {
    double y = before<1>(x);
    x = i - 1 >= lo ? x + y : x;
    y = before<2>(x);
    x = i - 2 >= lo ? x + y : x;
    y = before<4>(x);
    x = i - 4 >= lo ? x + y : x;
    y = before<8>(x);
    x = i - 8 >= lo ? x + y : x;
    y = __shfl(x, 15, kChunk);
    return i >= 16 && lo < 16 ? x + y : x;
  };
  auto from_on = [&](double x) __attribute__((always_inline)) {
    double y = after<1>(x);
    x = i + 1 <= hi ? x + y : x;
    y = after<2>(x);
    x = i + 2 <= hi ? x + y : x;
    y = after<4>(x);
    x = i + 4 <= hi ? x + y : x;
    y = after<8>(x);
    x = i + 8 <= hi ? x + y : x;
    y = __shfl(x, 16, kChunk);
    return i < 16 && hi >= 16 ? x + y : x;
  };
  const double on = from_on(net);
  left = from_on(left);
  right = up_to(right);
  if (i == 0) first[c] = reset ? 0.0 : left;
  if (i == kChunk - 1) {
    last[c] = right;
    whole[c] = !starts;
  }
  const double past = __shfl_up(up_to(net), 1, kChunk);
  right = __shfl_up(right, 1, kChunk);
  __syncthreads();
  double x = i - lo <= hi - i ? (i > lo ? -past : 0.0) : on;
  if (!upto) x += left;
  if (!later && i > lo) x += right;
  for (int j = (n - 1) / kChunk; j >= c; --j) {  // `beyond` becomes X of each chunk's first step
    const double around = whole[j] ? beyond - last[j] : 0.0;
    if (j == c && !starts) x += around;
    beyond = whole[j] ? around + first[j] : first[j];
  }
  if (reset) x = 0.0;
  if (in && dg) dg[(long(t) * a.B + b) * a.H + h] = float(x);
  if (!sums) return;
  double sum = in ? x : 0.0;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m, 64);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (tid == 0) sums[s * BH + bh] = (part[0] + part[1]) + (part[2] + part[3]);
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
  int first;  // head of a lane that the launch begins with
};
constexpr int kStepThreads = 256;

template <int W>
__global__ __launch_bounds__(kStepThreads) void k_token(StepArgs a) {
  __shared__ float part[kStepThreads * W];
  const int bh = a.first + int(blockIdx.x), b = bh / a.H, h = bh - b * a.H, G = a.H / a.share;
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

// Workgroups of 256 threads of one launch: its threads are counted in 32 bits, and
// a count that passes them starts what is left of it without an error.
constexpr long kMostGroups = 1L << 23;

// Every row of the operand starts on 16 bytes.
bool wide(const Operand& o) { return !o.p || (o.dim % 4 == 0 && aligned16(o.p)); }

template <bool LOCAL>
int launch_alike(ttrl_ctx* ctx, const SweepArgs& a, int count, int kp, int nw, const char* name) {
  bool vec = true;
  for (int i = 0; i < count; ++i) vec = vec && wide(a.s[i].y) && (LOCAL || wide(a.s[i].x));
  const dim3 grid(unsigned(a.B) * unsigned(a.H), unsigned((a.T + a.run - 1) / a.run), unsigned(count));
  auto go = [&](auto kpc, auto nwc) {
    constexpr int KP = decltype(kpc)::value, NW = decltype(nwc)::value;
    if (vec) hipLaunchKernelGGL((k_sweep<KP, NW, true, LOCAL>), grid, dim3(64 * NW), 0, stream_of(ctx), a);
    else hipLaunchKernelGGL((k_sweep<KP, NW, false, LOCAL>), grid, dim3(64 * NW), 0, stream_of(ctx), a);
  };
  auto width = [&](auto kpc) {
    if (decltype(kpc)::value <= 64 && nw == 2) go(kpc, std::integral_constant<int, decltype(kpc)::value <= 64 ? 2 : 4>{});
    else if (nw <= 4) go(kpc, std::integral_constant<int, 4>{});
    else if (nw == 6) go(kpc, std::integral_constant<int, 6>{});
    else go(kpc, std::integral_constant<int, 8>{});
  };
  if (kp == 32) width(std::integral_constant<int, 32>{});
  else if (kp == 64) width(std::integral_constant<int, 64>{});
  else if (kp == 96) width(std::integral_constant<int, 96>{});
  else width(std::integral_constant<int, 128>{});
  return check_launch(name);
}

// Sweeps of one shape go in one launch, others after them: together the widest
// one's tiles serve all (4001 steps, 2 sequences, 6 heads of 40 and 72: the
// backward's sweeps 111 us in one launch of 128-wide tiles, 81 in two).
template <bool LOCAL>
int launch_sweeps(ttrl_ctx* ctx, const SweepArgs& a, int count, const char* name) {
  auto class_of = [](int n) { return (n + 31) / 32; };
  bool gone[3] = {};
  for (int i = 0; i < count; ++i) {
    if (gone[i]) continue;
    SweepArgs b = a;
    const int kp = class_of(a.s[i].x.dim), nw = class_of(a.s[i].z.dim);
    int same = 0;
    for (int j = i; j < count; ++j)
      if (class_of(a.s[j].x.dim) == kp && class_of(a.s[j].z.dim) == nw) {
        b.s[same++] = a.s[j];
        gone[j] = true;
      }
    if (int rc = launch_alike<LOCAL>(ctx, b, same, 32 * kp, 2 * nw, name)) return rc;
  }
  return TTRL_OK;
}

// Segments of whole chunks, kMark steps at most, and whether they run side by
// side (`cut`): where heads and sequences alone do not fill the compute units,
// into as many as fill them once.  More cost more states to join and to read
// (4001 steps, 2 sequences, 6 heads, forward and backward: 1024 workgroups 255
// us, 512 224, 256 206; 2048 x 8 x 8 forward: 243, 210, 210).
struct Plan {
  int seg, nseg;
  bool cut;
};
Plan plan_of(int T, long BH) {
  const long chunks = std::max(1L, long(T + kChunk - 1) / kChunk);
  const long want = std::max(1L, (256 + BH - 1) / std::max(1L, BH));
  const bool cut = BH < 256 && chunks > 1;
  const long per = cut ? std::min(long(kMark / kChunk), (chunks + want - 1) / want) : kMark / kChunk;
  const int seg = int(per * kChunk);
  return {seg, std::max(1, (T + seg - 1) / seg), cut && T > seg};
}

struct Space {  // floats of the caller's buffers, in order
  long states, decays, grads, gdecays, qdots, kdots, dk, dv, sums;
};

int check_desc(const ttrl_linear_attention_desc* d, const char* name) {
  TTRL_REQUIRE(d, "%s: null description", name);
  TTRL_REQUIRE(d->T >= 0 && d->B >= 0 && d->H > 0 && d->kv_heads > 0 && d->H % d->kv_heads == 0,
               "%s: %d heads do not share %d key/value heads evenly (T=%d, B=%d)", name, d->H, d->kv_heads, d->T, d->B);
  TTRL_REQUIRE(d->K > 0 && d->V > 0 && d->K <= kMaxHead && d->V <= kMaxHead,
               "%s: head widths of 1 to %d are supported, got K=%d, V=%d", name, kMaxHead, d->K, d->V);
  TTRL_REQUIRE(long(d->B) * d->H <= 0x7fffffffL / 2, "%s: %d sequences of %d heads are too many", name, d->B, d->H);
  TTRL_REQUIRE(plan_of(d->T, long(d->B) * d->H).nseg <= 65535, "%s: %d steps are too many", name, d->T);
  TTRL_REQUIRE(long(d->B) * d->H * std::max(d->K, d->V) <= 1L << 24,
               "%s: %d sequences of %d heads are more than 2^24 values a step", name, d->B, d->H);
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
  a.run = p.cut ? p.seg : d->T;
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
  s.qdots = even(2 * long((d->K + 15) / 16) * BH * d->T);
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

int ttrl_linear_attention_space(const ttrl_linear_attention_desc* d, long* forward_floats, long* saved_floats,
                                long* work_floats) {
  if (int rc = check_desc(d, "ttrl_linear_attention_space")) return rc;
  TTRL_REQUIRE(forward_floats && saved_floats && work_floats, "ttrl_linear_attention_space: null output");
  const Plan p = plan_of(d->T, long(d->B) * d->H);
  const Space s = space_of(d, p.nseg);
  *saved_floats = s.states + s.decays;
  *forward_floats = p.cut ? *saved_floats : 0;
  *work_floats = s.grads + s.gdecays + s.qdots + s.kdots + s.dk + s.dv + s.sums;
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
  if (a.run == a.T) {
    s.marks = a.nseg > 1 ? d->saved : nullptr;
  } else {
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
  float *grads = take(sp.grads), *gdecays = take(sp.gdecays), *qdots = take(sp.qdots),
        *kdots = take(sp.kdots), *dkh = take(sp.dk), *dvh = take(sp.dv), *sums = take(sp.sums);
  const Operand q{d->q, d->H, d->K, 1}, k{d->k, d->kv_heads, d->K, share}, v{d->v, d->kv_heads, d->V, share},
      go{d->dout, d->H, d->V, 1};
  const bool cut = a.run < a.T;
  TTRL_REQUIRE(a.nseg == 1 || d->saved, "%s: null saved states", name);

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
  } else if (a.nseg > 1 && d->dlog_decay) {
    dv.marks = grads;
  }
  Sweep dk = dv;  // state G^T, (V, K)
  dk.x = v;
  dk.y = go;
  dk.z = q;
  dk.out = share > 1 ? dkh : d->dk;
  dk.end = nullptr;
  dk.marks = nullptr;
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
    TTRL_REQUIRE(!d->dfinal || d->final_state, "%s: the final state's gradient needs the final state", name);
    double* total = d->decay_steps ? nullptr : reinterpret_cast<double*>(sums);
    for (long from = 0; from < BH; from += kMostGroups) {
      const unsigned groups = unsigned(std::min(kMostGroups, BH - from));
      hipLaunchKernelGGL(k_decay_grad, dim3(groups, unsigned(a.nseg)), dim3(kGradThreads), 0, stream_of(ctx), a, d->saved,
                         grads, d->final_state, d->dfinal, int(DE), qdots, kdots, (d->K + 15) / 16,
                         d->decay_steps ? d->dlog_decay : nullptr, total, int(from));
      if (int rc = check_launch(name)) return rc;
    }
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
  StepArgs a{q, k, v, log_decay, done, state, out, decay_rows, B, H, H / kv_heads, K, V, scale, 0};
  const long BH = long(B) * H;
  for (long from = 0; from < BH; from += kMostGroups) {
    a.first = int(from);
    const dim3 grid(unsigned(std::min(kMostGroups, BH - from)));
    if (V % 4 == 0 && aligned16(state) && aligned16(v))
      hipLaunchKernelGGL(k_token<4>, grid, dim3(kStepThreads), 0, stream_of(ctx), a);
    else
      hipLaunchKernelGGL(k_token<1>, grid, dim3(kStepThreads), 0, stream_of(ctx), a);
    if (int rc = check_launch(name)) return rc;
  }
  return TTRL_OK;
}

}  // extern "C"
