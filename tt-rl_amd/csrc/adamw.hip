// AdamW over many tensors at once (Loshchilov and Hutter, "Decoupled Weight
// Decay Regularization", ICLR 2019), moments in 32 bits or in 8:
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = (1 - lr wd) p - (lr / bc1) m / (sqrt(v) / sqrt(bc2) + eps),  bci = 1 - bi^t.
//
// In 8 bits a moment is a code per element and a scale per block of 64
// elements, the block's largest magnitude (block-wise scales after Dettmers et
// al., "8-bit Optimizers via Block-wise Quantization", ICLR 2022; the codes
// are this file's own): m's code c is the nearest of 127 signed steps of
// sqrt(|m| / scale) and stands for c |c| / 127^2 scale, v's the nearest of 255
// steps of the fourth root and stands for (c / 255)^4 scale.  The roots spend
// the codes on small values (v down to 2.4e-10 of its block's largest, which
// squares of gradients reach), and a v that is not zero is held as at least
// code 1, so no step is ever divided by eps alone.  The update itself uses the
// new moments before they are rounded to codes.
//
// Each product and sum is rounded on its own (no contraction into FMAs), so
// that 32-bit states, 8-bit codes and parameters are the same bits however the
// compiler schedules the kernel.
//
// One launch takes up to 64 tensors: their addresses travel in the kernel's
// arguments, so the step can be captured into a graph and no table is uploaded.
// A workgroup takes one or four rounds of 1024 elements of one tensor, found by bisection over the
// tensors' first workgroups.  Bound: HBM, 28 bytes a parameter in 32 bits,
// 16.25 in 8 (4 + 4 + 4 of p and g, 2 + 2 of codes, 0.25 of scales): 67M parameters
// in 8 bits and the read-out of their moments (26.4 bytes with it) 338 us, 5.2
// TB/s, more than a large copy's 4.7; the ten tensors of a convolutional Q network (1.7M,
// 32 bits) 10.8 us, 4.4 TB/s.
//
// The update count and the next update's bias corrections live on the device;
// the last workgroup of a step's last launch moves them on, so a replayed
// graph counts by itself and no workgroup waits for the powers.
#include "common.hpp"

#include <algorithm>

namespace ttrl {
namespace {

constexpr int kThreads = 256, kRound = kThreads * 4;  // elements of a workgroup's round
constexpr int kRounds = 4;
constexpr long kMany = 1024;  // workgroups of kRounds rounds; below, one round each
constexpr int kTensors = 64, kBlock = 64;

// Tickets on one word cost 7 ns a workgroup, one after another, so workgroups
// take them on one of kDesks lines, and a desk's last one on the first line.
constexpr int kDesks = 32;
struct Counter {
  int t;             // updates done
  unsigned tickets;  // desks of the running launch that are done
  double bc1, root;  // 1 - b1^(t+1) and 1 / sqrt(1 - b2^(t+1))
  unsigned fill[10], desk[kDesks][16];
};
static_assert(sizeof(Counter) == TTRL_ADAMW_COUNTER_BYTES, "the size callers allocate");

// b^n by squares: the same for a count that was set and one that was reached,
// and short (pow() kept the last workgroup for 4 us).
__device__ double power(double b, int n) {
  double r = 1.0;
  for (; n; n >>= 1, b *= b)
    if (n & 1) r *= b;
  return r;
}
__device__ void set_count(Counter* c, int t, double b1, double b2) {
  c->t = t;
  c->tickets = 0;
  c->bc1 = 1.0 - power(b1, t + 1);
  c->root = 1.0 / sqrt(1.0 - power(b2, t + 1));
}

__global__ void k_adamw_set(Counter* c, int t, double b1, double b2) {
  c->desk[threadIdx.x][0] = 0;
  if (threadIdx.x == 0) set_count(c, t, b1, b2);
}

struct Item {
  float* p;
  const float* g;
  long at, n;  // its place in the moments, its elements
  int first;   // its first workgroup
  int wide;    // p and g on 16 bytes
};
struct AdamWArgs {
  Item item[kTensors];
  int count;
  void *m, *v;
  float *m_scale, *v_scale;
  Counter* counter;
  double lr, b1d, b2d;
  float b1, c1, b2, c2, eps, shrink;
  int last;  // the step's last launch
};

__device__ __forceinline__ f32x4 load4(const float* p, long i, long n, bool whole) {
  if (whole) return *reinterpret_cast<const f32x4*>(p + i);
  f32x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = i + j < n ? p[i + j] : 0.f;
  return x;
}
__device__ __forceinline__ void store4(float* p, long i, long n, bool whole, const f32x4& x) {
  if (whole) {
    *reinterpret_cast<f32x4*>(p + i) = x;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j < n) p[i + j] = x[j];
}

// A magnitude as bits, which order as magnitudes do, infinity and NaN above all.
__device__ __forceinline__ uint32_t size_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest over the 16 lanes (a DPP row) that hold a block.
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
#define TTRL_ROW_ROR(n) x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x120 + n, 0xf, 0xf, true)))
  TTRL_ROW_ROR(8);
  TTRL_ROW_ROR(4);
  TTRL_ROW_ROR(2);
  TTRL_ROW_ROR(1);
#undef TTRL_ROW_ROR
  return x;
}

__device__ __forceinline__ float held_m(int code, float scale) {
#pragma clang fp contract(off)
  const float c = float(code) * (1.f / 127.f);
  return c * fabsf(c) * scale;
}
__device__ __forceinline__ float held_v(unsigned code, float scale) {
#pragma clang fp contract(off)
  float c = float(code) * (1.f / 255.f);
  c = c * c;
  return c * c * scale;
}
__device__ __forceinline__ int code_m(float m, float scale) {
#pragma clang fp contract(off)
  const float r = scale > 0.f ? fabsf(m) / scale : 0.f;
  const int c = r > 0.f ? int(rintf(sqrtf(r) * 127.f)) : 0;  // 0 for NaN, whose block's scale tells
  return m < 0.f ? -c : c;
}
__device__ __forceinline__ unsigned code_v(float v, float scale) {
#pragma clang fp contract(off)
  const float r = scale > 0.f ? v / scale : 0.f;
  return r > 0.f ? unsigned(fmaxf(rintf(sqrtf(sqrtf(r)) * 255.f), 1.f)) : 0u;
}

// Four elements' codes.  Divided and rooted by the hardware's approximations (1
// ulp each), x = 127 sqrt(r) is off by under 4e-5 and 255 r^(1/4) by under 8e-5
// where scale and r are far from the range's ends, and the correctly rounded
// forms above by as much: no half step within kSure means the same code.  The
// rest (one wavefront's round in five or so) takes the forms above.  They cost
// two divisions and three roots an element, more time than the memory: 67M
// parameters 327 us, 245 so, and 210 to 280 with the tickets' desks below.
constexpr float kSure = 2e-4f;
__device__ __forceinline__ void codes4(const f32x4& m, const f32x4& v, float top_m, float top_v, uint32_t* cm, uint32_t* cv) {
  auto usual = [](float s) { return s > 1e-30f && s < 1e30f; };
  bool sure = usual(top_m) && usual(top_v);
  const float im = __builtin_amdgcn_rcpf(top_m), iv = __builtin_amdgcn_rcpf(top_v);
  uint32_t a = 0, b = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = __builtin_amdgcn_sqrtf(fabsf(m[j]) * im) * 127.f, r = v[j] * iv;
    const float y = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(r)) * 255.f;
    sure = sure && fabsf(__builtin_amdgcn_fractf(x) - 0.5f) > kSure && fabsf(__builtin_amdgcn_fractf(y) - 0.5f) > kSure &&
           (r > 1e-30f || v[j] == 0.f);
    const int c = int(fminf(rintf(x), 127.f));  // NaN, which is not sure, converts too
    a |= (uint32_t(m[j] < 0.f ? -c : c) & 255u) << (8 * j);
    b |= uint32_t(v[j] > 0.f ? fminf(fmaxf(rintf(y), 1.f), 255.f) : 0.f) << (8 * j);
  }
  if (!sure) {
    a = b = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a |= (uint32_t(code_m(m[j], top_m)) & 255u) << (8 * j);
      b |= (code_v(v[j], top_v) & 255u) << (8 * j);
    }
  }
  *cm = a;
  *cv = b;
}

__device__ __forceinline__ int item_of(const AdamWArgs& a, int block) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (block >= a.item[mid].first) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <bool HELD, int ROUNDS>
__global__ __launch_bounds__(kThreads) void k_adamw(AdamWArgs a) {
#pragma clang fp contract(off)
  const Item& it = a.item[item_of(a, int(blockIdx.x))];
  const long from = long(int(blockIdx.x) - it.first) * (kRound * ROUNDS) + threadIdx.x * 4, n = it.n;
  const double bc1 = a.counter->bc1, root64 = a.counter->root;
  f32x4 p[ROUNDS], g[ROUNDS], m[ROUNDS], v[ROUNDS];
  uint32_t mc[ROUNDS], vc[ROUNDS];
  float ms[ROUNDS], vs[ROUNDS];
  bool in[ROUNDS], whole[ROUNDS];
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const long i = from + u * kRound, s = it.at + i;
    in[u] = i < n;
    whole[u] = it.wide && i + 4 <= n;
    if (!in[u]) continue;
    p[u] = load4(it.p, i, n, whole[u]);
    g[u] = load4(it.g, i, n, whole[u]);
    if constexpr (HELD) {  // a tensor's moments end on a block: whole reads
      mc[u] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + s);
      vc[u] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + s);
      ms[u] = a.m_scale[s / kBlock];
      vs[u] = a.v_scale[s / kBlock];
    } else {
      m[u] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.m) + s);
      v[u] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.v) + s);
    }
  }
  const float size = float(a.lr / bc1), root = float(root64);
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const long i = from + u * kRound, s = it.at + i;
    uint32_t size_m = 0, size_v = 0;
    if (in[u]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float mj, vj;
        if constexpr (HELD) {
          mj = held_m(int(int8_t(mc[u] >> (8 * j))), ms[u]);
          vj = held_v(uint8_t(vc[u] >> (8 * j)), vs[u]);
        } else {
          mj = m[u][j];
          vj = v[u][j];
        }
        const float gj = g[u][j];
        mj = mj * a.b1 + gj * a.c1;
        vj = vj * a.b2 + (gj * gj) * a.c2;
        const float step = mj / (sqrtf(vj) * root + a.eps) * size;
        p[u][j] = p[u][j] * a.shrink - step;
        if (HELD && i + j >= n) mj = vj = 0.f;
        m[u][j] = mj;
        v[u][j] = vj;
        size_m = max(size_m, size_bits(mj));
        size_v = max(size_v, size_bits(vj));
      }
      store4(it.p, i, n, whole[u], p[u]);
      if constexpr (!HELD) {
        store4(static_cast<float*>(a.m) + it.at, i, n, i + 4 <= n, m[u]);
        store4(static_cast<float*>(a.v) + it.at, i, n, i + 4 <= n, v[u]);
      }
    }
    if constexpr (HELD) {  // every lane of a row takes part
      const float top_m = __uint_as_float(row_max(size_m)), top_v = __uint_as_float(row_max(size_v));
      if (in[u]) {
        uint32_t cm, cv;
        codes4(m[u], v[u], top_m, top_v, &cm, &cv);
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + s) = cm;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + s) = cv;
        if ((threadIdx.x & 15) == 0) {
          a.m_scale[s / kBlock] = top_m;
          a.v_scale[s / kBlock] = top_v;
        }
      }
    }
  }
  if (!a.last) return;
  // Every workgroup has read the corrections before it takes its ticket.
  __syncthreads();
  if (threadIdx.x) return;
  const unsigned desk = blockIdx.x % kDesks, here = (gridDim.x - desk + kDesks - 1) / kDesks;
  unsigned* tickets = a.counter->desk[desk];
  if (atomicAdd(tickets, 1u) != here - 1) return;
  *tickets = 0;
  if (atomicAdd(&a.counter->tickets, 1u) == min(gridDim.x, unsigned(kDesks)) - 1)
    set_count(a.counter, a.counter->t + 1, a.b1d, a.b2d);
}

struct HeldItem {
  float *m, *v;
  long at, n;
  int first;
};
struct HeldArgs {
  HeldItem item[kTensors];
  int count;
  const uint8_t *mc, *vc;
  const float *ms, *vs;
};

// The values that the codes stand for.
template <int ROUNDS>
__global__ __launch_bounds__(kThreads) void k_adamw_held(HeldArgs a) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (int(blockIdx.x) >= a.item[mid].first) lo = mid;
    else hi = mid - 1;
  }
  const HeldItem& it = a.item[lo];
  const long from = long(int(blockIdx.x) - it.first) * (kRound * ROUNDS) + threadIdx.x * 4;
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const long i = from + u * kRound, s = it.at + i;
    if (i >= it.n) continue;
    const uint32_t mc = *reinterpret_cast<const uint32_t*>(a.mc + s), vc = *reinterpret_cast<const uint32_t*>(a.vc + s);
    const float ms = a.ms[s / kBlock], vs = a.vs[s / kBlock];
    f32x4 m, v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = held_m(int(int8_t(mc >> (8 * j))), ms);
      v[j] = held_v(uint8_t(vc >> (8 * j)), vs);
    }
    const bool whole = i + 4 <= it.n;
    store4(it.m, i, it.n, whole && (reinterpret_cast<uintptr_t>(it.m) & 15) == 0, m);
    store4(it.v, i, it.n, whole && (reinterpret_cast<uintptr_t>(it.v) & 15) == 0, v);
  }
}

long blocks_of(long n, int rounds) { return (n + long(kRound) * rounds - 1) / (long(kRound) * rounds); }
// Rounds of a workgroup: few elements are spread over the compute
// units (0.35M in tensors of odd sizes 13.2 us with four, 8.3 with one; 1.7M
// 13.2 and 8.8).
template <typename T>
int rounds_of(const T* t, int count) {
  long blocks = 0;
  for (int i = 0; i < count; ++i) blocks += blocks_of(t[i].n, kRounds);
  return blocks < kMany ? 1 : kRounds;
}

}  // namespace
}  // namespace ttrl

using namespace ttrl;

extern "C" {

int ttrl_adamw_set_count(ttrl_ctx* ctx, void* counter, int t, double beta1, double beta2) {
  TTRL_REQUIRE(ctx && counter, "ttrl_adamw_set_count: null argument");
  TTRL_REQUIRE(t >= 0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0,
               "ttrl_adamw_set_count: t=%d, betas %g and %g", t, beta1, beta2);
  hipLaunchKernelGGL(k_adamw_set, dim3(1), dim3(kDesks), 0, stream_of(ctx), static_cast<Counter*>(counter), t, beta1, beta2);
  return check_launch("ttrl_adamw_set_count");
}

int ttrl_adamw_step(ttrl_ctx* ctx, int count, const ttrl_adamw_tensor* tensors, int state_bits, void* m, void* v,
                    float* m_scale, float* v_scale, void* counter, double lr, double beta1, double beta2, double eps,
                    double weight_decay) {
  const char* name = "ttrl_adamw_step";
  TTRL_REQUIRE(ctx && tensors && m && v && counter, "%s: null argument", name);
  TTRL_REQUIRE(count > 0, "%s: no tensors", name);
  TTRL_REQUIRE(state_bits == 32 || state_bits == 8, "%s: moments in 32 or 8 bits, not %d", name, state_bits);
  TTRL_REQUIRE(state_bits == 32 || (m_scale && v_scale), "%s: null scales", name);
  TTRL_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "%s: betas %g and %g", name, beta1, beta2);
  TTRL_REQUIRE(((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
               "%s: moments must be 16-byte aligned", name);
  for (int i = 0; i < count; ++i)
    TTRL_REQUIRE(tensors[i].p && tensors[i].g && tensors[i].n > 0 && tensors[i].n <= (1L << 40) && tensors[i].at >= 0 &&
                     tensors[i].at % kBlock == 0,
                 "%s: tensor %d: null, empty, or its moments do not start on a block of %d", name, i, kBlock);
  for (int from = 0; from < count; from += kTensors) {
    AdamWArgs a{};
    a.count = std::min(kTensors, count - from);
    const int rounds = rounds_of(tensors + from, a.count);
    long blocks = 0;
    for (int i = 0; i < a.count; ++i) {
      const ttrl_adamw_tensor& t = tensors[from + i];
      const bool wide = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) & 15) == 0;
      a.item[i] = {t.p, t.g, t.at, t.n, int(blocks), wide};
      blocks += blocks_of(t.n, rounds);
      TTRL_REQUIRE(blocks <= 0x7fffffffL, "%s: too many elements", name);
    }
    a.m = m;
    a.v = v;
    a.m_scale = m_scale;
    a.v_scale = v_scale;
    a.counter = static_cast<Counter*>(counter);
    a.lr = lr;
    a.b1d = beta1;
    a.b2d = beta2;
    a.b1 = float(beta1);
    a.c1 = float(1.0 - beta1);
    a.b2 = float(beta2);
    a.c2 = float(1.0 - beta2);
    a.eps = float(eps);
    a.shrink = float(1.0 - lr * weight_decay);
    a.last = from + kTensors >= count;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kThreads), 0, stream_of(ctx), a); };
    if (state_bits == 8) rounds == 1 ? go(k_adamw<true, 1>) : go(k_adamw<true, kRounds>);
    else rounds == 1 ? go(k_adamw<false, 1>) : go(k_adamw<false, kRounds>);
    if (int rc = check_launch(name)) return rc;
  }
  return TTRL_OK;
}

int ttrl_adamw_moments(ttrl_ctx* ctx, int count, const ttrl_adamw_moment* tensors, const void* m, const void* v,
                       const float* m_scale, const float* v_scale) {
  const char* name = "ttrl_adamw_moments";
  TTRL_REQUIRE(ctx && tensors && m && v && m_scale && v_scale, "%s: null argument", name);
  TTRL_REQUIRE(count > 0, "%s: no tensors", name);
  for (int i = 0; i < count; ++i)
    TTRL_REQUIRE(tensors[i].m && tensors[i].v && tensors[i].n > 0 && tensors[i].n <= (1L << 40) && tensors[i].at >= 0 &&
                     tensors[i].at % kBlock == 0,
                 "%s: tensor %d: null, empty, or its moments do not start on a block of %d", name, i, kBlock);
  for (int from = 0; from < count; from += kTensors) {
    HeldArgs a{};
    a.count = std::min(kTensors, count - from);
    const int rounds = rounds_of(tensors + from, a.count);
    long blocks = 0;
    for (int i = 0; i < a.count; ++i) {
      const ttrl_adamw_moment& t = tensors[from + i];
      a.item[i] = {t.m, t.v, t.at, t.n, int(blocks)};
      blocks += blocks_of(t.n, rounds);
      TTRL_REQUIRE(blocks <= 0x7fffffffL, "%s: too many elements", name);
    }
    a.mc = static_cast<const uint8_t*>(m);
    a.vc = static_cast<const uint8_t*>(v);
    a.ms = m_scale;
    a.vs = v_scale;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(kThreads), 0, stream_of(ctx), a); };
    rounds == 1 ? go(k_adamw_held<1>) : go(k_adamw_held<kRounds>);
    if (int rc = check_launch(name)) return rc;
  }
  return TTRL_OK;
}

}  // extern "C"
