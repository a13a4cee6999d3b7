// Group normalisation with an activation, channels last: x [B, S, C], groups of
// Cg = C / G consecutive channels, n = S * Cg values a group.
//
//   forward   mu = sum x / n, var = sum (x - mu)^2 / n, r = (var + eps)^-1/2,
//             z = (x - mu) r gamma + beta, y = drop(act(z))
//   backward  dz = drop'(dy) act'(z), A = sum_s dz, X = sum_s dz (x - mu) r,
//             dbeta = sum_b A, dgamma = sum_b X,
//             m1 = sum_g gamma A / n, m2 = sum_g gamma X / n,
//             dx = r (gamma dz - m1 - (x - mu) r m2)
//
// A few operations per element, so the floor is HBM traffic: x read and y
// written once (x, dy read and dx written once in the backward). Every sum is
// needed before the first output, so a sample is read twice; see the launchers
// for how the second read comes out of L2.
//
// Numerics. The sums are of d = x - K and d^2, float64 from the first addition on, and
// var = (n sum d^2 - (sum d)^2) / n^2 with split products: it may cancel to (mu - K)^2 / var
// of what the sums lost to rounding.
//   float32 maps: K is the group's first value. As one of the n values it has (mu - K)^2 <=
// (n - 1) var, and a few var in a map like any other, however far its mean lies from 0.
//   16-bit maps: K = 0. Where mu^2 / var is large nearly all values lie in one binade: they are
// whole multiples, of 8 or 11 bits, of one step, so their sums and those of their squares (22
// bits and log2 n) are exact; each other value costs a rounding, but has a share of var. (K
// here would be a third float64 operation an element, 4 % of instance norm's forward, and the
// registers of rows wider than a CTA: 248 us instead of 199 for 8 x 6400 x 2304.)
// A constant group's var is 0 exactly. (Plain E[x^2] - mu^2 left 1/std of float32 maps 1e-6
// off at mean / std = 1e5, 1e-4 off at 1e6. Float32 sums of d^2 over 110 rows left it
// 1.7e-7 off for bfloat16 maps: squares of odd integers are 1 modulo 8, so their roundings
// do not average out.) That matters because a rectifier's gradient jumps at z = 0: with
// 1.7e-7, one training step in three of a 67 million element map had elements on the wrong
// side. The backward therefore takes z = x a + b with a = gamma r, b = beta - mu a as
// pairs of floats, whose sign is that of the float64 value but for ~2^-45.
// The backward's sums of dz and dz (x - mu) are float32 over at most kRun rows of a thread,
// then over at most kRuns such sums, and float64 beyond; the plain kernels round a thread's
// and a slice's sum to float32 once each. So n equal terms are off by 17 2^-24 a level at
// most. (One float32 sum over a thread's rows left the gradient of a mean's bias 173 2^-24
// off at 1024 rows a thread: equal terms round the same way until the sum doubles.)
// Partial sums have slots of their own and are added in a fixed order, with no float
// atomics: results repeat bit for bit.
#pragma once

#include "feature_common.cuh"
#include "tc_ptx.cuh"

namespace lcb200 {

constexpr int kT = 256;      // threads of a CTA
constexpr int kOcc = 3;      // CTAs a multiprocessor holds
constexpr int kUnroll = 4;   // rows a thread has in flight
constexpr int kRun = 32;     // rows of a thread whose terms are added in float32
constexpr int kRuns = 32;    // such sums added in float32

// 1: a wait ran out and a kernel of this translation unit stopped early
static __device__ int norm_status;

// The work of a call is cut into units: slices of slice_rows rows of a sample, each
// with a first pass (sums) and a second pass (outputs).
struct NormArgs {
  const void* x;
  const void* dy;
  void* out;           // y or dx
  const void* weight;  // [C] or null
  const void* bias;
  int param_f32;       // weight/bias dtype: float32, else x's
  double2* stats;      // [B, G] (mean, 1/std)
  long long S;
  int B, C, G, Cg;
  int act;
  float slope;
  double eps;
  uint64_t wait_ns;     // after which a wait gives up
  int slices;           // of a sample
  long long slice_rows;
  int fan, sets;        // slices of a set (see finish_slice), sets of a sample
  uint32_t units, lag;  // B * slices; units between a first pass and its second
  uint32_t tickets;     // 2 * units, or units without a second pass (out null)
  // streamed kernels (see norm_stream.cu)
  int teams, ctas;      // teams of CTAs, CTAs of a team
  int stage_rows;
  int chunk, chunks;    // samples of a chunk
  // workspace
  uint32_t* ticket;     // [2]: next unit, finished samples
  uint32_t* done;       // [B, sets] finished first-pass slices of a set
  uint32_t* sets_done;  // [B] finished sets
  uint32_t* ready;      // [B] 1: statistics (backward: coef) are there
  // (the plain kernels' rows; the others have a row per slot or CTA)
  double2* part;        // forward: [B, slices, G] (sum d, sum d^2); streamed: [slots, G]
  float2* bpart;        // backward: [B, slices, C] (sum dz, sum dz (x - mu))
  double2* set_part;    // [B, sets, G (backward: C)] sums of a set's slices
  double2* sums;        // backward: [B, C] (A, X); otherwise a CTA's sum of them, [CTAs, C]
  float4* coef;         // backward: [B, G] (mu, k2, k3, 0): dx = gamma r dz + k2 (x - mu) + k3
  void* dweight;        // [C] or null
  void* dbias;
  DropArgs drop;
};

// What came of a launch of the streamed kernels. kNoRoom: their CTAs do not fit the context
// all at once (one that has a part of the GPU's multiprocessors), nothing was launched.
enum class Streamed { kDone, kFailed, kNoRoom };

// Runs of a chunk of the streamed kernels: one a CTA, fewer where that would leave less
// than a stage.
__host__ __device__ inline int chunk_parts(long long rows, int stage_rows, int ctas) {
  const long long stages = (rows + stage_rows - 1) / stage_rows;
  return (int)(stages < ctas ? stages : ctas);
}

// A barrier of the kT arithmetic threads (the streamed kernels have a producer
// warp besides).
__device__ __forceinline__ void cta_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kT) : "memory"); }

template <typename T>
__device__ __forceinline__ double param(const void* p, int f32, int c, double none) {
  if (!p) return none;
  return f32 ? (double)__ldg(reinterpret_cast<const float*>(p) + c)
             : (double)ldf(reinterpret_cast<const T*>(p) + c);
}

template <typename T>
__device__ __forceinline__ float param_f(const void* p, int f32, int c, float none) {
  if (!p) return none;
  return f32 ? __ldg(reinterpret_cast<const float*>(p) + c)
             : ldf(reinterpret_cast<const T*>(p) + c);
}

template <typename T>
__device__ __forceinline__ void put_param(void* p, int f32, int c, double v) {
  if (!p) return;
  if (f32) reinterpret_cast<float*>(p)[c] = (float)v;
  else stf(reinterpret_cast<T*>(p) + c, (float)v);
}

// sigma(z) by the fast exponential (2 + 1.173 |z| ulp) and quotient (2 ulp): their error counts
// times 1 - sigma, so z sigma(z) is within 6 ulp for z > -1 and within 5 + 1.2 |z| ulp of its
// shrinking value below. exp(-z) overflowing to infinity gives 0.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

__device__ __forceinline__ float act_value(float z, int act, float slope) {
  if (act == LCB200_ACT_SILU) return z * sigmoid(z);
  if (act == LCB200_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if (act == LCB200_ACT_LEAKY_RELU) return z < 0.f ? slope * z : z;
  return z;
}

__device__ __forceinline__ float act_grad(float z, float g, int act, float slope) {
  if (act == LCB200_ACT_SILU) {
    const float sg = sigmoid(z);
    return g * (sg * fmaf(z, 1.f - sg, 1.f));
  }
  if (act == LCB200_ACT_RELU) return z > 0.f ? g : 0.f;
  if (act == LCB200_ACT_LEAKY_RELU) return z > 0.f ? g : slope * g;
  return g;
}

// A thread's place in a CTA's rows x vector columns tiling.
struct Place {
  int nc;   // vector columns of the block starting at cb
  int rp;   // rows a CTA covers per step
  int col;  // vector column (of the whole row)
  int row;
  bool on;
  __device__ __forceinline__ Place(int cols, int cb, int threads = kT) {
    nc = min(cols - cb, threads);
    rp = threads / nc;
    col = cb + threadIdx.x % nc;
    row = threadIdx.x / nc;
    on = row < rp;
  }
};

__device__ __forceinline__ int pow2_below(int v) { return v < 1 ? 1 : 1 << (31 - __clz(v)); }

__device__ __forceinline__ double2 lanes_sum(double2 v, int width) {
  for (int o = width / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

// (factor, offset) of the channel, z = x a + b, as unevaluated float pairs.
struct Affine {
  float ah, al, bh, bl;
};
template <typename T>
__device__ __forceinline__ Affine affine(const NormArgs& p, double2 st, int c) {
  const double a = param<T>(p.weight, p.param_f32, c, 1.0) * st.y;
  const double b = param<T>(p.bias, p.param_f32, c, 0.0) - st.x * a;
  Affine f;
  f.ah = (float)a;
  f.al = (float)(a - (double)f.ah);
  f.bh = (float)b;
  f.bl = (float)(b - (double)f.bh);
  return f;
}
__device__ __forceinline__ float affine_z(const Affine& f, float x) {
  return fmaf(x, f.ah, f.bh) + fmaf(x, f.al, f.bl);
}

// ---- the end of a sample: statistics, or coefficients of dx --------------------
// The value K that a group's sums are centred on.
template <typename T>
__device__ __forceinline__ double group_shift(const NormArgs& p, int b, int g) {
  if (sizeof(T) < 4) return 0.0;
  return (double)ldf(reinterpret_cast<const T*>(p.x) + (long long)b * p.S * p.C +
                     (long long)g * p.Cg);
}

// One group's mean and 1/std from its (sum d, sum d^2).
__device__ __forceinline__ double2 finish_stats(const NormArgs& p, double2 v, double shift) {
  const double n = (double)p.S * p.Cg, inv = 1.0 / n;
  const double nq = n * v.y, ss = v.x * v.x;
  double var = ((nq - ss) + (fma(n, v.y, -nq) - fma(v.x, v.x, -ss))) * inv * inv;
  var = var < 0.0 ? 0.0 : var;  // rounding below zero; NaN stays
  return make_double2(fma(v.x, inv, shift), 1.0 / sqrt(var + p.eps));
}

// True in every thread of the CTA that finished last of `count` at *counter;
// what the others wrote before is then visible.
static __device__ bool last_of(uint32_t* counter, uint32_t count) {
  __shared__ int is_last;
  cta_sync();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicAdd(counter, 1u) == count - 1;
    __threadfence();
  }
  cta_sync();
  return is_last;
}

__device__ __forceinline__ double2 as_double2(float2 v) { return make_double2(v.x, v.y); }
__device__ __forceinline__ double2 as_double2(double2 v) { return v; }

// Column sums of an [n, C] matrix of pairs by the whole CTA, handed to
// put(c, sum) by one thread per column; a fixed order for fixed sizes.
template <typename P, typename F>
__device__ void column_sums(const P* src, long long n, int C, double2* sm, F put) {
  for (int cb = 0; cb < C; cb += kT) {
    const int nc = min(C - cb, kT);
    const int parts = (int)min((long long)(kT / nc), n);
    const int c = threadIdx.x % nc, part = threadIdx.x / nc;
    double2 v = make_double2(0.0, 0.0);
    if (part < parts) {
#pragma unroll 8
      for (long long i = part; i < n; i += parts) {
        const double2 e = as_double2(__ldcg(src + i * C + cb + c));
        v.x += e.x;
        v.y += e.y;
      }
    }
    sm[threadIdx.x] = v;
    cta_sync();
    if (part == 0) {
      for (int k = 1; k < parts; ++k) {
        v.x += sm[k * nc + c].x;
        v.y += sm[k * nc + c].y;
      }
      put(cb + c, v);
    }
    cta_sync();
  }
}

// Adds up a sample's per-slice sums part [slices, cols] after this slice's
// part is written; put(c, sum) runs in the CTA that finishes the sample, which gets
// true. Two levels: the CTA that finishes a set of about sqrt(slices) slices adds
// them, the one that finishes the last set adds the sets, so that no single CTA
// reads all slices (0.5 MB of a 33 MB sample's backward).
template <typename P, typename F>
__device__ bool finish_slice(const NormArgs& p, int b, int j, const P* part, int cols,
                             double2* sm, F put) {
  const int set = j / p.fan, members = min(p.fan, p.slices - set * p.fan);
  if (!last_of(p.done + (long long)b * p.sets + set, members)) return false;
  double2* sp = p.set_part + (long long)b * p.sets * cols;
  column_sums(part + ((long long)b * p.slices + set * p.fan) * cols, members, cols, sm,
              [&](int c, double2 v) { sp[(long long)set * cols + c] = v; });
  if (!last_of(p.sets_done + b, p.sets)) return false;
  column_sums(sp, p.sets, cols, sm, put);
  return true;
}

// (A, X) of a channel from the sums centred on mu rounded to float32.
__device__ __forceinline__ double2 finish_channel(const NormArgs& p, int b, int c, double2 v) {
  const double2 st = __ldg(p.stats + (long long)b * p.G + c / p.Cg);
  return make_double2(v.x, st.y * (v.y - (st.x - (double)(float)st.x) * v.x));
}

// dx = gamma r dz - r m1 - r^2 m2 (x - mu) with mu = muh + mul, from a group's
// sums of gamma dz and gamma dz (x - muh).
__device__ __forceinline__ float4 finish_coef(const NormArgs& p, double2 st, double2 v) {
  const double inv = 1.0 / ((double)p.S * p.Cg);
  const double muh = (double)(float)st.x, mul = st.x - muh;
  const double k2 = -st.y * st.y * st.y * (v.y - mul * v.x) * inv;
  return make_float4((float)st.x, (float)k2, (float)(-st.y * v.x * inv - k2 * mul), 0.f);
}

// dx's coefficients [G] of a sample whose channel sums [C] this CTA has just written.
template <typename T>
__device__ void finish_coef(const NormArgs& p, int b, const double2* sums, float4* coef) {
  const double2* stats = p.stats + (long long)b * p.G;
  __threadfence_block();
  cta_sync();
  const double inv = 1.0 / ((double)p.S * p.Cg);
  const int width = min(32, max(1, pow2_below(min(p.Cg, kT / min(p.G, kT)))));
  const int lane = threadIdx.x % width;
  for (int g0 = 0; g0 < p.G; g0 += kT / width) {
    const int g = g0 + threadIdx.x / width;
    double2 v = make_double2(0.0, 0.0);
    if (g < p.G) {
      for (int i = lane; i < p.Cg; i += width) {
        const int c = g * p.Cg + i;
        const double w = param<T>(p.weight, p.param_f32, c, 1.0);
        const double2 e = __ldcg(sums + c);
        v.x += w * e.x;
        v.y += w * e.y;
      }
    }
    v = lanes_sum(v, width);
    if (g < p.G && lane == 0) {
      const double2 st = __ldg(stats + g);
      // dx = gamma r dz - r m1 - r^2 m2 (x - mu), mu = muh + mul
      const double k2 = -st.y * st.y * v.y * inv;
      const double k3 = -st.y * v.x * inv - k2 * (st.x - (double)(float)st.x);
      coef[g] = make_float4((float)st.x, (float)k2, (float)k3, 0.f);
    }
  }
}

template <typename T>
__device__ void param_grads(const NormArgs& p, double2* sm) {
  column_sums(p.sums, p.B, p.C, sm, [&](int c, double2 v) {
    put_param<T>(p.dbias, p.param_f32, c, v.x);
    put_param<T>(p.dweight, p.param_f32, c, v.y);
  });
}

// ---- the plain kernels' order of work --------------------------------------------
// CTAs draw units from a ticket counter in the order
//   first(0) ... first(lag - 1) | first(lag), second(0), first(lag + 1), second(1), ... |
//   second(units - lag) ... second(units - 1)
// so a unit's second pass runs behind its first by its sample and the time that
// adding up the sums takes, with its rows still in L2, and HBM reads (first passes)
// overlap HBM writes (second passes). A second pass waits for all first passes of
// its sample; lag >= slices, so they have lower tickets, and a CTA finishes its
// tickets in increasing order: the lowest unfinished unit never waits, so every
// wait ends, however many CTAs are resident.
struct Unit {
  bool second;
  int b, j;
};
__device__ __forceinline__ Unit decode(const NormArgs& p, uint32_t t) {
  Unit u{false, 0, 0};
  uint32_t i = t;
  if (t >= p.lag && p.out) {
    const uint32_t r = t - p.lag, rest = p.units - p.lag;
    if (r < 2 * rest) {
      u.second = r & 1;
      i = r / 2 + (u.second ? 0 : p.lag);
    } else {
      u.second = true;
      i = r - rest;
    }
  }
  u.b = (int)(i / p.slices);
  u.j = (int)(i % p.slices);
  return u;
}

__device__ __forceinline__ void publish(uint32_t* flag) {
  cta_sync();
  if (threadIdx.x == 0) {
    __threadfence();
    asm volatile("st.release.gpu.u32 [%0], %1;" ::"l"(flag), "r"(1u) : "memory");
  }
}

static inline int read_norm_status(bool reset) {
  int v = 0;
  const int z = 0;
  if (cudaMemcpyFromSymbol(&v, norm_status, sizeof(int)) != cudaSuccess) return 0;
  if (reset && v) cudaMemcpyToSymbol(norm_status, &z, sizeof(int));
  return v;
}

// False, for every thread of the CTA, when the wait ran out: the CTA stops.
static __device__ bool wait_for(const NormArgs& p, const uint32_t* flag) {
  __shared__ int ok;
  if (threadIdx.x == 0) {
    const uint64_t t0 = tc::globaltimer();
    uint32_t v = 0;
    for (;;) {
      asm volatile("ld.acquire.gpu.u32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
      if (v || tc::globaltimer() - t0 >= p.wait_ns) break;
      __nanosleep(100);
    }
    if (!v) atomicExch(&norm_status, 1);
    ok = v != 0;
  }
  cta_sync();
  return ok;
}

}  // namespace lcb200
