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
// Numerics. A thread sums x - K and (x - K)^2 in float32 over its few dozen
// rows, K being its first value of the channel: what a far-off K costs is
// bounded by K's own share of the variance. Everything beyond a thread
// (partial sums, mean, 1/std, the per-channel factors) is float64, so the sums
// of different slices add without cancellation and the result does not depend
// on the order the slices finish in: partial sums have slots of their own and
// are added in a fixed order, with no float atomics.
// z = x a + b with a = gamma r, b = beta - mu a split into two floats each,
// which leaves the sign of z exact to ~2^-48: a rectifier's gradient jumps
// there, and forward and backward must agree on the side.
#include "feature_common.cuh"

namespace lcb200 {
namespace {

constexpr int kT = 256;      // threads of a CTA
constexpr int kUnroll = 4;   // rows a thread has in flight

struct NormArgs {
  const void* x;
  const void* dy;
  void* out;           // y or dx
  const void* weight;  // [C] or null
  const void* bias;    // [C] or null
  int param_f32;       // weight/bias dtype: float32, else x's
  double2* stats;      // [B, G] (mean, 1/std)
  long long S;
  int B, C, G, Cg;
  int act;
  float slope;
  double eps;
  int slices;           // slices of one sample
  long long slice_rows;
  // workspace
  uint32_t* done;       // [B + 1] finished slices per sample, finished samples
  double2* part;        // forward: [B, slices, G] (sum x, sum x^2)
  float2* bpart;        // backward: [B, slices, C] (sum dz, sum dz (x - mu))
  double2* sums;        // backward: [B, C] (A, X)
  float4* coef;         // backward: [B, G] (mu, k2, k3, 0): dx = gamma r dz + k2 (x - mu) + k3
  void* dweight;        // [C] or null
  void* dbias;
  DropArgs drop;
};

template <typename T>
__device__ __forceinline__ double param(const void* p, int f32, int c, double none) {
  if (!p) return none;
  return f32 ? (double)__ldg(reinterpret_cast<const float*>(p) + c)
             : (double)ldf(reinterpret_cast<const T*>(p) + c);
}

template <typename T>
__device__ __forceinline__ void put_param(void* p, int f32, int c, double v) {
  if (!p) return;
  if (f32) reinterpret_cast<float*>(p)[c] = (float)v;
  else stf(reinterpret_cast<T*>(p) + c, (float)v);
}

// sigma(z); exp(-z) overflowing to infinity gives 0.
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
  __device__ __forceinline__ Place(int cols, int cb) {
    nc = min(cols - cb, kT);
    rp = kT / nc;
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

// ---- forward, first pass: slice sums, and the sample's statistics -----------------
template <typename T, int V>
__device__ void stats_slice(const NormArgs& p, int b, int j, double2* sm) {
  const int cols = p.C / V;
  const long long r0 = j * p.slice_rows, r1 = min(p.S, r0 + p.slice_rows);
  const T* xb = reinterpret_cast<const T*>(p.x) + (long long)b * p.S * p.C;
  double2* out = p.part + ((long long)b * p.slices + j) * p.G;
  const bool whole = p.Cg % V == 0;  // a vector lies in one group
  const int per = whole ? 1 : V;     // shared entries of a thread
  const int gw = p.Cg * per / V;     // entries of one group and row (whole: Cg / V)
  for (int cb = 0; cb < cols; cb += kT) {
    const Place at(cols, cb);
    if (at.on) {
      float s[V], q[V], k[V];
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = q[v] = k[v] = 0.f;
      int n = 0;
      const T* ptr = xb + (long long)at.col * V;
      long long r = r0 + at.row;
      if (r < r1) {
        Vec<T, V>::unpack(Vec<T, V>::load(ptr + r * p.C), k);
        n = 1;
        r += at.rp;
      }
      const long long step = at.rp;
      for (; r + (kUnroll - 1) * step < r1; r += kUnroll * step) {
        typename Vec<T, V>::Raw raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) raw[u] = Vec<T, V>::load(ptr + (r + u * step) * p.C);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          float f[V];
          Vec<T, V>::unpack(raw[u], f);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float d = f[v] - k[v];
            s[v] += d;
            q[v] = fmaf(d, d, q[v]);
          }
        }
        n += kUnroll;
      }
      for (; r < r1; r += step) {
        float f[V];
        Vec<T, V>::unpack(Vec<T, V>::load(ptr + r * p.C), f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = f[v] - k[v];
          s[v] += d;
          q[v] = fmaf(d, d, q[v]);
        }
        ++n;
      }
      // sum x = s + n K, sum x^2 = q + 2 K s + n K^2, in float64
      double2 tot = make_double2(0.0, 0.0);
      double2* dst = sm + ((long long)at.row * at.nc + (at.col - cb)) * per;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const double kv = k[v], sv = s[v];
        const double2 e = make_double2(sv + n * kv, (double)q[v] + kv * (2.0 * sv + n * kv));
        if (whole) {
          tot.x += e.x;
          tot.y += e.y;
        } else {
          dst[v] = e;
        }
      }
      if (whole) dst[0] = tot;
    }
    __syncthreads();
    // groups that overlap this column block, `width` lanes each
    const int ne = at.nc * per;                  // entries of one row
    const int first = (int)((long long)cb * V / p.Cg);
    const int last = (int)(((long long)(cb + at.nc) * V - 1) / p.Cg);
    const int width = min(32, max(1, pow2_below(min(at.rp * gw, kT / (last - first + 1)))));
    const int lane = threadIdx.x % width;
    for (int g0 = first; g0 <= last; g0 += kT / width) {
      const int g = g0 + threadIdx.x / width;
      double2 v = make_double2(0.0, 0.0);
      if (g <= last) {
        const int e0 = max(0, g * gw - cb * per), e1 = min(ne, (g + 1) * gw - cb * per);
        const int w = e1 - e0;
        for (int i = lane; i < at.rp * w; i += width) {
          const double2 e = sm[(i / w) * ne + e0 + i % w];
          v.x += e.x;
          v.y += e.y;
        }
      }
      v = lanes_sum(v, width);
      if (g <= last && lane == 0) {
        // a group cut by the previous column block adds to its first part
        if ((long long)g * p.Cg < (long long)cb * V) {
          v.x += out[g].x;
          v.y += out[g].y;
        }
        out[g] = v;
      }
    }
    __syncthreads();
  }
}

__device__ void stats_finish(const NormArgs& p, int b) {
  const int width = min(32, max(1, pow2_below(min(p.slices, kT / min(p.G, kT)))));
  const int lane = threadIdx.x % width;
  const double inv = 1.0 / ((double)p.S * p.Cg);
  for (int g0 = 0; g0 < p.G; g0 += kT / width) {
    const int g = g0 + threadIdx.x / width;
    double2 v = make_double2(0.0, 0.0);
    if (g < p.G) {
      const double2* src = p.part + (long long)b * p.slices * p.G + g;
#pragma unroll 4
      for (int j = lane; j < p.slices; j += width) {
        const double2 e = __ldcg(src + (long long)j * p.G);
        v.x += e.x;
        v.y += e.y;
      }
    }
    v = lanes_sum(v, width);
    if (g < p.G && lane == 0) {
      const double mean = v.x * inv;
      double var = v.y * inv - mean * mean;
      var = var < 0.0 ? 0.0 : var;  // rounding below zero; NaN stays
      p.stats[(long long)b * p.G + g] = make_double2(mean, 1.0 / sqrt(var + p.eps));
    }
  }
}

// True in every thread of the CTA that finished last of `count` at *counter;
// what the others wrote before is then visible.
__device__ bool last_of(uint32_t* counter, uint32_t count) {
  __shared__ int is_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicAdd(counter, 1u) == count - 1;
    __threadfence();
  }
  __syncthreads();
  return is_last;
}

template <typename T, int V>
__global__ void __launch_bounds__(kT) norm_stats_kernel(NormArgs p) {
  __shared__ double2 sm[kT * V];
  const int b = blockIdx.x / p.slices, j = blockIdx.x % p.slices;
  stats_slice<T, V>(p, b, j, sm);
  if (last_of(p.done + b, p.slices)) stats_finish(p, b);
}

// ---- forward, second pass ------------------------------------------------------------
template <typename T, int V, bool DROP>
__device__ void apply_slice(const NormArgs& p, int b, int j) {
  const int cols = p.C / V;
  const long long r0 = j * p.slice_rows, r1 = min(p.S, r0 + p.slice_rows);
  const long long base = (long long)b * p.S * p.C;
  DropStream ds;
  if (DROP) ds = drop_stream(p.drop);
  for (int cb = 0; cb < cols; cb += kT) {
    const Place at(cols, cb);
    if (!at.on) continue;
    Affine f[V];
    const int c0 = at.col * V;
#pragma unroll
    for (int v = 0; v < V; ++v)
      f[v] = affine<T>(p, __ldcg(p.stats + (long long)b * p.G + (c0 + v) / p.Cg), c0 + v);
    uint32_t keep = ~0u;
    if (DROP && p.drop.channel) keep = drop_keep<V>(ds, p.drop.threshold, (long long)b * p.C + c0);
    const T* src = reinterpret_cast<const T*>(p.x) + base + c0;
    T* dst = reinterpret_cast<T*>(p.out) + base + c0;
    auto one = [&](typename Vec<T, V>::Raw raw, long long r) {
      float x[V];
      Vec<T, V>::unpack(raw, x);
      uint32_t m = keep;
      if (DROP && !p.drop.channel) m = drop_keep<V>(ds, p.drop.threshold, base + r * p.C + c0);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = act_value(affine_z(f[v], x[v]), p.act, p.slope);
        if (DROP) x[v] = (m >> v) & 1 ? x[v] * p.drop.factor : 0.f;
      }
      Vec<T, V>::store(dst + r * p.C, Vec<T, V>::pack(x));
    };
    long long r = r0 + at.row;
    const long long step = at.rp;
    for (; r + (kUnroll - 1) * step < r1; r += kUnroll * step) {
      typename Vec<T, V>::Raw raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) raw[u] = Vec<T, V>::load_last(src + (r + u * step) * p.C);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) one(raw[u], r + u * step);
    }
    for (; r < r1; r += step) one(Vec<T, V>::load_last(src + r * p.C), r);
  }
}

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT) norm_apply_kernel(NormArgs p) {
  drop_keep_stream(p.drop);
  apply_slice<T, V, DROP>(p, blockIdx.x / p.slices, blockIdx.x % p.slices);
}

// ---- backward, first pass: per-channel sums of dz and dz (x - mu) --------------------
// dz of one vector, in place of the output gradient g.
template <int V, bool DROP>
__device__ __forceinline__ void to_dz(const NormArgs& p, const Affine (&f)[V],
                                      const float (&x)[V], float (&g)[V], uint32_t m) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (DROP) g[v] = (m >> v) & 1 ? g[v] * p.drop.factor : 0.f;
    if (p.act != LCB200_ACT_NONE) g[v] = act_grad(affine_z(f[v], x[v]), g[v], p.act, p.slope);
  }
}

template <typename T, int V, bool DROP>
__device__ void grad_sums_slice(const NormArgs& p, int b, int j, float2* sm) {
  const int cols = p.C / V;
  const long long r0 = j * p.slice_rows, r1 = min(p.S, r0 + p.slice_rows);
  const long long base = (long long)b * p.S * p.C;
  float2* out = p.bpart + ((long long)b * p.slices + j) * p.C;
  DropStream ds;
  if (DROP) ds = drop_stream(p.drop);
  for (int cb = 0; cb < cols; cb += kT) {
    const Place at(cols, cb);
    if (at.on) {
      Affine f[V];
      float mu[V], sa[V], sx[V];
      const int c0 = at.col * V;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const double2 st = __ldg(p.stats + (long long)b * p.G + (c0 + v) / p.Cg);
        f[v] = affine<T>(p, st, c0 + v);
        mu[v] = (float)st.x;
        sa[v] = sx[v] = 0.f;
      }
      uint32_t keep = ~0u;
      if (DROP && p.drop.channel)
        keep = drop_keep<V>(ds, p.drop.threshold, (long long)b * p.C + c0);
      const T* xs = reinterpret_cast<const T*>(p.x) + base + c0;
      const T* gs = reinterpret_cast<const T*>(p.dy) + base + c0;
      auto one = [&](typename Vec<T, V>::Raw xr, typename Vec<T, V>::Raw gr, long long r) {
        float x[V], g[V];
        Vec<T, V>::unpack(xr, x);
        Vec<T, V>::unpack(gr, g);
        uint32_t m = keep;
        if (DROP && !p.drop.channel) m = drop_keep<V>(ds, p.drop.threshold, base + r * p.C + c0);
        to_dz<V, DROP>(p, f, x, g, m);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          sa[v] += g[v];
          sx[v] = fmaf(g[v], x[v] - mu[v], sx[v]);
        }
      };
      long long r = r0 + at.row;
      const long long step = at.rp;
      constexpr int U = kUnroll / 2;
      for (; r + (U - 1) * step < r1; r += U * step) {
        typename Vec<T, V>::Raw xr[U], gr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          xr[u] = Vec<T, V>::load(xs + (r + u * step) * p.C);
          gr[u] = Vec<T, V>::load(gs + (r + u * step) * p.C);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) one(xr[u], gr[u], r + u * step);
      }
      for (; r < r1; r += step)
        one(Vec<T, V>::load(xs + r * p.C), Vec<T, V>::load(gs + r * p.C), r);
#pragma unroll
      for (int v = 0; v < V; ++v)
        sm[(at.row * at.nc + (at.col - cb)) * V + v] = make_float2(sa[v], sx[v]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < at.nc * V; i += kT) {
      float2 v = make_float2(0.f, 0.f);
      for (int k = 0; k < at.rp; ++k) {
        const float2 e = sm[k * at.nc * V + i];
        v.x += e.x;
        v.y += e.y;
      }
      out[cb * V + i] = v;
    }
    __syncthreads();
  }
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
    __syncthreads();
    if (part == 0) {
      for (int k = 1; k < parts; ++k) {
        v.x += sm[k * nc + c].x;
        v.y += sm[k * nc + c].y;
      }
      put(cb + c, v);
    }
    __syncthreads();
  }
}

template <typename T>
__device__ void grad_finish(const NormArgs& p, int b, double2* sm) {
  const double2* stats = p.stats + (long long)b * p.G;
  double2* sums = p.sums + (long long)b * p.C;
  column_sums(p.bpart + (long long)b * p.slices * p.C, p.slices, p.C, sm, [&](int c, double2 v) {
    // the slices centred on mu rounded to float32
    const double2 st = __ldg(stats + c / p.Cg);
    sums[c] = make_double2(v.x, st.y * (v.y - (st.x - (double)(float)st.x) * v.x));
  });
  __threadfence_block();
  __syncthreads();
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
      p.coef[(long long)b * p.G + g] = make_float4((float)st.x, (float)k2, (float)k3, 0.f);
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

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT) norm_grad_sums_kernel(NormArgs p) {
  __shared__ __align__(16) float2 sm[kT * (V < 2 ? 2 : V)];  // also kT double2 sums
  const int b = blockIdx.x / p.slices, j = blockIdx.x % p.slices;
  grad_sums_slice<T, V, DROP>(p, b, j, sm);
  double2* smd = reinterpret_cast<double2*>(sm);
  if (!last_of(p.done + b, p.slices)) return;
  grad_finish<T>(p, b, smd);
  if (last_of(p.done + p.B, p.B)) param_grads<T>(p, smd);
}

// ---- backward, second pass --------------------------------------------------------------
template <typename T, int V, bool DROP>
__device__ void grad_input_slice(const NormArgs& p, int b, int j) {
  const int cols = p.C / V;
  const long long r0 = j * p.slice_rows, r1 = min(p.S, r0 + p.slice_rows);
  const long long base = (long long)b * p.S * p.C;
  DropStream ds;
  if (DROP) ds = drop_stream(p.drop);
  for (int cb = 0; cb < cols; cb += kT) {
    const Place at(cols, cb);
    if (!at.on) continue;
    Affine f[V];
    float mu[V], k2[V], k3[V];
    const int c0 = at.col * V;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const long long g = (long long)b * p.G + (c0 + v) / p.Cg;
      f[v] = affine<T>(p, __ldg(p.stats + g), c0 + v);
      const float4 k = __ldcg(p.coef + g);
      mu[v] = k.x;
      k2[v] = k.y;
      k3[v] = k.z;
    }
    uint32_t keep = ~0u;
    if (DROP && p.drop.channel) keep = drop_keep<V>(ds, p.drop.threshold, (long long)b * p.C + c0);
    const T* xs = reinterpret_cast<const T*>(p.x) + base + c0;
    const T* gs = reinterpret_cast<const T*>(p.dy) + base + c0;
    T* dst = reinterpret_cast<T*>(p.out) + base + c0;
    auto one = [&](typename Vec<T, V>::Raw xr, typename Vec<T, V>::Raw gr, long long r) {
      float x[V], g[V];
      Vec<T, V>::unpack(xr, x);
      Vec<T, V>::unpack(gr, g);
      uint32_t m = keep;
      if (DROP && !p.drop.channel) m = drop_keep<V>(ds, p.drop.threshold, base + r * p.C + c0);
      to_dz<V, DROP>(p, f, x, g, m);
#pragma unroll
      for (int v = 0; v < V; ++v)
        g[v] = fmaf(f[v].ah, g[v], fmaf(k2[v], x[v] - mu[v], k3[v]));
      Vec<T, V>::store(dst + r * p.C, Vec<T, V>::pack(g));
    };
    long long r = r0 + at.row;
    const long long step = at.rp;
    constexpr int U = kUnroll / 2;
    for (; r + (U - 1) * step < r1; r += U * step) {
      typename Vec<T, V>::Raw xr[U], gr[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        xr[u] = Vec<T, V>::load_last(xs + (r + u * step) * p.C);
        gr[u] = Vec<T, V>::load_last(gs + (r + u * step) * p.C);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) one(xr[u], gr[u], r + u * step);
    }
    for (; r < r1; r += step)
      one(Vec<T, V>::load_last(xs + r * p.C), Vec<T, V>::load_last(gs + r * p.C), r);
  }
}

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT) norm_grad_input_kernel(NormArgs p) {
  grad_input_slice<T, V, DROP>(p, blockIdx.x / p.slices, blockIdx.x % p.slices);
}

// ---- host ---------------------------------------------------------------------------------
// Slices of a sample: about 64 KB of rows each, smaller while the batch does
// not give every multiprocessor four of them, but at least four rows a thread
// when rows are as narrow as the CTA.
void plan_slices(int B, long long S, int C, int dtype, int* slices, long long* slice_rows) {
  const size_t es = dtype_bytes(dtype);
  const long long row_bytes = (long long)C * es;
  const long long rp = std::max<long long>(1, kT * 16ll / row_bytes);  // rows of one CTA step
  long long rows = std::max<long long>(1, 65536 / row_bytes);
  const long long want = 4ll * device_sms();
  const long long even = (long long)((double)S * B / want) + 1;
  rows = std::min(rows, even);
  rows = std::min(S, std::max(rows, 4 * rp));
  *slice_rows = rows;
  *slices = (int)((S + rows - 1) / rows);
}

struct Layout {
  size_t done, part, sums, coef, total;
};
Layout layout(int B, int C, int G, int slices, bool backward) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  Layout l{};
  size_t at = 0;
  l.done = at;
  at = up(at + sizeof(uint32_t) * ((size_t)B + 1));
  l.part = at;
  at = up(at + (backward ? sizeof(float2) * (size_t)C : sizeof(double2) * (size_t)G) * B * slices);
  if (backward) {
    l.sums = at;
    at = up(at + sizeof(double2) * (size_t)B * C);
    l.coef = at;
    at = up(at + sizeof(float4) * (size_t)B * G);
  }
  l.total = at;
  return l;
}

template <typename T, int V, bool DROP>
bool launch_forward(const NormArgs& p, cudaStream_t s) {
  const unsigned grid = (unsigned)((long long)p.B * p.slices);
  norm_stats_kernel<T, V><<<grid, kT, 0, s>>>(p);
  norm_apply_kernel<T, V, DROP><<<grid, kT, 0, s>>>(p);
  count_launch(2);
  return check_launch("group norm");
}

template <typename T, int V, bool DROP>
bool launch_backward(const NormArgs& p, cudaStream_t s) {
  const unsigned grid = (unsigned)((long long)p.B * p.slices);
  norm_grad_sums_kernel<T, V, DROP><<<grid, kT, 0, s>>>(p);
  count_launch();
  if (p.out) {
    norm_grad_input_kernel<T, V, DROP><<<grid, kT, 0, s>>>(p);
    count_launch();
  }
  return check_launch("group norm backward");
}

template <typename T, int V>
bool launch_v(const NormArgs& p, bool backward, cudaStream_t s) {
  const bool drop = p.drop.threshold != 0;
  if (backward) return drop ? launch_backward<T, V, true>(p, s) : launch_backward<T, V, false>(p, s);
  return drop ? launch_forward<T, V, true>(p, s) : launch_forward<T, V, false>(p, s);
}

template <typename T>
bool launch_t(const NormArgs& p, int dtype, bool backward, cudaStream_t s) {
  switch (vec_width(dtype, p.C, p.x, p.out, p.dy)) {
    case 8: return launch_v<T, (sizeof(T) == 2 ? 8 : 4)>(p, backward, s);
    case 4: return launch_v<T, 4>(p, backward, s);
    case 2: return launch_v<T, 2>(p, backward, s);
    default: return launch_v<T, 1>(p, backward, s);
  }
}

bool launch(const NormArgs& p, int dtype, bool backward, cudaStream_t s) {
  if (dtype == LCB200_F32) return launch_t<float>(p, dtype, backward, s);
  if (dtype == LCB200_F16) return launch_t<__half>(p, dtype, backward, s);
  return launch_t<__nv_bfloat16>(p, dtype, backward, s);
}

}  // namespace

size_t feature_norm_workspace(int B, long long S, int C, int G, int dtype, bool backward) {
  int slices;
  long long rows;
  plan_slices(B, S, C, dtype, &slices, &rows);
  return layout(B, C, G, slices, backward).total;
}

bool feature_norm(const void* x, const void* dy, const void* weight, const void* bias, void* out,
                  double* stats, void* dweight, void* dbias, int B, long long S, int C, int G,
                  int dtype, bool param_f32, double eps, int act, float slope,
                  const DropArgs& drop, void* ws, size_t ws_bytes, bool backward,
                  cudaStream_t s) {
  NormArgs p{};
  p.x = x;
  p.dy = dy;
  p.out = out;
  p.weight = weight;
  p.bias = bias;
  p.param_f32 = param_f32;
  p.stats = reinterpret_cast<double2*>(stats);
  p.S = S;
  p.B = B;
  p.C = C;
  p.G = G;
  p.Cg = C / G;
  p.act = act;
  p.slope = slope;
  p.eps = eps;
  p.dweight = dweight;
  p.dbias = dbias;
  p.drop = drop;
  plan_slices(B, S, C, dtype, &p.slices, &p.slice_rows);
  if ((long long)B * p.slices > 0x7fffffffll) {
    set_error("group norm: too many samples");
    return false;
  }
  const Layout l = layout(B, C, G, p.slices, backward);
  if (!ws || ws_bytes < l.total || (reinterpret_cast<uintptr_t>(ws) & 15)) {
    set_error("group norm: needs a 16-byte aligned workspace of " + std::to_string(l.total) +
              " B, got " + std::to_string(ws_bytes));
    return false;
  }
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.done = reinterpret_cast<uint32_t*>(w + l.done);
  p.part = reinterpret_cast<double2*>(w + l.part);
  p.bpart = reinterpret_cast<float2*>(w + l.part);
  p.sums = reinterpret_cast<double2*>(w + l.sums);
  p.coef = reinterpret_cast<float4*>(w + l.coef);
  if (cudaMemsetAsync(p.done, 0, sizeof(uint32_t) * ((size_t)B + 1), s) != cudaSuccess)
    return check_launch("group norm: memset of the counters");
  return launch(p, dtype, backward, s);
}

}  // namespace lcb200
