// Group norm: plan and launch, the kernels for whole samples, and the plain kernels for
// maps that the streamed ones (norm_stream.cu) do not take: rows that are no whole
// number of aligned 16-byte vectors, too wide, or of too many groups. The plain kernels
// move 0.6 to 2.4 TB/s where the streamed ones move 2.7 to 4.2: 8 x 32400 x 99 float16, element
// by element, takes 97 us forward and 211 backward, x 96 takes 32 and 54; 8 x 6400 x 2304,
// wider than a CTA, takes 200 and 1105 (each slice of 16 rows writes and reads again a pair
// of sums for every channel).
#include <atomic>

#include "norm_common.cuh"

namespace lcb200 {

Streamed stream_norm(const NormArgs& p, int dtype, bool backward, cudaStream_t s);
int stream_norm_status(bool reset);
int stream_ctas();  // resident CTAs
int stream_stage_rows(int C, int dtype, bool backward);  // rows of a stage, at least 1

namespace {

std::atomic<long long> wait_limit{2000000000};  // ns

// ---- forward, first pass: slice sums, and the sample's statistics -----------------
template <typename T, int V>
__device__ void stats_slice(const NormArgs& p, int b, int j, double2* out, double2* sm) {
  const int cols = p.C / V;
  const long long r0 = j * p.slice_rows, r1 = min(p.S, r0 + p.slice_rows);
  const T* xb = reinterpret_cast<const T*>(p.x) + (long long)b * p.S * p.C;
  const bool whole = p.Cg % V == 0;  // a vector lies in one group
  const int per = whole ? 1 : V;     // shared entries of a thread
  const int gw = whole ? p.Cg / V : p.Cg;  // entries of one group and row
  for (int cb = 0; cb < cols; cb += kT) {
    const Place at(cols, cb);
    if (at.on) {
      double s[V], q[V], k[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[v] = q[v] = 0.0;
        k[v] = group_shift<T>(p, b, (at.col * V + v) / p.Cg);
      }
      const T* ptr = xb + (long long)at.col * V;
      const long long step = at.rp;
      auto one = [&](typename Vec<T, V>::Raw raw) {
        float f[V];
        Vec<T, V>::unpack(raw, f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const double d = (double)f[v] - k[v];
          s[v] += d;
          q[v] = fma(d, d, q[v]);
        }
      };
      long long r = r0 + at.row;
      for (; r + (kUnroll - 1) * step < r1; r += kUnroll * step) {
        typename Vec<T, V>::Raw raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) raw[u] = Vec<T, V>::load(ptr + (r + u * step) * p.C);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) one(raw[u]);
      }
      for (; r < r1; r += step) one(Vec<T, V>::load(ptr + r * p.C));
      double2 tot = make_double2(0.0, 0.0);
      double2* dst = sm + ((long long)at.row * at.nc + (at.col - cb)) * per;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const double2 e = make_double2(s[v], q[v]);
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

// ---- forward, second pass ------------------------------------------------------------
// z = (x - muh) a + b with muh = mu rounded to float32 and b = beta - (mu - muh) a.
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
    float mu[V], a[V], c[V];
    const int c0 = at.col * V;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const double2 st = __ldcg(p.stats + (long long)b * p.G + (c0 + v) / p.Cg);
      mu[v] = (float)st.x;
      a[v] = (float)(param<T>(p.weight, p.param_f32, c0 + v, 1.0) * st.y);
      c[v] = (float)(param<T>(p.bias, p.param_f32, c0 + v, 0.0) -
                     (st.x - (double)mu[v]) * (double)a[v]);
    }
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
        x[v] = act_value(fmaf(x[v] - mu[v], a[v], c[v]), p.act, p.slope);
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
__device__ void grad_sums_slice(const NormArgs& p, int b, int j, float2* out, float2* sm) {
  const int cols = p.C / V;
  const long long r0 = j * p.slice_rows, r1 = min(p.S, r0 + p.slice_rows);
  const long long base = (long long)b * p.S * p.C;
  DropStream ds;
  if (DROP) ds = drop_stream(p.drop);
  for (int cb = 0; cb < cols; cb += kT) {
    const Place at(cols, cb);
    if (at.on) {
      Affine f[V];
      float mu[V], sa[V], sx[V];
      double ta[V], tx[V];
      const int c0 = at.col * V;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const double2 st = __ldg(p.stats + (long long)b * p.G + (c0 + v) / p.Cg);
        f[v] = affine<T>(p, st, c0 + v);
        mu[v] = (float)st.x;
        sa[v] = sx[v] = 0.f;
        ta[v] = tx[v] = 0.0;
      }
      auto fold = [&]() {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          ta[v] += sa[v];
          tx[v] += sx[v];
          sa[v] = sx[v] = 0.f;
        }
      };
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
      // 16-byte vectors: 16 rows a thread at most, narrower ones up to 150
      constexpr bool kFolds = V * sizeof(T) < 16;
      for (int n = 1; r + (U - 1) * step < r1; r += U * step, ++n) {
        typename Vec<T, V>::Raw xr[U], gr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          xr[u] = Vec<T, V>::load(xs + (r + u * step) * p.C);
          gr[u] = Vec<T, V>::load(gs + (r + u * step) * p.C);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) one(xr[u], gr[u], r + u * step);
        if (kFolds && n % (kRun / U) == 0) fold();
      }
      for (; r < r1; r += step)
        one(Vec<T, V>::load(xs + r * p.C), Vec<T, V>::load(gs + r * p.C), r);
      fold();
#pragma unroll
      for (int v = 0; v < V; ++v)
        sm[(at.row * at.nc + (at.col - cb)) * V + v] = make_float2((float)ta[v], (float)tx[v]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < at.nc * V; i += kT) {
      double2 v = make_double2(0.0, 0.0);
      for (int k = 0; k < at.rp; ++k) {
        const float2 e = sm[k * at.nc * V + i];
        v.x += e.x;
        v.y += e.y;
      }
      out[cb * V + i] = make_float2((float)v.x, (float)v.y);
    }
    __syncthreads();
  }
}

// ---- backward, second pass --------------------------------------------------------------
template <typename T, int V, bool DROP>
__device__ void grad_input_slice(const NormArgs& p, int b, int j, const float4* coef) {
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
      const int g = (c0 + v) / p.Cg;
      f[v] = affine<T>(p, __ldg(p.stats + (long long)b * p.G + g), c0 + v);
      const float4 k = __ldcg(coef + g);
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

// ---- the kernels: both passes of every chunk --------------------------------------------
template <typename F>
__device__ void run_units(const NormArgs& p, F unit) {
  __shared__ uint32_t s_next;
  if (threadIdx.x == 0) s_next = atomicAdd(p.ticket, 1u);
  __syncthreads();
  uint32_t t = s_next;
  while (t < p.tickets) {
    uint32_t next = 0;
    if (threadIdx.x == 0) next = atomicAdd(p.ticket, 1u);  // arrives during the unit
    const Unit u = decode(p, t);
    if (!unit(u.second, u.b, u.j)) return;
    __syncthreads();
    if (threadIdx.x == 0) s_next = next;
    __syncthreads();
    t = s_next;
  }
}

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT, kOcc) norm_forward_kernel(NormArgs p) {
  __shared__ double2 sm[kT * V];
  drop_keep_stream(p.drop);
  run_units(p, [&](bool second, int b, int j) {
    if (!second) {
      stats_slice<T, V>(p, b, j, p.part + ((long long)b * p.slices + j) * p.G, sm);
      if (finish_slice(p, b, j, p.part, p.G, sm, [&](int g, double2 t) {
            p.stats[(long long)b * p.G + g] = finish_stats(p, t, group_shift<T>(p, b, g));
          }))
        publish(p.ready + b);
      return true;
    }
    if (!wait_for(p, p.ready + b)) return false;
    apply_slice<T, V, DROP>(p, b, j);
    return true;
  });
}

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT, kOcc) norm_backward_kernel(NormArgs p) {
  __shared__ __align__(16) float2 sm[kT * (V < 2 ? 2 : V)];  // also kT double2 sums
  double2* smd = reinterpret_cast<double2*>(sm);
  run_units(p, [&](bool second, int b, int j) {
    if (!second) {
      grad_sums_slice<T, V, DROP>(p, b, j, p.bpart + ((long long)b * p.slices + j) * p.C, sm);
      double2* sums = p.sums + (long long)b * p.C;
      if (finish_slice(p, b, j, p.bpart, p.C, smd,
                       [&](int c, double2 t) { sums[c] = finish_channel(p, b, c, t); })) {
        finish_coef<T>(p, b, sums, p.coef + (long long)b * p.G);
        publish(p.ready + b);
        if (last_of(p.ticket + 1, p.B)) param_grads<T>(p, smd);
      }
      return true;
    }
    if (!wait_for(p, p.ready + b)) return false;
    grad_input_slice<T, V, DROP>(p, b, j, p.coef + (long long)b * p.G);
    return true;
  });
}

// ---- whole samples ------------------------------------------------------------------------
// A CTA makes both passes of a sample: nothing to exchange, one ordinary launch, the
// second read out of L1 and L2. For samples too small to divide and for many small ones.
// Partial sums, coefficients and sums of the parameters' gradients are the CTA's own.
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT, kOcc) norm_forward_samples(NormArgs p) {
  __shared__ double2 sm[kT * V];
  drop_keep_stream(p.drop);
  double2* part = p.part + (long long)blockIdx.x * p.G;
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    stats_slice<T, V>(p, b, 0, part, sm);
    for (int g = threadIdx.x; g < p.G; g += kT)
      p.stats[(long long)b * p.G + g] = finish_stats(p, __ldcg(part + g), group_shift<T>(p, b, g));
    cta_sync();
    apply_slice<T, V, DROP>(p, b, 0);
  }
}

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(kT, kOcc) norm_backward_samples(NormArgs p) {
  __shared__ __align__(16) float2 sm[kT * (V < 2 ? 2 : V)];
  const long long own = blockIdx.x;
  float2* bpart = p.bpart + own * p.C;
  double2 *sums = p.set_part + own * p.C, *total = p.sums + own * p.C;
  float4* coef = p.coef + own * p.G;
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    grad_sums_slice<T, V, DROP>(p, b, 0, bpart, sm);
    for (int c = threadIdx.x; c < p.C; c += kT) {
      const double2 v = finish_channel(p, b, c, as_double2(__ldcg(bpart + c)));
      sums[c] = v;
      double2 t = b < (int)gridDim.x ? make_double2(0.0, 0.0) : total[c];
      t.x += v.x;
      t.y += v.y;
      total[c] = t;
      if (gridDim.x == 1 && b + 1 == p.B) {
        put_param<T>(p.dbias, p.param_f32, c, t.x);
        put_param<T>(p.dweight, p.param_f32, c, t.y);
      }
    }
    finish_coef<T>(p, b, sums, coef);
    cta_sync();
    if (p.out) grad_input_slice<T, V, DROP>(p, b, 0, coef);
    cta_sync();
  }
}

// Weight and bias gradients from the CTAs' channel sums [n, C]: two channels
// a CTA (a 32-byte sector a row), rows over its threads, a fixed order throughout.
constexpr int kParamChannels = 2;
template <typename T>
__global__ void __launch_bounds__(kT) norm_params_kernel(NormArgs p, int n) {
  __shared__ double2 sm[kT];
  constexpr int kRows = kT / kParamChannels;
  const int k = threadIdx.x % kParamChannels, c = blockIdx.x * kParamChannels + k;
  double2 v = make_double2(0.0, 0.0);
  if (c < p.C) {
#pragma unroll 4
    for (int i = threadIdx.x / kParamChannels; i < n; i += kRows) {
      const double2 e = __ldg(p.sums + (long long)i * p.C + c);
      v.x += e.x;
      v.y += e.y;
    }
  }
  sm[threadIdx.x] = v;
  for (int o = kT / 2; o >= kParamChannels; o /= 2) {
    __syncthreads();
    if (threadIdx.x < o) {
      sm[threadIdx.x].x += sm[threadIdx.x + o].x;
      sm[threadIdx.x].y += sm[threadIdx.x + o].y;
    }
  }
  if (threadIdx.x < kParamChannels && c < p.C) {
    put_param<T>(p.dbias, p.param_f32, c, sm[threadIdx.x].x);
    put_param<T>(p.dweight, p.param_f32, c, sm[threadIdx.x].y);
  }
}

template <typename T>
bool launch_params(const NormArgs& p, int n, cudaStream_t s) {
  if (!p.dweight && !p.dbias) return true;
  norm_params_kernel<T><<<(p.C + kParamChannels - 1) / kParamChannels, kT, 0, s>>>(p, n);
  count_launch();
  return check_launch("group norm parameter gradients");
}

// ---- host ---------------------------------------------------------------------------------
// The streamed kernels take rows of whole 16-byte vectors, one a thread at most, and up
// to 512 groups: their per-group values share a CTA's memory with the ring, and two
// CTAs have to fit a multiprocessor.
bool streams(int C, int G, int dtype, int width) {
  const int full = 16 / (int)dtype_bytes(dtype);
  return width == full && C / full <= kT && G <= 512;
}

struct Plan {
  bool samples;  // whole samples
  int slices, fan, sets;
  long long slice_rows;
  uint32_t units, lag;
  int teams, ctas, stage_rows, chunk, chunks;
  long long slots;
  bool ok;
};

Plan make_plan(int B, long long S, int C, int dtype, bool backward) {
  Plan q{};
  const size_t es = dtype_bytes(dtype);
  const double maps = backward ? 2 : 1;
  // plain kernels: units of 64 KB, fewer rows while the batch does not give every CTA
  // two of them; a second pass 32 MB behind its first
  const long long rp = std::max<long long>(1, (long long)kT * 16 / (long long)(C * es));
  const long long step = 4 * rp, slots = (long long)device_sms() * kOcc;
  const long long n = (long long)std::min<double>(4, (double)S * B / (double)(2 * slots * step));
  q.slice_rows = std::min<long long>(S, std::max<long long>(1, n) * step);
  // whole samples where one CTA's two passes cost less than the exchange between CTAs.
  // Measured with C = 256 float16, 1 and 300 samples, whole against divided: forward
  // 64 KB a sample 8.6 and 14.7 us against 12.4 and 26.4, 256 KB 18.9 and 47.7 against
  // 10.3 and 45.7; backward 8 KB 9.6 and 17.5 against 15.4 and 30.1, 32 KB 14.4 against
  // 16.5, 64 KB 21.4 and 39.2 against 14.4 and 42.4
  q.samples = (double)S * C * es <= (backward ? 32 : 128) * 1024;
  if (q.samples) q.slice_rows = S;
  const long long slices = (S + q.slice_rows - 1) / q.slice_rows, units = slices * B;
  q.slices = (int)slices;
  q.units = (uint32_t)units;
  q.lag = (uint32_t)std::min<long long>(
      units, slices + (long long)((32 << 20) / (maps * q.slice_rows * C * es)));
  // streamed kernels: up to 16 MB one chunk for both teams together, else an even number
  // of chunks of up to 72 MB, backward 160 MB. Smaller ones would be read a second time
  // out of L2 altogether, but each exchange of sums costs more than that saves. In chunks
  // of 33, 66 and 133 MB 8 x 135 x 240 x 256 float16 takes 74, 72 and 72 us forward, 142,
  // 129 and 119 us backward; 8 x 540 x 960 x 64 in chunks of 66 and 133 MB 254 and 264 us
  const double total = maps * (double)S * B * C * es, target = (backward ? 160 : 72) << 20;
  const long long k = std::min<long long>(
      B, total < (16 << 20) ? 1 : 2 * (long long)(total / (2 * target)) + 2);
  q.chunk = (int)((B + k - 1) / k);
  q.chunks = (B + q.chunk - 1) / q.chunk;
  q.teams = q.chunks > 1 ? 2 : 1;
  q.stage_rows = stream_stage_rows(C, dtype, backward);
  q.ctas = chunk_parts(q.chunk * S, q.stage_rows, stream_ctas() / q.teams);
  q.slots = (long long)q.chunks * (q.ctas + q.chunk);
  q.ok = slices < (1ll << 30) && units < 2000000000ll && S * q.chunk < (1ll << 40) &&
         q.slots < (1ll << 31);
  if (q.samples) {
    q.ctas = (int)std::min<long long>(B, device_sms() * kOcc);
    q.teams = 1;
    q.slots = 0;
  }
  q.fan = 1;
  while ((long long)q.fan * q.fan < slices) ++q.fan;
  q.sets = (int)((slices + q.fan - 1) / q.fan);
  return q;
}

// Streamed maps have the plain kernels' rows too: a context may have no room for all CTAs of
// the streamed ones at once.
struct Layout {  // byte offsets
  size_t flags, part, set_part, bpart, sums, coef, total;
};
// [0, flags): counters of the plain kernels, set to 0. part: set to all ones for the
// streamed kernels.
Layout layout(const Plan& q, int B, int C, int G, bool backward) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at = (at + bytes + 255) / 256 * 256;
    return from;
  };
  Layout l{};
  take(l.flags = sizeof(uint32_t) * (2 + (2 + (size_t)q.sets) * B));
  // whole samples: a row of each for every CTA
  const size_t rows = q.samples ? q.ctas : q.units, sets = q.samples ? q.ctas : (size_t)B * q.sets;
  l.part = take(sizeof(double2) * (size_t)G * std::max<size_t>(rows, q.slots));
  l.set_part = take(sizeof(double2) * (size_t)(backward ? C : G) * sets);
  if (backward) {
    l.bpart = take(sizeof(float2) * (size_t)C * rows);
    l.sums = take(sizeof(double2) * (size_t)C *
                  (q.samples ? q.ctas : std::max(B, q.ctas * q.teams)));
    l.coef = take(sizeof(float4) * (size_t)G * (q.samples ? q.ctas : B));
  }
  l.total = at;
  return l;
}

template <typename T, int V, bool DROP>
bool launch_kernel(const NormArgs& p, bool backward, bool samples, cudaStream_t s) {
  const int grid = samples ? p.ctas : (int)std::min<unsigned>(p.tickets, device_sms() * kOcc);
  if (samples) {
    if (backward) norm_backward_samples<T, V, DROP><<<grid, kT, 0, s>>>(p);
    else norm_forward_samples<T, V, DROP><<<grid, kT, 0, s>>>(p);
  } else {
    if (backward) norm_backward_kernel<T, V, DROP><<<grid, kT, 0, s>>>(p);
    else norm_forward_kernel<T, V, DROP><<<grid, kT, 0, s>>>(p);
  }
  count_launch();
  if (!check_launch(backward ? "group norm backward" : "group norm")) return false;
  return !(samples && backward && grid > 1) || launch_params<T>(p, grid, s);
}

template <typename T, int V>
bool launch_v(const NormArgs& p, bool backward, bool samples, cudaStream_t s) {
  return p.drop.threshold != 0 ? launch_kernel<T, V, true>(p, backward, samples, s)
                               : launch_kernel<T, V, false>(p, backward, samples, s);
}

template <typename T>
bool launch_t(const NormArgs& p, int dtype, bool backward, bool samples, cudaStream_t s) {
  switch (vec_width(dtype, p.C, p.x, p.out, p.dy)) {
    case 8: return launch_v<T, (sizeof(T) == 2 ? 8 : 4)>(p, backward, samples, s);
    case 4: return launch_v<T, 4>(p, backward, samples, s);
    case 2: return launch_v<T, 2>(p, backward, samples, s);
    default: return launch_v<T, 1>(p, backward, samples, s);
  }
}

bool launch(const NormArgs& p, int dtype, bool backward, bool samples, cudaStream_t s) {
  if (dtype == LCB200_F32) return launch_t<float>(p, dtype, backward, samples, s);
  if (dtype == LCB200_F16) return launch_t<__half>(p, dtype, backward, samples, s);
  return launch_t<__nv_bfloat16>(p, dtype, backward, samples, s);
}

}  // namespace

size_t feature_norm_workspace(int B, long long S, int C, int G, int dtype, bool backward) {
  const Plan q = make_plan(B, S, C, dtype, backward);
  return q.ok ? layout(q, B, C, G, backward).total : 0;
}

bool feature_norm(const void* x, const void* dy, const void* weight, const void* bias, void* out,
                  double* stats, void* dweight, void* dbias, int B, long long S, int C, int G,
                  int dtype, bool param_f32, double eps, int act, float slope,
                  const DropArgs& drop, void* ws, size_t ws_bytes, bool backward,
                  cudaStream_t s) {
  const Plan q = make_plan(B, S, C, dtype, backward);
  if (!q.ok) {
    set_error("group norm: too many samples");
    return false;
  }
  const Layout l = layout(q, B, C, G, backward);
  if (!ws || ws_bytes < l.total || (reinterpret_cast<uintptr_t>(ws) & 15)) {
    set_error("group norm: needs a 16-byte aligned workspace of " + std::to_string(l.total) +
              " B, got " + std::to_string(ws_bytes));
    return false;
  }
  uint8_t* w = static_cast<uint8_t*>(ws);
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
  // the limit for each started GB: a CTA takes up to half a second for rows of a GB
  p.wait_ns = (uint64_t)wait_limit.load(std::memory_order_relaxed) *
              (1 + ((uint64_t)B * S * C * dtype_bytes(dtype) >> 30));
  p.slices = q.slices;
  p.slice_rows = q.slice_rows;
  p.fan = q.fan;
  p.sets = q.sets;
  p.units = q.units;
  p.lag = q.lag;
  p.teams = q.teams;
  p.ctas = q.ctas;
  p.stage_rows = q.stage_rows;
  p.chunk = q.chunk;
  p.chunks = q.chunks;
  p.tickets = out ? 2 * q.units : q.units;
  bool stream = !q.samples && streams(C, G, dtype, vec_width(dtype, C, x, out, dy));
  p.ticket = reinterpret_cast<uint32_t*>(w);
  p.done = p.ticket + 2;
  p.sets_done = p.done + (size_t)B * q.sets;
  p.ready = p.sets_done + B;
  p.part = reinterpret_cast<double2*>(w + l.part);
  p.bpart = reinterpret_cast<float2*>(w + l.bpart);
  p.set_part = reinterpret_cast<double2*>(w + l.set_part);
  p.sums = reinterpret_cast<double2*>(w + l.sums);
  p.coef = reinterpret_cast<float4*>(w + l.coef);
  p.dweight = dweight;
  p.dbias = dbias;
  p.drop = drop;
  if (stream) {
    if (cudaMemsetAsync(w + l.part, 0xff, sizeof(double2) * (size_t)G * q.slots, s) !=
        cudaSuccess)
      return check_launch("group norm: memset of the entries");
    const Streamed done = stream_norm(p, dtype, backward, s);
    if (done == Streamed::kFailed) return false;
    stream = done == Streamed::kDone;  // else the plain kernels, which need no co-residency
  }
  if (!stream) {
    if (!q.samples && cudaMemsetAsync(w, 0, l.flags, s) != cudaSuccess)
      return check_launch("group norm: memset of the counters");
    return launch(p, dtype, backward, q.samples, s);
  }
  if (!backward) return true;
  if (dtype == LCB200_F32) return launch_params<float>(p, p.ctas * p.teams, s);
  if (dtype == LCB200_F16) return launch_params<__half>(p, p.ctas * p.teams, s);
  return launch_params<__nv_bfloat16>(p, p.ctas * p.teams, s);
}

long long feature_wait_limit(long long ns) {
  return ns < 0 ? wait_limit.load() : wait_limit.exchange(std::min(ns, 1000000000000ll));
}

int feature_device_status(bool reset) {
  return read_norm_status(reset) | stream_norm_status(reset);
}

}  // namespace lcb200
