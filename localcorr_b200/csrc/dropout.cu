// Dropout with counter-based draws: y = residual + (kept ? factor * x : 0).
// The mask is a function of (seed, offset, element), so it is never stored and
// the backward pass is the same kernel on the output gradient. What drops
// becomes 0 whatever it held (a select, no product with 0).
#include "feature_common.cuh"

namespace lcb200 {
namespace {

constexpr int kThreads = 256;

// Elementwise draws. A thread owns blocks of eight elements, one Philox block
// each: the sums are exact copies of the plain formula, so only the accesses
// depend on alignment (A elements at a time, A = 1 for unaligned maps).
template <typename T, int A>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y, long long n,
               DropArgs d) {
  drop_keep_stream(d);
  const DropStream s = drop_stream(d);
  const long long blocks = (n + 7) / 8;
  for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < blocks;
       i += (long long)gridDim.x * kThreads) {
    const long long e0 = 8 * i;
    const uint32_t keep = drop_keep<8>(s, d.threshold, e0);
    if (A > 1 && e0 + 8 <= n) {
      typename Vec<T, A>::Raw xr[8 / A], rr[8 / A];
#pragma unroll
      for (int k = 0; k < 8 / A; ++k) {
        xr[k] = Vec<T, A>::load_last(x + e0 + k * A);
        if (res) rr[k] = Vec<T, A>::load_last(res + e0 + k * A);
      }
#pragma unroll
      for (int k = 0; k < 8 / A; ++k) {
        float v[A], r[A] = {};
        Vec<T, A>::unpack(xr[k], v);
        if (res) Vec<T, A>::unpack(rr[k], r);
#pragma unroll
        for (int j = 0; j < A; ++j) {
          v[j] = (keep >> (k * A + j)) & 1 ? v[j] * d.factor : 0.f;
          if (res) v[j] += r[j];
        }
        Vec<T, A>::store(y + e0 + k * A, Vec<T, A>::pack(v));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (e0 + j < n) {
          float v = (keep >> j) & 1 ? ldf(x + e0 + j) * d.factor : 0.f;
          if (res) v += ldf(res + e0 + j);
          stf(y + e0 + j, v);
        }
      }
    }
  }
}

// One draw per (sample, channel), C a multiple of V: a thread owns V channels
// of a slice of rows and draws once for all of them.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
dropout_channel_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
                       long long rows, int C, int slices, long long slice_rows, DropArgs d) {
  drop_keep_stream(d);
  const DropStream s = drop_stream(d);
  const long long b = blockIdx.x / slices;
  const long long r0 = (blockIdx.x % slices) * slice_rows;
  const long long r1 = min(rows, r0 + slice_rows);
  const int cols = C / V;
  const int nc = min(cols, kThreads), rp = kThreads / nc;
  const int row = threadIdx.x / nc;
  if (row >= rp) return;
  for (int c = threadIdx.x % nc; c < cols; c += nc) {
    const uint32_t keep = drop_keep<V>(s, d.threshold, b * C + (long long)c * V);
    const long long base = b * rows * C + (long long)c * V;
#pragma unroll 4
    for (long long r = r0 + row; r < r1; r += rp) {
      const long long e = base + r * C;
      float v[V], q[V] = {};
      Vec<T, V>::unpack(Vec<T, V>::load_last(x + e), v);
      if (res) Vec<T, V>::unpack(Vec<T, V>::load_last(res + e), q);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = (keep >> j) & 1 ? v[j] * d.factor : 0.f;
        if (res) v[j] += q[j];
      }
      Vec<T, V>::store(y + e, Vec<T, V>::pack(v));
    }
  }
}

// y = x + residual (p = 0) is the elementwise kernel with threshold 0; p = 1
// keeps nothing and its factor is 0.
template <typename T, int A>
bool launch_elements(const void* x, const void* res, void* y, long long n, const DropArgs& d,
                     cudaStream_t s) {
  const long long want = ((n + 7) / 8 + kThreads - 1) / kThreads;
  const int grid = (int)std::min<long long>(want, (long long)device_sms() * 8);
  dropout_kernel<T, A><<<grid, kThreads, 0, s>>>((const T*)x, (const T*)res, (T*)y, n, d);
  count_launch();
  return check_launch("dropout");
}

template <typename T, int V>
bool launch_channels(const void* x, const void* res, void* y, int B, long long rows, int C,
                     const DropArgs& d, cudaStream_t s) {
  const int nc = std::min(C / V, kThreads), rp = kThreads / nc;
  const long long want = std::max<long long>(1, (long long)device_sms() * 16 / B);
  long long slice = std::max<long long>((rows + want - 1) / want, 4ll * rp);
  slice = std::min(slice, rows);
  const long long slices = (rows + slice - 1) / slice;
  if (slices * B > 0x7fffffffll) {
    set_error("dropout: too many samples");
    return false;
  }
  dropout_channel_kernel<T, V><<<(unsigned)(slices * B), kThreads, 0, s>>>(
      (const T*)x, (const T*)res, (T*)y, rows, C, (int)slices, slice, d);
  count_launch();
  return check_launch("dropout (channels)");
}

template <typename T>
bool launch(const void* x, const void* res, void* y, int B, long long rows, int C, int dtype,
            const DropArgs& d, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  if (!d.channel) {
    const long long n = (long long)B * rows * C;
    return vec_width(dtype, kV, x, y, res) == kV ? launch_elements<T, kV>(x, res, y, n, d, s)
                                                 : launch_elements<T, 1>(x, res, y, n, d, s);
  }
  switch (vec_width(dtype, C, x, y, res)) {
    case 8: return launch_channels<T, (kV >= 8 ? 8 : 4)>(x, res, y, B, rows, C, d, s);
    case 4: return launch_channels<T, 4>(x, res, y, B, rows, C, d, s);
    case 2: return launch_channels<T, 2>(x, res, y, B, rows, C, d, s);
    default: return launch_channels<T, 1>(x, res, y, B, rows, C, d, s);
  }
}

}  // namespace

bool feature_dropout(const void* x, const void* residual, void* y, int B, long long rows, int C,
                     int dtype, const DropArgs& d, cudaStream_t s) {
  if (dtype == LCB200_F32) return launch<float>(x, residual, y, B, rows, C, dtype, d, s);
  if (dtype == LCB200_F16) return launch<__half>(x, residual, y, B, rows, C, dtype, d, s);
  return launch<__nv_bfloat16>(x, residual, y, B, rows, C, dtype, d, s);
}

}  // namespace lcb200
