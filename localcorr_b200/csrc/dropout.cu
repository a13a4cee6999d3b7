// Dropout with counter-based draws: y = residual + (kept ? factor * x : 0).
// The mask is a function of (seed, offset, element), so it is never stored and
// the backward pass is the same kernel on the output gradient. What drops
// becomes 0 whatever it held (a select, no product with 0).
//
// Floor: each map moved once. 8 x 135 x 240 x 256 bfloat16 (265 MB): 57 us, 4.6 TB/s,
// where whole-channel draws, which cost nothing, take 50; the difference is the draws'
// integer multiplications. With a residual (398 MB) 67 us, 6.0 TB/s.
#include "feature_common.cuh"

namespace lcb200 {
namespace {

constexpr int kThreads = 256;

// Elementwise draws. A thread owns blocks of eight elements, one Philox block each,
// kBlocks of them in flight: their loads are issued before the draws are computed.
// Accesses are A elements wide (A = 1 for unaligned maps).
template <typename T, int A, int kBlocks>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y, long long n,
               DropArgs d) {
  drop_keep_stream(d);
  const DropStream s = drop_stream(d);
  using Raw = typename Vec<T, A>::Raw;
  constexpr int kPer = 8 / A;
  const long long step = (long long)gridDim.x * kThreads;
  long long i = blockIdx.x * (long long)kThreads + threadIdx.x;
  if constexpr (A > 1) {
    const long long whole = n / 8;
    for (; i < whole; i += kBlocks * step) {
      Raw xr[kBlocks][kPer], rr[kBlocks][kPer];
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const long long e0 = 8 * min(i + k * step, whole - 1);
#pragma unroll
        for (int v = 0; v < kPer; ++v) {
          xr[k][v] = Vec<T, A>::load_last(x + e0 + v * A);
          if (res) rr[k][v] = Vec<T, A>::load_last(res + e0 + v * A);
        }
      }
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        if (i + k * step >= whole) break;
        const long long e0 = 8 * (i + k * step);
        if constexpr (sizeof(T) == 2) {
          if (!res) {  // masks of whole words
            const uint4 w = drop_block(s, i + k * step);
            float f[8];
            Vec<T, 8>::unpack(xr[k][0], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= d.factor;
            uint4 o = Vec<T, 8>::pack(f);
            o.x &= drop_mask2(w.x, d.threshold);
            o.y &= drop_mask2(w.y, d.threshold);
            o.z &= drop_mask2(w.z, d.threshold);
            o.w &= drop_mask2(w.w, d.threshold);
            Vec<T, 8>::store(y + e0, o);
            continue;
          }
        }
        const uint32_t keep = drop_keep<8>(s, d.threshold, e0);
#pragma unroll
        for (int v = 0; v < kPer; ++v) {
          float f[A], r[A] = {};
          Vec<T, A>::unpack(xr[k][v], f);
          if (res) Vec<T, A>::unpack(rr[k][v], r);
#pragma unroll
          for (int j = 0; j < A; ++j) {
            f[j] = (keep >> (v * A + j)) & 1 ? f[j] * d.factor : 0.f;
            if (res) f[j] += r[j];
          }
          Vec<T, A>::store(y + e0 + v * A, Vec<T, A>::pack(f));
        }
      }
    }
    // the last, partial block
    if (n % 8 == 0 || blockIdx.x != 0 || threadIdx.x != 0) return;
    i = whole;
  }
  for (; 8 * i < n; i += step) {
    const long long e0 = 8 * i;
    const uint32_t keep = drop_keep<8>(s, d.threshold, e0);
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
    constexpr int U = 4;  // rows in flight
    for (long long r = r0 + row; r < r1; r += U * rp) {
      typename Vec<T, V>::Raw xr[U], rr[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long e = base + min(r + u * rp, r1 - 1) * C;
        xr[u] = Vec<T, V>::load_last(x + e);
        if (res) rr[u] = Vec<T, V>::load_last(res + e);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + u * rp >= r1) break;
        float v[V], q[V] = {};
        Vec<T, V>::unpack(xr[u], v);
        if (res) Vec<T, V>::unpack(rr[u], q);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[j] = (keep >> j) & 1 ? v[j] * d.factor : 0.f;
          if (res) v[j] += q[j];
        }
        Vec<T, V>::store(y + base + (r + u * rp) * C, Vec<T, V>::pack(v));
      }
    }
  }
}

// y = x + residual (p = 0) is the elementwise kernel with threshold 0; p = 1
// keeps nothing and its factor is 0.
template <typename T, int A>
bool launch_elements(const void* x, const void* res, void* y, long long n, const DropArgs& d,
                     cudaStream_t s) {
  // Blocks in flight a thread and CTAs a multiprocessor, measured on 8 x 135 x 240 x 256
  // without and with a residual: 16-bit maps 57 and 67 us with one block and 6 CTAs, 60
  // and 68 with 2 and 8; float32 105 and 145 with one and 6, 91 and 122 with 2 and 8.
  constexpr int kBlocks = sizeof(T) == 2 ? 1 : 2, kCtas = sizeof(T) == 2 ? 6 : 8;
  const long long want = ((n + 7) / 8 + kBlocks * kThreads - 1) / (kBlocks * kThreads);
  const int grid = (int)std::min<long long>(want, (long long)device_sms() * kCtas);
  dropout_kernel<T, A, kBlocks><<<grid, kThreads, 0, s>>>((const T*)x, (const T*)res, (T*)y, n, d);
  count_launch();
  return check_launch("dropout");
}

template <typename T, int V>
bool launch_channels(const void* x, const void* res, void* y, int B, long long rows, int C,
                     const DropArgs& d, cudaStream_t s) {
  const int nc = std::min(C / V, kThreads), rp = kThreads / nc;
  // 16 slices a multiprocessor: 98.6 us for the training step of 64 x 64 x 128 x 128
  // float16, 98.5 with 8, 102.5 with 32
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
