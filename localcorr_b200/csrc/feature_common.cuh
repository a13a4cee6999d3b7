// Shared parts of the feature-map operators (dropout.cu, group_norm.cu):
// element types, vector accesses and the counter-based dropout draws.
#pragma once

#include <cuda_bf16.h>

#include "lc_common.cuh"

namespace lcb200 {

template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
};

inline size_t dtype_bytes(int dtype) { return dtype == LCB200_F32 ? 4 : 2; }

// ---- V consecutive elements moved as one access -----------------------------
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

template <typename T, int V>
struct Vec {
  using Raw = typename RawOf<sizeof(T) * V>::type;
  union U {
    Raw raw;
    T e[V];
    __device__ __forceinline__ U() {}
  };
  static __device__ __forceinline__ Raw load(const T* p) {
    return __ldg(reinterpret_cast<const Raw*>(p));
  }
  // read once: leaves L2 first
  static __device__ __forceinline__ Raw load_last(const T* p) {
    return __ldcs(reinterpret_cast<const Raw*>(p));
  }
  static __device__ __forceinline__ void store(T* p, Raw r) {
    __stcs(reinterpret_cast<Raw*>(p), r);
  }
  static __device__ __forceinline__ void unpack(Raw r, float (&f)[V]) {
    U u;
    u.raw = r;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Elem<T>::to_f(u.e[i]);
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[V]) {
    U u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.e[i] = Elem<T>::from_f(f[i]);
    return u.raw;
  }
};

// ---- dropout draws -----------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011). Block i of the stream (seed, offset) has the counter
// (i, offset), 64 bits each, and the key seed; it holds eight 16-bit draws, the
// low half of a word first. Draw e drops when it is below the threshold
// round(65536 p). 16 bits a draw: with 32 the ten rounds of integer
// multiplications for every four elements bound a 16-bit map's pass (130 us
// against 94 us for 256 MB in and out, a plain copy 88 us).
struct DropArgs {
  uint32_t threshold;      // 0: nothing drops; 65536: everything does
  float factor;            // 65536 / (65536 - threshold), 0 when everything drops
  int channel;             // one draw per (sample, channel) instead of per element
  long long seed, offset;  // used when rng is null
  const long long* rng;    // device, {seed, offset}
  long long* rng_used;     // device, receives {seed, offset}; may be null
};

// The key schedule is kept (20 registers): the integer pipes are what a 16-bit map's
// draws use most of.
struct DropStream {
  uint32_t k0[10], k1[10], c2, c3;
};

__device__ __forceinline__ DropStream drop_stream(const DropArgs& d) {
  const unsigned long long seed = d.rng ? __ldg(d.rng) : d.seed;
  const unsigned long long off = d.rng ? __ldg(d.rng + 1) : d.offset;
  DropStream s;
#pragma unroll
  for (uint32_t r = 0; r < 10; ++r) {
    s.k0[r] = (uint32_t)seed + r * 0x9E3779B9u;
    s.k1[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
  }
  s.c2 = (uint32_t)off;
  s.c3 = (uint32_t)(off >> 32);
  return s;
}

// Leaves the stream that a forward call used for its backward pass: the caller
// may advance its own copy in between.
__device__ __forceinline__ void drop_keep_stream(const DropArgs& d) {
  if (d.rng_used && blockIdx.x == 0 && threadIdx.x == 0) {
    d.rng_used[0] = d.rng ? d.rng[0] : d.seed;
    d.rng_used[1] = d.rng ? d.rng[1] : d.offset;
  }
}

__device__ __forceinline__ uint4 drop_block(const DropStream& s, unsigned long long i) {
  uint32_t c0 = (uint32_t)i, c1 = (uint32_t)(i >> 32), c2 = s.c2, c3 = s.c3;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)0xD2511F53u * c0;
    const unsigned long long p1 = (unsigned long long)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ s.k0[r];
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ s.k1[r];
    c3 = (uint32_t)p0;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t drop_piece(const uint4& w, int e) {
  const uint32_t word = e < 4 ? (e < 2 ? w.x : w.y) : (e < 6 ? w.z : w.w);
  return (e & 1) ? word >> 16 : word & 0xffffu;
}

// All ones in the halves of word w whose draws stay: the sign of draw - threshold,
// spread over a half.
__device__ __forceinline__ uint32_t drop_mask2(uint32_t w, uint32_t threshold) {
  return ~__byte_perm((w & 0xffffu) - threshold, (w >> 16) - threshold, 0xffbb);
}

// Bit v: element e0 + v stays. V divides 8 and e0 is a multiple of V.
template <int V>
__device__ __forceinline__ uint32_t drop_keep(const DropStream& s, uint32_t threshold,
                                              long long e0) {
  static_assert(V == 8 || V == 4 || V == 2 || V == 1, "a vector lies in one block");
  const uint4 w = drop_block(s, (unsigned long long)e0 >> 3);
  uint32_t m = 0;
  if (V == 8) {
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m |= (uint32_t)((q[i] & 0xffffu) >= threshold) << (2 * i);
      m |= (uint32_t)((q[i] >> 16) >= threshold) << (2 * i + 1);
    }
  } else {
    const int at = (int)(e0 & 7);
#pragma unroll
    for (int v = 0; v < V; ++v) m |= (uint32_t)(drop_piece(w, at + v) >= threshold) << v;
  }
  return m;
}

// ---- host side ------------------------------------------------------------------
// Largest V in {16 bytes' worth, ..., 1} such that rows of C elements at these
// addresses can be moved V elements at a time.
inline int vec_width(int dtype, int C, const void* a, const void* b, const void* c = nullptr,
                     const void* d = nullptr) {
  const size_t es = dtype_bytes(dtype);
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
                        reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d);
  int v = (int)(16 / es);
  while (v > 1 && (C % v != 0 || all % (v * es) != 0)) v >>= 1;
  return v;
}

int device_sms();  // multiprocessors of the current device

}  // namespace lcb200
