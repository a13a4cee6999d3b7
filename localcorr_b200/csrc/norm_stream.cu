// Group norm for rows of aligned 16-byte vectors, no wider than a CTA's threads.
//
// The floor is HBM traffic, so the aim is loads that never pause and few instructions a
// vector (a pass of 16-bit maps has about 90 issue slots per 16 bytes read and written
// before it falls behind HBM). The rows of a chunk of samples are divided evenly over
// a team of CTAs; a CTA makes its first pass (sums) over its rows of a chunk and then
// its second pass (outputs), in part out of L2. A producer warp copies the rows into a
// ring of stages with bulk copies, running on across passes; the other warps do the
// arithmetic, two float32 operations an instruction.
//
// Between the passes the team's CTAs wait for each other's sums, about 5 us. So there are
// two teams, one CTA of each on every multiprocessor, that take the chunks in turn: while
// one waits, the other streams, and reads of one overlap writes of the other. That is so
// from the second chunk of a team on; with one each (maps up to 150 MB forward, 167 MB
// backward) the teams start together and overlap only as far as they drift apart.
//
// Measured: 8 x 135 x 240 x 256 float16 moves 3.7 TB/s forward (HBM 51 % busy, issue slots
// 48 %) and 3.3 backward (62 and 51 %; 442 MB are read where 265 are needed): neither HBM nor
// issue is full, the warps mostly wait for their stages (long scoreboard) in between.
//
// The sums travel through 16-byte entries that are written whole and start out as all
// ones: a reader polls the entry itself, so no fence, counter or flag stands between a
// sum and its reader, and every CTA adds up the entries of its samples itself, two
// round trips after the last of them is written. Waiting needs every CTA resident: the
// kernels are launched cooperatively. (Dynamic units finished by the last arriver of
// an atomic counter made the statistics wait 13 to 18 us: a round trip takes 2 to 3 us
// while the copies saturate HBM.)
#include "norm_common.cuh"
#include "tc_ptx.cuh"

namespace lcb200 {
namespace {

constexpr int kS = 256;          // arithmetic threads
constexpr int kBlock = kS + 32;  // and the producer warp
constexpr int kPerSm = 2;        // CTAs of a multiprocessor
// Vectors of a thread per stage and map: 16 KB stages. A stage costs a CTA about 570
// cycles from barrier to barrier however small it is: reading 531 MB with one CTA a
// multiprocessor takes 264 us in 4 KB stages, 141 in 8, 90 in 16 and 86 in 32 KB.
template <int NM> constexpr int kVecs = 4 / NM;

__device__ __forceinline__ void stream_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kS) : "memory");
}

// A barrier that tells every thread whether all of them came with true.
__device__ __forceinline__ bool all_threads(bool ok) {
  int r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 q, %1, 0;\n\tbar.red.and.pred p, 1, %2, q;\n\t"
      "selp.s32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((int)ok), "n"(kS)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint64_t bits(float2 v) { return *reinterpret_cast<uint64_t*>(&v); }
__device__ __forceinline__ float2 pair(uint64_t v) { return *reinterpret_cast<float2*>(&v); }
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return pair(r);
}

// One 16-byte vector as float pairs, and back.
template <typename T> struct Vec2;
template <> struct Vec2<float> {
  static __device__ __forceinline__ void unpack(uint4 r, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    f[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  }
  static __device__ __forceinline__ uint32_t relu(uint32_t v) {  // NaN stays
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(__uint_as_float(v)));
    return __float_as_uint(r);
  }
};
template <> struct Vec2<__half> {
  static __device__ __forceinline__ void unpack(uint4 r, float2 (&f)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<__half2*>(&w[i]) = __float22half2_rn(f[i]);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint32_t relu(uint32_t v) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0u));
    return r;
  }
};
template <> struct Vec2<__nv_bfloat16> {
  static __device__ __forceinline__ void unpack(uint4 r, float2 (&f)[4]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<__nv_bfloat162*>(&w[i]) = __float22bfloat162_rn(f[i]);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint32_t relu(uint32_t v) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0u));
    return r;
  }
};

__device__ __forceinline__ void keep2(float2& v, uint32_t m) {
  v.x = m & 1 ? v.x : 0.f;
  v.y = m & 2 ? v.y : 0.f;
}

// ---- entries --------------------------------------------------------------------------
// 16 bytes as two words; all ones: not written yet.
struct Entry {
  unsigned long long lo, hi;
  __device__ __forceinline__ bool ready() const { return (lo & hi) != ~0ull; }
};
__device__ __forceinline__ Entry entry_of(double2 v) {
  Entry e{(unsigned long long)__double_as_longlong(v.x),
          (unsigned long long)__double_as_longlong(v.y)};
  if (!e.ready()) e.lo = 0x7ff8000000000000ull;  // a NaN like any other
  return e;
}
__device__ __forceinline__ double2 pair_of(const Entry& e) {
  return make_double2(__longlong_as_double((long long)e.lo), __longlong_as_double((long long)e.hi));
}
__device__ __forceinline__ Entry get(const void* p) {
  Entry e;
  asm volatile(
      "{\n\t.reg .b128 v;\n\tld.relaxed.gpu.global.b128 v, [%2];\n\tmov.b128 {%0, %1}, v;\n\t}"
      : "=l"(e.lo), "=l"(e.hi)
      : "l"(p)
      : "memory");
  return e;
}
__device__ __forceinline__ void put(void* p, const Entry& e) {
  asm volatile(
      "{\n\t.reg .b128 v;\n\tmov.b128 v, {%1, %2};\n\tst.relaxed.gpu.global.b128 [%0], v;\n\t}" ::"l"(p),
      "l"(e.lo), "l"(e.hi)
      : "memory");
}

// ---- the ring ------------------------------------------------------------------------
struct StageInfo {
  long long off;  // element offset of the stage's first row
  int b;          // sample
  int seg;        // slot of the segment's sums
  int rows;       // of the stage, and flags
};
enum : int {
  kRowsMask = 0xffff,
  kSecond = 1 << 16,
  kLast = 2 << 16,
  kEnd = 4 << 16,
  kTop = 8 << 16,  // starts the sample
};

template <int NM, int STAGES>
struct RingShared {
  uint4 data[STAGES][NM][kVecs<NM> * kS];
  uint64_t full[STAGES], empty[STAGES];
  StageInfo info[STAGES];
  int b, seg;   // of a first pass's unit, for its end
  int started;  // whether the CTA's row of parameter sums holds something
  int abort;
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1], %2, [%3], %4;" ::"r"(tc::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(tc::smem_u32(bar)), "l"(policy)
      : "memory");
}

template <int NM, int STAGES>
__device__ void ring_init(RingShared<NM, STAGES>& r) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(&r.full[i], 1);
      tc::mbar_init(&r.empty[i], kS / 32);
    }
    r.abort = r.started = 0;
    tc::fence_mbar_init();
  }
  __syncthreads();
}

// ---- the division of the work -----------------------------------------------------------
// Chunk k: samples [k m, k m + count), its rows cut into `parts` runs of equal length
// (to a row), run q starting at row q rows / parts and belonging to CTA q of team
// k % teams. A run is cut again where a sample ends: segments, the s-th sample's in run q
// with slot q + s of the chunk's.
struct Chunk {
  int first, count, parts;
  long long rows;
  long long slots;  // of the chunks before
  __device__ __forceinline__ Chunk(const NormArgs& p, int k) {
    first = k * p.chunk;
    count = min(p.chunk, p.B - first);
    rows = count * p.S;
    parts = chunk_parts(rows, p.stage_rows, p.ctas);
    slots = (long long)k * (p.ctas + p.chunk);
  }
  __device__ __forceinline__ long long start(int q) const {
    return (long long)((unsigned long long)q * (unsigned long long)rows / (unsigned)parts);
  }
  // the run that holds row r
  __device__ __forceinline__ int run_of(long long r) const {
    return (int)(((unsigned long long)(r + 1) * (unsigned)parts - 1) / (unsigned long long)rows);
  }
};

// seg(sample of the chunk, first row, end row within the sample) for rows
// [start, end) of a chunk, backwards if `back`.
template <typename F>
__device__ __forceinline__ void each_segment(const NormArgs& p, long long start, long long end,
                                             bool back, F seg) {
  const int s0 = (int)(start / p.S), s1 = (int)((end - 1) / p.S);
  for (int i = 0; i <= s1 - s0; ++i) {
    const int s = back ? s1 - i : s0 + i;
    seg(s, max(start - s * p.S, 0ll), min(end - s * p.S, p.S));
  }
}

// One thread. A segment is a run of whole rows, so its bytes are contiguous.
template <typename T, int NM, int STAGES>
__device__ void produce(const NormArgs& p, RingShared<NM, STAGES>& r, const T* m0, const T* m1) {
  uint64_t stay, go;  // a first pass's rows are read again, a second pass's are not
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(stay));
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(go));
  uint32_t n = 0;  // stages issued
  bool good = true;
  auto claim = [&]() {
    return tc::mbar_wait(&r.empty[n % STAGES], ((n / STAGES) & 1) ^ 1, &r.abort, p.wait_ns);
  };
  auto run = [&](const Chunk& c, int q, bool second) {
    if (q >= c.parts) return;
    const uint64_t policy = second ? go : stay;
    // a second pass runs backwards: what was read last is what L2 still holds
    each_segment(p, c.start(q), c.start(q + 1), second, [&](int s, long long r0, long long r1) {
      const int seg = (int)(c.slots + q + s);
      const int stages = (int)((r1 - r0 + p.stage_rows - 1) / p.stage_rows);
      const int flags = (second ? kSecond : 0) | (r0 == 0 ? kTop : 0);
      for (int t = 0; t < stages && good && (good = claim()); ++t) {
        const int at = n % STAGES;
        const long long row = r0 + (long long)(second ? stages - 1 - t : t) * p.stage_rows;
        const int rows = (int)min((long long)p.stage_rows, r1 - row);
        const uint32_t bytes = (uint32_t)(rows * p.C * sizeof(T));
        const long long off = ((long long)(c.first + s) * p.S + row) * p.C;
        r.info[at] =
            StageInfo{off, c.first + s, seg, rows | flags | (t == stages - 1 ? kLast : 0)};
        tc::mbar_arrive_expect_tx(&r.full[at], bytes * NM);
        bulk_copy(r.data[at][0], m0 + off, bytes, &r.full[at], policy);
        if (NM > 1) bulk_copy(r.data[at][NM - 1], m1 + off, bytes, &r.full[at], policy);
        ++n;
      }
    });
  };
  const int q = blockIdx.x % p.ctas;
  for (int k = blockIdx.x / p.ctas; k < p.chunks && good; k += p.teams) {
    const Chunk c(p, k);
    run(c, q, false);
    if (p.out) run(c, q, true);
  }
  if (good && claim()) {
    r.info[n % STAGES] = StageInfo{0, 0, 0, kEnd};
    tc::mbar_arrive(&r.full[n % STAGES]);
  } else {  // gave up: no copy may be in flight when the CTA ends
    for (uint32_t k = n > STAGES ? n - STAGES : 0; k < n; ++k)
      tc::mbar_wait_drain(&r.full[k % STAGES], (k / STAGES) & 1);
  }
}

// The arithmetic warps' side. A wait that runs out (here or in poll) ends the kernel, but
// threads see it at different times: one may give up on a copy that lands for another. So a
// thread that gave up has a stage of no rows, its warp learns of it at the stage's end, and
// the CTA at the next barrier that the unit has for all threads anyway (all_threads). No
// thread leaves by itself, and none waits at a barrier for one that left. (The vote costs 1 %
// of a backward pass: 8 x 540 x 960 x 64 float16 431 us with it and 427 without.)
template <int NM, int STAGES>
struct Consumer {
  const NormArgs& p;
  RingShared<NM, STAGES>& r;
  uint32_t n = 0;
  long long off = 0;  // of the stage, see StageInfo
  int now = 0;

  __device__ __forceinline__ Consumer(const NormArgs& args, RingShared<NM, STAGES>& ring)
      : p(args), r(ring) {}
  // Waits for the next stage. now is 0 in a thread whose wait ran out.
  __device__ __forceinline__ void open() {
    if (tc::mbar_wait(&r.full[n % STAGES], (n / STAGES) & 1, &r.abort, p.wait_ns)) {
      off = r.info[n % STAGES].off;
      now = r.info[n % STAGES].rows;
    } else {
      atomicExch(&norm_status, 1);
      now = 0;
    }
  }
  __device__ __forceinline__ int rows() const { return now & kRowsMask; }
  __device__ __forceinline__ int sample() const { return r.info[n % STAGES].b; }
  __device__ __forceinline__ int segment() const { return r.info[n % STAGES].seg; }
  __device__ __forceinline__ const uint4* map(int m) const { return r.data[n % STAGES][m]; }
  // The warp is done with the stage; false when it did not open for all of its threads: the
  // stage then stays the producer's, whose copy may still be under way.
  __device__ __forceinline__ bool close() {
    const bool opened = __all_sync(0xffffffffu, now);
    if (opened && threadIdx.x % 32 == 0) tc::mbar_arrive(&r.empty[n % STAGES]);
    ++n;
    return opened;
  }
};

// Calls unit() for each unit's first stage until the producer's end, or until a wait ran out
// for any thread. The barrier between units also keeps one unit's shared values until every
// thread has read them.
template <typename C, typename F>
__device__ __forceinline__ void each_unit(C& in, F unit) {
  bool ok = true;
  for (;;) {
    if (ok) in.open();
    if (!all_threads(ok && in.now)) break;
    if (in.now & kEnd) return;
    ok = unit();
  }
  in.r.abort = 1;  // the producer stops too
}

// Calls row(i-th vector of the stage's map 0, row) for this thread's rows of a stage.
template <int VECS, typename F>
__device__ __forceinline__ void stage_rows(const Place& at, int rows, F row) {
  const int active = at.nc * at.rp;
  if (rows == at.rp * VECS) {
    if (at.on) {
#pragma unroll
      for (int i = 0; i < VECS; ++i) row(threadIdx.x + i * active, at.row + i * at.rp);
    }
  } else if (at.on) {
#pragma unroll 1
    for (int i = 0; at.row + i * at.rp < rows; ++i)
      row(threadIdx.x + i * active, at.row + i * at.rp);
  }
}

// ---- the sums of a sample ------------------------------------------------------------
// Polls an entry that was not ready. Gives up when the limit is reached, or when another
// thread of the CTA did, with NaN: the kernel ends at its next wait, and what it still
// writes shows.
__device__ __forceinline__ Entry poll(const void* p, uint64_t limit, volatile int* abort) {
  const uint64_t t0 = tc::globaltimer();
  for (uint32_t i = 1;; ++i) {
    const Entry e = get(p);
    if (e.ready()) return e;
    if ((i % 32 == 0 || limit == 0) && (*abort || tc::globaltimer() - t0 >= limit)) {
      *abort = 1;
      atomicExch(&norm_status, 1);
      return Entry{0x7ff8000000000000ull, 0x7ff8000000000000ull};
    }
    __nanosleep(200);
  }
}

// done(g, sum of the sample's entries of group g) by one thread per group, in an order
// that only the sizes decide; `red` is room for kS double2. The entries of a sample lie
// together, [runs, G]: a warp reads lines of them whole (one group's entries a warp at
// a time, 32 lines a load, kept L2 busy for longer than the map's own rows).
template <typename F>
__device__ __forceinline__ void sample_sums(const NormArgs& p, int b, volatile int* abort,
                                            double2* red, F done) {
  constexpr int kFlight = 5, kWarps = kS / 32;
  const Chunk c(p, b / p.chunk);
  const int s = b - c.first;
  const int first = c.run_of(s * p.S), runs = c.run_of((s + 1) * p.S - 1) - first + 1;
  const double2* part = p.part + (c.slots + first + s) * p.G;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // One warp waits for the runs, by their first group, so that the others do not flood L2
  // with polls meanwhile: a 66 MB chunk took 64 us with all polling, 41 with one warp, and
  // 35 once the entries were read in whole lines.
  if (warp == 0) {
#pragma unroll 1
    for (int at = lane; at < runs; at += kFlight * 32) {
      Entry e[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u)  // past the end: the last one again
        e[u] = get(part + (long long)min(at + u * 32, runs - 1) * p.G);
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        if (!e[u].ready())
          poll(part + (long long)min(at + u * 32, runs - 1) * p.G, p.wait_ns, abort);
    }
  }
  stream_sync();
  // a block of `wide` groups by `team` warps, 32 / wide runs a warp at a time
  const int wide = p.G >= 32 ? 32 : p.G <= 1 ? 1 : 2 * pow2_below(p.G - 1);
  const int blocks = (p.G + wide - 1) / wide, rows = 32 / wide;
  const int team = blocks >= kWarps ? 1 : kWarps / (blocks <= 1 ? 1 : 2 * pow2_below(blocks - 1));
  for (int k0 = 0; k0 < blocks; k0 += kWarps / team) {
    const int k = k0 + warp / team, g = k * wide + lane % wide;
    double2 v = make_double2(0.0, 0.0);
    if (g < p.G) {
      const double2* src = part + g;
      const int step = team * rows;
#pragma unroll 1
      for (int at = warp % team * rows + lane / wide; at < runs; at += kFlight * step) {
        Entry e[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u)
          e[u] = get(src + (long long)min(at + u * step, runs - 1) * p.G);
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          if (at + u * step < runs) {
            if (!e[u].ready())
              e[u] = poll(src + (long long)(at + u * step) * p.G, p.wait_ns, abort);
            const double2 d = pair_of(e[u]);
            v.x += d.x;
            v.y += d.y;
          }
        }
      }
    }
    for (int o = wide; o < 32; o *= 2) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (team > 1) {
      red[threadIdx.x] = v;
      stream_sync();
      if (warp % team == 0)
        for (int w = 1; w < team; ++w) {
          v.x += red[threadIdx.x + 32 * w].x;
          v.y += red[threadIdx.x + 32 * w].y;
        }
      stream_sync();
    }
    if (g < p.G && warp % team == 0 && lane < wide) done(g, v);
  }
}

// ---- forward -------------------------------------------------------------------------
// WHOLE: a vector lies in one group, so its V channels share their sums.
template <typename T, bool WHOLE>
struct ForwardShared {
  static constexpr int kV = 16 / sizeof(T), kStages = WHOLE ? 5 : 4;
  RingShared<1, kStages> ring;
  double2 sums[kS * (WHOLE ? 1 : kV)];  // (sum d, sum d^2) of each thread
  double2 stats[1];                     // [G] of the second pass's sample
};

template <typename T, bool WHOLE, typename C>
__device__ __forceinline__ bool stats_unit(const NormArgs& p, const Place& at, C& in,
                                           ForwardShared<T, WHOLE>& sh) {
  constexpr int V = 16 / sizeof(T), N = WHOLE ? 1 : V, A = WHOLE ? 2 : V;
  double s[A], q[A], k[N];
#pragma unroll
  for (int v = 0; v < A; ++v) s[v] = q[v] = 0.0;
#pragma unroll
  for (int v = 0; v < N; ++v) k[v] = group_shift<T>(p, in.sample(), (at.col * V + v) / p.Cg);
  const int seg = in.segment();
  bool ok = true;
  for (;;) {
    const uint4* data = in.map(0);
    stage_rows<kVecs<1>>(at, in.rows(), [&](int i, int) {
      float2 f[V / 2];
      Vec2<T>::unpack(data[i], f);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const double d = (double)(v & 1 ? f[v / 2].y : f[v / 2].x) - k[v % N];
        s[v % A] += d;
        q[v % A] = fma(d, d, q[v % A]);
      }
    });
    const bool last = in.now & kLast;
    ok = in.close();
    if (last || !ok) break;
    in.open();
  }
  if (WHOLE) {
    sh.sums[threadIdx.x] = make_double2(s[0] + s[1], q[0] + q[1]);
  } else {
#pragma unroll
    for (int v = 0; v < N; ++v) sh.sums[threadIdx.x * N + v] = make_double2(s[v], q[v]);
  }
  if (!all_threads(ok)) return false;
  // one group by `width` lanes
  const int ne = at.nc * N, gw = p.Cg * N / V;
  const int width = min(32, max(1, pow2_below(min(at.rp * gw, kS / min(p.G, kS)))));
  const int lane = threadIdx.x % width;
  for (int g0 = 0; g0 < p.G; g0 += kS / width) {
    const int g = g0 + threadIdx.x / width;
    double2 t = make_double2(0.0, 0.0);
    if (g < p.G) {
      for (int i = lane; i < at.rp * gw; i += width) {
        const int r = i / gw;
        const double2 e = sh.sums[r * ne + g * gw + (i - r * gw)];
        t.x += e.x;
        t.y += e.y;
      }
    }
    t = lanes_sum(t, width);
    if (g < p.G && lane == 0) put(p.part + (long long)seg * p.G + g, entry_of(t));
  }
  return true;
}

template <typename T, bool WHOLE, bool DROP, typename C>
__device__ __forceinline__ bool apply_unit(const NormArgs& p, const Place& at, C& in,
                                           double2* red, double2* stats) {
  constexpr int V = 16 / sizeof(T), N = WHOLE ? 1 : V / 2;
  const int b = in.sample(), c0 = at.col * V;
  const bool top = in.now & kTop;
  // K by the last warps, on its way while the first one polls: a barrier follows
  for (int g = kS - 1 - threadIdx.x; g < p.G; g += kS) stats[g].x = group_shift<T>(p, b, g);
  sample_sums(p, b, &in.r.abort, red, [&](int g, double2 t) {
    stats[g] = finish_stats(p, t, stats[g].x);
    if (top) p.stats[(long long)b * p.G + g] = stats[g];
  });
  stream_sync();
  // z = (x - mu) a + c, mu rounded to float32, c = beta - (what the rounding left) a. a is
  // rounded twice, 1/std and the product: 2^-24 of (x - mu) a more than the plain kernels'
  // float64 product leaves, which costs 1 % of the pass here.
  float2 mu[N], a[V / 2], c[V / 2];  // mu: minus mu
  float rstd = 0.f, left = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (!WHOLE || v == 0) {
      const double2 st = stats[(c0 + v) / p.Cg];
      const float m = -(float)st.x;
      left = (float)(st.x + (double)m);
      rstd = (float)st.y;
      if (WHOLE) mu[0] = twice(m);
      else (v & 1 ? mu[v / 2 % N].y : mu[v / 2 % N].x) = m;
    }
    const float av = param_f<T>(p.weight, p.param_f32, c0 + v, 1.f) * rstd;
    const float cv = fmaf(-left, av, param_f<T>(p.bias, p.param_f32, c0 + v, 0.f));
    (v & 1 ? a[v / 2].y : a[v / 2].x) = av;
    (v & 1 ? c[v / 2].y : c[v / 2].x) = cv;
  }
  DropStream ds;
  uint32_t keep = ~0u;
  if (DROP) {
    ds = drop_stream(p.drop);
    if (p.drop.channel) keep = drop_keep<V>(ds, p.drop.threshold, (long long)b * p.C + c0);
  }
  T* dst = reinterpret_cast<T*>(p.out);
  const int act = p.act;
  for (;;) {
    const uint4* data = in.map(0);
    const long long first = in.off + c0;
    stage_rows<kVecs<1>>(at, in.rows(), [&](int i, int row) {
      float2 x[V / 2];
      Vec2<T>::unpack(data[i], x);
      const long long e = first + (long long)row * p.C;
      if (DROP && !p.drop.channel) keep = drop_keep<V>(ds, p.drop.threshold, e);
#pragma unroll
      for (int v = 0; v < V / 2; ++v) x[v] = fma2(add2(x[v], mu[WHOLE ? 0 : v % N]), a[v], c[v]);
      if (act == LCB200_ACT_SILU) {
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          x[v].x *= sigmoid(x[v].x);
          x[v].y *= sigmoid(x[v].y);
        }
      } else if (act == LCB200_ACT_LEAKY_RELU) {
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          x[v].x *= x[v].x < 0.f ? p.slope : 1.f;
          x[v].y *= x[v].y < 0.f ? p.slope : 1.f;
        }
      }
      if (DROP) {
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          x[v] = mul2(x[v], twice(p.drop.factor));
          keep2(x[v], keep >> (2 * v));
        }
      }
      uint4 r = Vec2<T>::pack(x);
      if (act == LCB200_ACT_RELU) {  // commutes with the factor and the rounding
        r.x = Vec2<T>::relu(r.x);
        r.y = Vec2<T>::relu(r.y);
        r.z = Vec2<T>::relu(r.z);
        r.w = Vec2<T>::relu(r.w);
      }
      __stcs(reinterpret_cast<uint4*>(dst + e), r);
    });
    const bool last = in.now & kLast;
    if (!in.close()) return false;
    if (last) return true;
    in.open();
  }
}

template <typename T, bool WHOLE, bool DROP>
__global__ void __launch_bounds__(kBlock, kPerSm) norm_forward_stream(NormArgs p) {
  extern __shared__ __align__(128) unsigned char smem[];
  auto& sh = *reinterpret_cast<ForwardShared<T, WHOLE>*>(smem);
  drop_keep_stream(p.drop);
  ring_init(sh.ring);
  if (threadIdx.x >= kS) {
    if (threadIdx.x == kS) {
      const T* x = reinterpret_cast<const T*>(p.x);
      produce<T, 1>(p, sh.ring, x, x);
    }
    return;
  }
  const Place at(p.C / (16 / (int)sizeof(T)), 0, kS);
  Consumer<1, ForwardShared<T, WHOLE>::kStages> in(p, sh.ring);
  each_unit(in, [&]() {
    return in.now & kSecond ? apply_unit<T, WHOLE, DROP>(p, at, in, sh.sums, sh.stats)
                                  : stats_unit<T, WHOLE>(p, at, in, sh);
  });
}

// ---- backward ------------------------------------------------------------------------
// RECT: a rectifier, whose side needs z to more than float32 (see norm_common.cuh).
template <typename T, bool WHOLE>
struct BackwardShared {
  static constexpr int kV = 16 / sizeof(T), kStages = 5;
  RingShared<2, kStages> ring;
  alignas(16) float2 sums[kS * kV];  // sum dz, sum dz (x - mu); also kS double2
  float4 coef[1];  // [G] of the second pass's sample; as double2 a first pass's group sums
};

// What z of a thread's channels takes, and dz in place of the output gradient.
template <typename T, bool WHOLE, bool RECT, bool DROP>
struct Slope {
  static constexpr int V = 16 / sizeof(T), N = WHOLE ? 1 : V / 2, H = RECT ? V / 2 : 1;
  float2 mu[N], a[V / 2], b[V / 2], al[H], bl[H];  // mu: minus mu
  DropStream ds;
  uint32_t keep = ~0u;

  __device__ __forceinline__ Slope(const NormArgs& p, int sample, int c0) {
    float m = 0.f, ml = 0.f, rh = 0.f, rl = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (!WHOLE || v == 0) {
        const double2 st = __ldg(p.stats + (long long)sample * p.G + (c0 + v) / p.Cg);
        m = (float)st.x;
        ml = (float)(st.x - (double)m);
        rh = (float)st.y;
        rl = (float)(st.y - (double)rh);
        if (WHOLE) mu[0] = twice(-m);
        else (v & 1 ? mu[v / 2 % N].y : mu[v / 2 % N].x) = -m;
      }
      const float w = param_f<T>(p.weight, p.param_f32, c0 + v, 1.f);
      const float beta = param_f<T>(p.bias, p.param_f32, c0 + v, 0.f);
      const float av = __fmul_rn(w, rh);  // no contraction: the pairs below need this rounding
      float bv;
      if (RECT) {
        // a and b = beta - mu a as float pairs: products split by fma, sums by two-sum
        const float alv = fmaf(w, rh, -av) + w * rl;
        const float ph = __fmul_rn(-m, av), pl = -fmaf(m, av, ph);
        bv = beta + ph;
        const float z = bv - beta;
        const float blv = ((beta - (bv - z)) + (ph - z)) + (pl - fmaf(m, alv, ml * av));
        (v & 1 ? al[v / 2 % H].y : al[v / 2 % H].x) = alv;
        (v & 1 ? bl[v / 2 % H].y : bl[v / 2 % H].x) = blv;
      } else {
        bv = fmaf(-ml, av, beta);  // for x - mu
      }
      (v & 1 ? a[v / 2].y : a[v / 2].x) = av;
      (v & 1 ? b[v / 2].y : b[v / 2].x) = bv;
    }
    if (DROP) {
      ds = drop_stream(p.drop);
      if (p.drop.channel) keep = drop_keep<V>(ds, p.drop.threshold, (long long)sample * p.C + c0);
    }
  }

  // g: output gradient -> dz; d: x -> x - mu
  __device__ __forceinline__ void apply(const NormArgs& p, long long e, float2 (&d)[V / 2],
                                        float2 (&g)[V / 2]) {
    if (DROP) {
      if (!p.drop.channel) keep = drop_keep<V>(ds, p.drop.threshold, e);
#pragma unroll
      for (int v = 0; v < V / 2; ++v) {
        g[v] = mul2(g[v], twice(p.drop.factor));
        keep2(g[v], keep >> (2 * v));
      }
    }
    if (RECT) {
      auto side = [&](auto closed) {  // closed(v): what stays of g[v] below the corner
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          const float2 z = add2(fma2(d[v], a[v], b[v]), fma2(d[v], al[v % H], bl[v % H]));
          const float2 low = closed(v);
          g[v].x = z.x > 0.f ? g[v].x : low.x;
          g[v].y = z.y > 0.f ? g[v].y : low.y;
          d[v] = add2(d[v], mu[WHOLE ? 0 : v % N]);
        }
      };
      if (p.act == LCB200_ACT_RELU) side([&](int) { return twice(0.f); });
      else side([&](int v) { return mul2(g[v], twice(p.slope)); });
    } else {
#pragma unroll
      for (int v = 0; v < V / 2; ++v) d[v] = add2(d[v], mu[WHOLE ? 0 : v % N]);
      if (p.act == LCB200_ACT_SILU) {
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          const float2 z = fma2(d[v], a[v], b[v]);
          const float sx = sigmoid(z.x), sy = sigmoid(z.y);
          g[v].x *= sx * fmaf(z.x, 1.f - sx, 1.f);
          g[v].y *= sy * fmaf(z.y, 1.f - sy, 1.f);
        }
      }
    }
  }
};

// Adds up what the CTA's threads have in `sums` [rp, C], in float64: the parameters' gradients
// into the CTA's own row of p.sums, the groups' sums into acc [G] (from 0 if `first`), and
// with `last` the latter into the segment's entries. Every arithmetic thread calls it; false
// when one of them comes without its sums.
template <typename T, typename R>
__device__ __forceinline__ bool reduce_sums(const NormArgs& p, const Place& at, R& ring,
                                            float2* sums, double2* acc, bool ok, bool first,
                                            bool last) {
  if (!all_threads(ok)) return false;
  const int b = ring.b, seg = ring.seg;
  const bool started = ring.started;
  // X = r sum dz (x - mu), the sums centred on mu rounded to float32
  const double2* stats = p.stats + (long long)b * p.G;
  const bool params = p.dweight || p.dbias;
  for (int c = threadIdx.x; c < p.C; c += kS) {
    double2 v = as_double2(sums[c]);
    for (int r = 1; r < at.rp; ++r) {
      const float2 e = sums[r * p.C + c];
      v.x += e.x;
      v.y += e.y;
    }
    if (at.rp > 1) {  // the channel's sum in place, as float pairs
      const float2 high = make_float2((float)v.x, (float)v.y);
      sums[c] = high;
      sums[p.C + c] = make_float2((float)(v.x - high.x), (float)(v.y - high.y));
    }
    if (params) {
      const double2 st = __ldg(stats + c / p.Cg);
      double2* row = p.sums + (long long)blockIdx.x * p.C + c;
      double2 t = started ? *row : make_double2(0.0, 0.0);
      t.x += v.x;
      t.y += st.y * (v.y - (st.x - (double)(float)st.x) * v.x);
      *row = t;
    }
  }
  stream_sync();
  if (threadIdx.x == 0) ring.started = 1;
  if (p.out) {
    const int width = min(32, max(1, pow2_below(min(p.Cg, kS / min(p.G, kS)))));
    const int lane = threadIdx.x % width;
    for (int g0 = 0; g0 < p.G; g0 += kS / width) {
      const int g = g0 + threadIdx.x / width;
      double2 t = make_double2(0.0, 0.0);
      if (g < p.G) {
        for (int i = lane; i < p.Cg; i += width) {
          const int c = g * p.Cg + i;
          const double w = param_f<T>(p.weight, p.param_f32, c, 1.f);
          double2 e = as_double2(sums[c]);
          if (at.rp > 1) {
            const float2 low = sums[p.C + c];
            e.x += low.x;
            e.y += low.y;
          }
          t.x += w * e.x;
          t.y += w * e.y;
        }
      }
      t = lanes_sum(t, width);
      if (g < p.G && lane == 0) {
        if (!first) {
          t.x += acc[g].x;
          t.y += acc[g].y;
        }
        if (last) put(p.part + (long long)seg * p.G + g, entry_of(t));
        else acc[g] = t;
      }
    }
    if (!last) stream_sync();  // the sums have been read
  }
  return true;
}

template <typename T, bool WHOLE, bool RECT, bool DROP, typename C>
__device__ __forceinline__ bool grad_sums_unit(const NormArgs& p, const Place& at, C& in,
                                               float2* sums, double2* acc) {
  constexpr int V = 16 / sizeof(T), kFold = kRun / kVecs<2>;  // stages of a run
  const int c0 = at.col * V;
  Slope<T, WHOLE, RECT, DROP> f(p, in.sample(), c0);
  if (threadIdx.x == 0) {
    in.r.b = in.sample();
    in.r.seg = in.segment();
  }
  float2 sa[V / 2], sx[V / 2];
#pragma unroll
  for (int v = 0; v < V / 2; ++v) sa[v] = sx[v] = twice(0.f);
  float4* mine = reinterpret_cast<float4*>(sums) + threadIdx.x * (V / 2);
  constexpr int kAll = kFold * kRuns;  // stages until float64 takes over
  for (int n = 0;;) {  // stages so far
    const uint4 *xd = in.map(0), *gd = in.map(1);
    const long long from = in.off + c0;
    stage_rows<kVecs<2>>(at, in.rows(), [&](int i, int row) {
      float2 d[V / 2], g[V / 2];
      Vec2<T>::unpack(xd[i], d);
      Vec2<T>::unpack(gd[i], g);
      f.apply(p, from + (long long)row * p.C, d, g);
#pragma unroll
      for (int v = 0; v < V / 2; ++v) {
        sa[v] = add2(sa[v], g[v]);
        sx[v] = fma2(g[v], d[v], sx[v]);
      }
    });
    const bool last = in.now & kLast;
    const bool ok = in.close();
    const int at_run = n % kAll;  // of the stage in its runs
    ++n;
    if (last || !ok || n % kFold == 0) {
      // a run of rows ends: its sums go to the thread's own in shared memory
#pragma unroll
      for (int v = 0; v < V / 2; ++v) {
        float4 t = make_float4(sa[v].x, sx[v].x, sa[v].y, sx[v].y);
        if (at_run >= kFold) {
          const float4 e = mine[v];
          t = make_float4(t.x + e.x, t.y + e.y, t.z + e.z, t.w + e.w);
        }
        mine[v] = t;
        sa[v] = sx[v] = twice(0.f);
      }
      if (last || !ok || n % kAll == 0) {
        if (!reduce_sums<T>(p, at, in.r, sums, acc, ok, n <= kAll, last)) return false;
        if (last) return true;
      }
    }
    in.open();
  }
}

template <typename T, bool WHOLE, bool RECT, bool DROP, typename C>
__device__ __forceinline__ bool grad_input_unit(const NormArgs& p, const Place& at, C& in,
                                                double2* red, float4* coef) {
  constexpr int V = 16 / sizeof(T), N = WHOLE ? 1 : V / 2;
  const int b = in.sample(), c0 = at.col * V;
  sample_sums(p, b, &in.r.abort, red, [&](int g, double2 t) {
    coef[g] = finish_coef(p, __ldg(p.stats + (long long)b * p.G + g), t);
  });
  stream_sync();
  Slope<T, WHOLE, RECT, DROP> f(p, b, c0);
  float2 k2[N], k3[N];
#pragma unroll
  for (int v = 0; v < 2 * N; ++v) {
    const float4 k = coef[(c0 + (WHOLE ? 0 : v)) / p.Cg];
    (v & 1 ? k2[v / 2].y : k2[v / 2].x) = k.y;
    (v & 1 ? k3[v / 2].y : k3[v / 2].x) = k.z;
  }
  T* dst = reinterpret_cast<T*>(p.out);
  for (;;) {
    const uint4 *xd = in.map(0), *gd = in.map(1);
    const long long first = in.off + c0;
    stage_rows<kVecs<2>>(at, in.rows(), [&](int i, int row) {
      float2 d[V / 2], g[V / 2];
      Vec2<T>::unpack(xd[i], d);
      Vec2<T>::unpack(gd[i], g);
      const long long e = first + (long long)row * p.C;
      f.apply(p, e, d, g);
#pragma unroll
      for (int v = 0; v < V / 2; ++v)
        g[v] = fma2(f.a[v], g[v], fma2(k2[WHOLE ? 0 : v % N], d[v], k3[WHOLE ? 0 : v % N]));
      __stcs(reinterpret_cast<uint4*>(dst + e), Vec2<T>::pack(g));
    });
    const bool last = in.now & kLast;
    if (!in.close()) return false;
    if (last) return true;
    in.open();
  }
}

template <typename T, bool WHOLE, bool RECT, bool DROP>
__global__ void __launch_bounds__(kBlock, kPerSm) norm_backward_stream(NormArgs p) {
  extern __shared__ __align__(128) unsigned char smem[];
  auto& sh = *reinterpret_cast<BackwardShared<T, WHOLE>*>(smem);
  ring_init(sh.ring);
  if (threadIdx.x >= kS) {
    if (threadIdx.x == kS)
      produce<T, 2>(p, sh.ring, reinterpret_cast<const T*>(p.x),
                    reinterpret_cast<const T*>(p.dy));
    return;
  }
  const Place at(p.C / (16 / (int)sizeof(T)), 0, kS);
  Consumer<2, BackwardShared<T, WHOLE>::kStages> in(p, sh.ring);
  each_unit(in, [&]() {
    return in.now & kSecond
               ? grad_input_unit<T, WHOLE, RECT, DROP>(p, at, in,
                                                       reinterpret_cast<double2*>(sh.sums), sh.coef)
               : grad_sums_unit<T, WHOLE, RECT, DROP>(p, at, in, sh.sums,
                                                      reinterpret_cast<double2*>(sh.coef));
  });
  if (!sh.ring.started && (p.dweight || p.dbias))
    for (int c = threadIdx.x; c < p.C; c += kS)
      p.sums[(long long)blockIdx.x * p.C + c] = make_double2(0.0, 0.0);
}

// ---- host ----------------------------------------------------------------------------
template <typename K>
Streamed launch_kernel(K kernel, size_t smem, const NormArgs& p, const char* what,
                       cudaStream_t s) {
  // the static shared memory counts towards the 48 KB that need no opt-in
  if (!ensure_smem_attr((const void*)kernel, smem + 1024)) return Streamed::kFailed;
  NormArgs args = p;
  void* argv[] = {&args};
  const cudaError_t e = cudaLaunchCooperativeKernel((const void*)kernel, dim3(p.ctas * p.teams),
                                                    dim3(kBlock), argv, smem, s);
  if (e == cudaErrorCooperativeLaunchTooLarge) {
    cudaGetLastError();
    return Streamed::kNoRoom;
  }
  if (e == cudaSuccess) count_launch();
  return check_launch(what) ? Streamed::kDone : Streamed::kFailed;
}

template <typename T, bool WHOLE, bool DROP>
Streamed launch_w(const NormArgs& p, bool backward, cudaStream_t s) {
  if (!backward)
    return launch_kernel(norm_forward_stream<T, WHOLE, DROP>,
                         sizeof(ForwardShared<T, WHOLE>) + sizeof(double2) * p.G, p, "group norm",
                         s);
  const size_t smem = sizeof(BackwardShared<T, WHOLE>) + sizeof(float4) * p.G;
  const bool rect = p.act == LCB200_ACT_RELU || p.act == LCB200_ACT_LEAKY_RELU;
  return rect ? launch_kernel(norm_backward_stream<T, WHOLE, true, DROP>, smem, p,
                              "group norm backward", s)
              : launch_kernel(norm_backward_stream<T, WHOLE, false, DROP>, smem, p,
                              "group norm backward", s);
}

template <typename T>
Streamed launch_t(const NormArgs& p, bool backward, cudaStream_t s) {
  const bool drop = p.drop.threshold != 0;
  if (p.Cg % (16 / sizeof(T)) == 0)
    return drop ? launch_w<T, true, true>(p, backward, s) : launch_w<T, true, false>(p, backward, s);
  return drop ? launch_w<T, false, true>(p, backward, s) : launch_w<T, false, false>(p, backward, s);
}

}  // namespace

Streamed stream_norm(const NormArgs& p, int dtype, bool backward, cudaStream_t s) {
  if (dtype == LCB200_F32) return launch_t<float>(p, backward, s);
  if (dtype == LCB200_F16) return launch_t<__half>(p, backward, s);
  return launch_t<__nv_bfloat16>(p, backward, s);
}

int stream_ctas() { return device_sms() * kPerSm; }

int stream_stage_rows(int C, int dtype, bool backward) {
  const int cols = std::max(1, C / (16 / (int)dtype_bytes(dtype)));
  return (backward ? kVecs<2> : kVecs<1>) * std::max(1, kS / cols);
}

int stream_norm_status(bool reset) { return read_norm_status(reset); }

}  // namespace lcb200
