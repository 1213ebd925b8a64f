// Log probabilities of given tokens with the entropy, the token's rank and the top alternatives
// (dspark_token_logprobs).
//
// With x the row's logits, c = 1 / T, m = max x, l = sum exp(c (x - m)), s = sum exp(c (x - m)) c (x - m):
//   logprob(t) = c (x_t - m) - ln l,   entropy = ln l - s / l,   rank = #{v before t in the order below}.
// One pass: a thread keeps m, l and s of the values it has seen (fp32), raising m for 64 bytes at a time. The
// order of tokens is by logit, then the lower token first.
//
// Alternatives without a second pass: a thread's m is the largest value of its strips of the row, so the top-th
// largest of several groups' maxima bounds the block's top-th largest value from below, and only strips whose largest
// value reaches it hold any of the block's alternatives: little more than as many strips as alternatives are read again.
//
// A row is a cluster of 1 to 8 blocks, each with a slice of its 16-byte vectors; the first block joins them.
// Bound: HBM and the exponentials' unit for many rows (2049 of 151,936 in bf16 124 us, 0.77 of the measured rate; 272 in
// fp32 with 20 alternatives 42.4, 0.59, for the search of alternatives, which no other block's pass covers), latency for few
// (one row 9). A ring of bulk copies in shared memory in place of plain loads: 132 beside 132, one row 14.
#include <algorithm>
#include <cfloat>

#include "elem.cuh"
#include "host_common.h"

namespace dspark {
namespace score {

constexpr int THREADS = 256;
constexpr int U = 4;          // vectors of a chunk a thread
constexpr int CHUNK = U * THREADS;
constexpr int MAX_TOP = 32;
constexpr int MAX_CLUSTER = 8;
constexpr int CAND = 512;     // values at or above the bound that a block sorts at once
constexpr int PARTS = 4;      // parts of the block's chunks whose largest values are kept by thread

// A logit at or below kLow (NaN and -inf among them) is a masked token's, one above kHigh counts as kHigh.
constexpr float kLow = -0x1p28f, kHigh = 0x1p28f;

template <typename T>
struct Vec;

// n = VE values of a 16-byte vector, masked ones as kLow, and the largest of them (not yet held to kHigh).
template <>
struct Vec<bf16> {
  static constexpr int VE = 8;
  static constexpr float MAXV = kHigh;
  static __device__ __forceinline__ float split(uint4 w, float* x) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t y;  // (the number of the two where one is NaN)
      asm("max.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(in[i]), "r"(0xCD80CD80u));
      x[2 * i] = bf16_lo(y);
      x[2 * i + 1] = bf16_hi(y);
    }
    return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
  }
  static __device__ __forceinline__ float one(bf16 v) { return fmaxf(__bfloat162float(v), kLow); }
};

template <>
struct Vec<__half> {
  static constexpr int VE = 8;
  static constexpr float MAXV = 65504.f;
  static __device__ __forceinline__ float split(uint4 w, float* x) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t low = 0x7BFF7BFFu;  // the smallest
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t y;
      asm("max.f16x2 %0, %1, %2;" : "=r"(y) : "r"(in[i]), "r"(0xFBFFFBFFu));
      asm("min.f16x2 %0, %0, %1;" : "+r"(low) : "r"(y));
      const float2 f = Elem<__half>::unpack(y);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    if ((low & 0xffffu) == 0xFBFFu || (low >> 16) == 0xFBFFu) {  // masked values: below all that an fp16 can be
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] <= -65504.f ? kLow : x[i];
    }
    return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
  }
  static __device__ __forceinline__ float one(__half v) {
    const float f = fmaxf(__half2float(v), -65504.f);
    return f <= -65504.f ? kLow : f;
  }
};

template <>
struct Vec<float> {
  static constexpr int VE = 4;
  static constexpr float MAXV = kHigh;
  static __device__ __forceinline__ float split(uint4 w, float* x) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaxf(__uint_as_float(in[i]), kLow);
    return fmaxf(max3(x[0], x[1], x[2]), x[3]);
  }
  static __device__ __forceinline__ float one(float v) { return fmaxf(v, kLow); }
};

// What a part of a row adds up to; sums are in units of log2, relative to the reference of m. Without a temperature
// that is m c as it is rounded, y = x c - (m c) one operation (x c is exact in it) and no value is lost to the rounding of the
// reference (|m c| < 2^29: it is off by less than 2^6). With one it is m itself, y = (x - m) c.
struct Sums {
  float m, l, s;
};

template <bool TEMP>
__device__ __forceinline__ void raise(Sums& a, float m, float c) {
  const float d = TEMP ? (a.m - m) * c : __fmul_rn(a.m, c) - __fmul_rn(m, c);  // at most 0
  a.m = m;
  if (d < -200.f) {  // (also the start, where m was kLow)
    a.l = 0.f;
    a.s = 0.f;
  } else {
    const float f = ex2(d);
    a.s = f * (a.s + d * a.l);
    a.l *= f;
  }
}

template <bool TEMP>
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  const float m = fmaxf(a.m, b.m);
  raise<TEMP>(a, m, c);
  raise<TEMP>(b, m, c);
  return Sums{m, a.l + b.l, a.s + b.s};
}

// Larger first, then the lower token; a zero of either sign is the same value.
__device__ __forceinline__ uint64_t key_of(float x, int v) {
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | uint32_t(~v);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = uint32_t(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct Shared {
  float last[THREADS];  // the threads' largest values
  Sums warp[THREADS / 32];
  int rank[THREADS / 32];
  uint64_t top[MAX_TOP];  // the block's alternatives in order, 0 behind the last
  Sums sum;
  int before;
  float bound;
  int n_strip, n_cand;
  uint64_t best[THREADS / 32];
  union {
    float maxima[PARTS][THREADS];  // of the strips
    uint64_t cand[CAND];
  };
  uint16_t strip[PARTS * THREADS];
};

__device__ __forceinline__ uint64_t remote_u64(const void* p, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

template <typename T>
struct Row {
  const T* p;     // the row
  int V, head;    // values, those before the first 16-byte vector
  int nvec;       // vectors
  int v0, v1;     // the block's
  int chunks, part;  // its chunks, those of a part
  bool first, last;
};

// Sorts the block's candidates sh.cand[0 .. n) by counting into sh.top.
__device__ __forceinline__ void place_top(Shared& sh, const uint64_t* cand, int n, int top, uint64_t* out) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const uint64_t k = cand[i];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += cand[j] > k;
    if (before < top && k) out[before] = k;
  }
}

// The block's alternatives into sh.top. m: the largest value that the thread has seen in its vectors, all parts' strips.
template <typename T>
__device__ __noinline__ void find_top(Shared& sh, const Row<T>& r, float m, int top) {
  constexpr int VE = Vec<T>::VE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) {
    // The top-th largest of 32 values, each the largest of 8 threads' (of 64 and 4 threads' for more than 16 alternatives):
    // a value's place is the number of those before it, equal ones by lane.
    float y[THREADS / 32];
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) y[i] = sh.last[32 * i + lane];
    float g0 = fmaxf(max3(y[0], y[1], y[2]), y[3]), g1 = fmaxf(max3(y[4], y[5], y[6]), y[7]);
    const bool wide = top > 16;
    if (!wide) g0 = fmaxf(g0, g1);
    int at0 = 0, at1 = 0;
#pragma unroll
    for (int o = 1; o < 32; ++o) {
      const float x = __shfl_xor_sync(0xffffffffu, g0, o);
      at0 += x > g0 || (x == g0 && (lane ^ o) < lane);
    }
    if (wide) {
      at0 += g1 > g0;
      at1 = g0 >= g1;
#pragma unroll
      for (int o = 1; o < 32; ++o) {
        const float x0 = __shfl_xor_sync(0xffffffffu, g0, o), x1 = __shfl_xor_sync(0xffffffffu, g1, o);
        at0 += x1 > g0;
        at1 += (x0 >= g1) + (x1 > g1 || (x1 == g1 && (lane ^ o) < lane));
      }
    }
    if (at0 == top - 1) sh.bound = g0;
    if (wide && at1 == top - 1) sh.bound = g1;
  }
  __syncthreads();
  const float bound = sh.bound;
  if (m >= bound && m > kLow) {
    for (int p = 0; p < PARTS; ++p) {
      const float x = sh.maxima[p][tid];
      if (x >= bound && x > kLow) sh.strip[atomicAdd(&sh.n_strip, 1)] = uint16_t(p * THREADS + tid);
    }
  }
  __syncthreads();  // (the maxima have been read: the candidates take their place)
  auto offer = [&](float x, int v) {
    if (x > kLow && x >= bound) {
      const int at = atomicAdd(&sh.n_cand, 1);
      if (at < CAND) sh.cand[at] = key_of(x, v);
    }
  };
  const int per = r.part * U, n = sh.n_strip * per;
  const uint4* vec = reinterpret_cast<const uint4*>(r.p + r.head);
  for (int j0 = tid; j0 < n; j0 += 4 * THREADS) {
    uint4 w[4];
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * THREADS, g = j / per, k = j - g * per, s = j < n ? sh.strip[g] : 0;
      at[i] = r.v0 + (s / THREADS * r.part * U + k) * THREADS + s % THREADS;
      if (j >= n || at[i] >= r.v1) at[i] = -1;
      if (at[i] >= 0) w[i] = ldcg_v4(vec + at[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[VE];
      if (at[i] < 0 || Vec<T>::split(w[i], x) < bound) continue;
#pragma unroll
      for (int e = 0; e < VE; ++e) offer(fminf(x[e], Vec<T>::MAXV), r.head + at[i] * VE + e);
    }
  }
  if (r.first && tid < r.head) offer(fminf(Vec<T>::one(r.p[tid]), Vec<T>::MAXV), tid);
  const int t0 = r.head + r.nvec * VE;
  if (r.last && tid < r.V - t0) offer(fminf(Vec<T>::one(r.p[t0 + tid]), Vec<T>::MAXV), t0 + tid);
  __syncthreads();
  if (sh.n_cand <= CAND) {
    place_top(sh, sh.cand, sh.n_cand, top, sh.top);
    __syncthreads();
    return;
  }
  // Too many equal or nearly equal values for the list: the alternatives one after the other, each by a pass
  // over the block's slice.
  uint64_t prev = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    auto see = [&](float x, int v) {
      const uint64_t key = key_of(x, v);
      if (x > kLow && key < prev && key > best) best = key;
    };
    for (int v = r.v0 + tid; v < r.v1; v += THREADS) {
      float x[VE];
      Vec<T>::split(ldcg_v4(vec + v), x);
#pragma unroll
      for (int e = 0; e < VE; ++e) see(fminf(x[e], Vec<T>::MAXV), r.head + v * VE + e);
    }
    if (r.first && tid < r.head) see(fminf(Vec<T>::one(r.p[tid]), Vec<T>::MAXV), tid);
    if (r.last && tid < r.V - t0) see(fminf(Vec<T>::one(r.p[t0 + tid]), Vec<T>::MAXV), t0 + tid);
    for (int o = 16; o; o >>= 1) best = max(best, uint64_t(__shfl_xor_sync(0xffffffffu, best, o)));
    if (lane == 0) sh.best[warp] = best;
    __syncthreads();
    for (int i = 0; i < THREADS / 32; ++i) best = max(best, sh.best[i]);
    if (tid == 0) sh.top[k] = best;
    __syncthreads();
    if (best == 0) break;
    prev = best;
  }
}

// What a thread has taken in, and the token that it looks out for: its logit, the next larger value, log2(e) / T.
struct Taken {
  Sums z;
  float xt, after, c;
  int tok, before;
};

// N vectors of a thread (masked values kLow); vm[u] is the largest of x[u], tk + u * step the token of x[u][0]. Returns the
// largest of all.
template <typename T, bool TEMP, int N>
__device__ __forceinline__ float take(Taken& t, float (&x)[N][Vec<T>::VE], float (&vm)[N], int tk, int step) {
  constexpr int VE = Vec<T>::VE;
  float bm = vm[0];
#pragma unroll
  for (int u = 1; u < N; ++u) bm = fmaxf(bm, vm[u]);
  if (bm > Vec<T>::MAXV) {  // rare: values above the largest that counts
    bm = Vec<T>::MAXV;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      vm[u] = fminf(vm[u], Vec<T>::MAXV);
#pragma unroll
      for (int e = 0; e < VE; ++e) x[u][e] = fminf(x[u][e], Vec<T>::MAXV);
    }
  }
  if (bm >= t.xt) {  // some may come before the token: as large ones before it, and larger ones
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int t0 = tk + u * step;
      if (vm[u] < t.xt) continue;
      if (t0 <= t.tok && t.tok < t0 + VE) {
#pragma unroll
        for (int e = 0; e < VE; ++e) t.before += x[u][e] >= (t0 + e < t.tok ? t.xt : t.after);
      } else {
        const float at = t0 < t.tok ? t.xt : t.after;
#pragma unroll
        for (int e = 0; e < VE; ++e) t.before += x[u][e] >= at;
      }
    }
  }
  if (bm > t.z.m) raise<TEMP>(t.z, bm, t.c);
  const float ref = TEMP ? -t.z.m : -__fmul_rn(t.z.m, t.c);
  const f32x2 m2 = pack2(ref, ref), c2 = pack2(t.c, t.c);
  f32x2 l2 = pack2(0.f, 0.f), s2 = pack2(0.f, 0.f);
#pragma unroll
  for (int u = 0; u < N; ++u) {
#pragma unroll
    for (int e = 0; e < VE; e += 2) {
      const f32x2 v = pack2(x[u][e], x[u][e + 1]), y = TEMP ? mul2(add2(v, m2), c2) : fma2(v, c2, m2);
      float y0, y1;
      unpack2(y, y0, y1);
      const f32x2 p = pack2(ex2(y0), ex2(y1));
      l2 = add2(l2, p);
      s2 = fma2(p, y, s2);
    }
  }
  float a0, a1;
  unpack2(l2, a0, a1);
  t.z.l += a0 + a1;
  unpack2(s2, a0, a1);
  t.z.s += a0 + a1;
  return bm;
}

template <typename T, bool TOP, bool TEMP, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) score_kernel(const dspark_score_args a, const int cluster) {
  constexpr int VE = Vec<T>::VE;
  __shared__ Shared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = int(blockIdx.x) / cluster, part = int(blockIdx.x) - row * cluster;
  pdl_launch_dependents();
  pdl_wait();
  const int tok = a.tokens[row];
  if (tok < 0 || tok >= a.V) {  // (every block of the cluster)
    if (part == 0) {
      if (tid == 0) {
        a.logprob[row] = 0.f;
        a.entropy[row] = 0.f;
        a.rank[row] = -1;
      }
      for (int k = tid; k < a.top; k += THREADS) {
        a.top_ids[int64_t(row) * a.top + k] = -1;
        a.top_logprob[int64_t(row) * a.top + k] = -INFINITY;
      }
    }
    return;
  }
  Row<T> r;
  r.p = static_cast<const T*>(a.logits) + int64_t(row) * a.ld;
  r.V = a.V;
  r.head = min(int((16 - (reinterpret_cast<uintptr_t>(r.p) & 15)) & 15) / int(sizeof(T)), a.V);
  r.nvec = (a.V - r.head) / VE;
  r.v0 = int(int64_t(r.nvec) * part / cluster);
  r.v1 = int(int64_t(r.nvec) * (part + 1) / cluster);
  r.chunks = (r.v1 - r.v0 + CHUNK - 1) / CHUNK;
  r.part = max(1, (r.chunks + PARTS - 1) / PARTS);
  r.first = part == 0;
  r.last = part == cluster - 1;
  float T1 = 1.f;
  bool greedy = false;
  if (TEMP) {
    T1 = a.temperature[row];
    greedy = !(T1 > 1e-6f);
    T1 = greedy ? 1.f : fminf(T1, 1e6f);
  }
  const float c = 1.4426950408889634f / T1;
  const float xt = fminf(Vec<T>::one(r.p[tok]), Vec<T>::MAXV);
  Sums z{kLow, 0.f, 0.f};

  Taken t{z, xt, xt == 0.f ? __int_as_float(1) : xt >= Vec<T>::MAXV ? INFINITY : __int_as_float(__float_as_int(xt) + (xt > 0.f ? 1 : -1)),
          c, tok, 0};
  const uint4* vec = reinterpret_cast<const uint4*>(r.p + r.head) + r.v0 + tid;
  float part_max = kLow;
  int left = r.part;
  for (int k = 0; k < r.chunks; ++k) {
    const int tk = r.head + (r.v0 + k * CHUNK + tid) * VE, n = r.v1 - r.v0 - k * CHUNK;
    uint4 w[U];
    float x[U][VE], vm[U];
    if (n >= CHUNK) {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = ldcg_v4(vec + k * CHUNK + u * THREADS);
    } else {  // the last chunk: missing vectors are masked ones
      const uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u;  // -inf
#pragma unroll
      for (int u = 0; u < U; ++u)
        w[u] = u * THREADS + tid < n ? ldcg_v4(vec + k * CHUNK + u * THREADS) : make_uint4(none, none, none, none);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) vm[u] = Vec<T>::split(w[u], x[u]);
    part_max = fmaxf(part_max, take<T, TEMP, U>(t, x, vm, tk, THREADS * VE));
    if (TOP && (--left == 0 || k + 1 == r.chunks)) {
      sh.maxima[k / r.part][tid] = part_max;
      part_max = kLow;
      left = r.part;
    }
  }
  if (TOP) {  // parts without chunks
    for (int p = (r.chunks + r.part - 1) / r.part; p < PARTS; ++p) sh.maxima[p][tid] = kLow;
  }
  const float strip = t.z.m;
  const int t0 = r.head + r.nvec * VE;
  if ((r.first && tid < r.head) || (r.last && tid >= 32 && tid - 32 < a.V - t0)) {  // the ragged ends
    const int at = tid < 32 ? tid : t0 + tid - 32;
    float x[1][VE], vm[1];
#pragma unroll
    for (int e = 1; e < VE; ++e) x[0][e] = kLow;
    x[0][0] = vm[0] = Vec<T>::one(r.p[at]);
    // (the others are nobody's: they add nothing, and a token among them is not this thread's)
    take<T, TEMP, 1>(t, x, vm, at, 0);
  }
  z = t.z;
  int before = t.before;
  // (masked values were counted while nothing else had been seen; raise() has dropped them where something was)
  for (int o = 16; o; o >>= 1) {
    const Sums y{__shfl_xor_sync(0xffffffffu, z.m, o), __shfl_xor_sync(0xffffffffu, z.l, o),
                 __shfl_xor_sync(0xffffffffu, z.s, o)};
    z = join<TEMP>(z, y, c);
  }
  before = int(__reduce_add_sync(0xffffffffu, unsigned(before)));
  if (lane == 0) {
    sh.warp[warp] = z;
    sh.rank[warp] = before;
  }
  if (TOP) {
    sh.last[tid] = strip;
    if (tid < MAX_TOP) sh.top[tid] = 0;
    if (tid == 0) sh.n_strip = sh.n_cand = 0;
  }
  __syncthreads();
  if (warp == 1) {  // (warp 0 has the alternatives' bound to find)
    Sums y = sh.warp[lane & 7];
#pragma unroll
    for (int o = 1; o < THREADS / 32; o <<= 1) {
      const Sums q{__shfl_xor_sync(0xffffffffu, y.m, o), __shfl_xor_sync(0xffffffffu, y.l, o),
                   __shfl_xor_sync(0xffffffffu, y.s, o)};
      y = join<TEMP>(y, q, c);
    }
    const int n = __reduce_add_sync(0xffffffffu, lane < THREADS / 32 ? unsigned(sh.rank[lane]) : 0u);
    if (lane == 0) {
      sh.sum = y;
      sh.before = n;
    }
  }
  if (TOP) find_top<T>(sh, r, strip, a.top);
  if (cluster > 1) {
    cluster_sync_all();
    if (part == 0) {
      if (TOP) {
        const int n = cluster * a.top;  // at most CAND / 2
        if (tid < n) {
          const int q = tid / a.top;
          sh.cand[tid] = remote_u64(&sh.top[tid - q * a.top], q);
        }
        if (tid < a.top) sh.cand[CAND / 2 + tid] = 0;  // (nothing is left behind the last)
      }
      if (warp == THREADS / 32 - 1) {  // a lane a block
        const uint32_t q = lane < cluster ? lane : 0, at = mapa_shared(smem_u32(&sh.sum), q);
        Sums y{ld_dsmem_f32(at), ld_dsmem_f32(at + 4), ld_dsmem_f32(at + 8)};
        int n = __float_as_int(ld_dsmem_f32(mapa_shared(smem_u32(&sh.before), q)));
        for (int o = 1; o < cluster; o <<= 1) {
          const Sums z1{__shfl_xor_sync(0xffffffffu, y.m, o), __shfl_xor_sync(0xffffffffu, y.l, o),
                        __shfl_xor_sync(0xffffffffu, y.s, o)};
          y = join<TEMP>(y, z1, c);
          n += __shfl_xor_sync(0xffffffffu, n, o);
        }
        if (lane == 0) {
          sh.sum = y;
          sh.before = n;
        }
      }
      if (TOP) {
        __syncthreads();
        place_top(sh, sh.cand, cluster * a.top, a.top, sh.cand + CAND / 2);
      }
    }
  }
  __syncthreads();
  if (part == 0) {
    const Sums y = sh.sum;
    const bool any = y.m > kLow;
    const float ln = any ? logf(y.l) : 0.f;
    auto lp = [&](float v) {
      return (TEMP ? (v - y.m) / T1 : fmaf(v, c, -__fmul_rn(y.m, c)) * 0.6931471805599453f) - ln;
    };
    if (tid == 0) {
      const bool live = any && xt > kLow;
      a.logprob[row] = !live ? -INFINITY : greedy ? (sh.before == 0 ? 0.f : -INFINITY) : lp(xt);
      a.entropy[row] = !any || greedy ? 0.f : fmaxf(ln - y.s / y.l * 0.6931471805599453f, 0.f);
      a.rank[row] = live ? sh.before : -1;
    }
    if (TOP) {
      const uint64_t* list = cluster > 1 ? sh.cand + CAND / 2 : sh.top;
      for (int k = tid; k < a.top; k += THREADS) {
        const uint64_t key = list[k];
        const float v = value_of(key);
        a.top_ids[int64_t(row) * a.top + k] = key ? int32_t(~uint32_t(key)) : -1;
        a.top_logprob[int64_t(row) * a.top + k] =
            !key ? -INFINITY : greedy ? (k == 0 ? 0.f : -INFINITY) : lp(v);
      }
    }
  }
  if (cluster > 1) cluster_sync_all();  // the first block has read the others' shared memory
}

template <typename T, int PER_SM>
static cudaError_t launch_as(const dspark_score_args& a, int cluster, cudaStream_t s) {
  auto kernel = a.top ? (a.temperature ? score_kernel<T, true, true, PER_SM> : score_kernel<T, true, false, PER_SM>)
                      : (a.temperature ? score_kernel<T, false, true, PER_SM> : score_kernel<T, false, false, PER_SM>);
  return launch_ex(kernel, dim3(unsigned(a.R) * cluster), dim3(THREADS), 0, s, cluster, true, a, cluster);
}

template <typename T>
static cudaError_t launch(const dspark_score_args& a, cudaStream_t s) {
  // Blocks a row: as many as there is room for at once, for two of them some more, in slices of 4 KB or more. 151,936 values
  // in bf16 without / with 5 alternatives, us by blocks a row (1, 2, 4, 8): 74 rows 26 16 14 12 / 32 21 20 18, 110 rows 33 23 17
  // 18 / 38 29 24 30, 200 rows 42 29 24 28 / 48 35 35 45, 296 rows 46 30 30 39 / 52 36 42 61, 500 rows 50 43 45 61 / 57 55 62
  // 95, 740 rows 52 55 63 86 / 59 69 88 136.
  const int64_t sms = sm_count(current_device());
  int cluster = 1;
  while (cluster < MAX_CLUSTER && int64_t(a.R) * cluster * 4 <= (cluster == 1 ? 14 : cluster == 2 ? 11 : 10) * sms &&
         int64_t(a.V) * int(sizeof(T)) >= int64_t(cluster) * 2 * 4096)
    cluster *= 2;
  // Four or five blocks an SM (64 or 48 registers a thread) by which takes fewer rounds of blocks; clusters of more than two are
  // not packed that closely. Us, 5 / 4: 272 rows in bf16 29.3 / 25.5, in fp32 with 20 alternatives 46.7 / 42.4, 1480 in bf16
  // 94.6 / 98.7, 2049 with 5 alternatives 140 / 149.
  const int64_t n = int64_t(a.R) * cluster, rounds4 = (n + 4 * sms - 1) / (4 * sms), rounds5 = (n + 5 * sms - 1) / (5 * sms);
  const bool four = cluster <= 2 && 4 * rounds4 <= 5 * rounds5;
  return four ? launch_as<T, 4>(a, cluster, s) : launch_as<T, 5>(a, cluster, s);
}

}  // namespace score
}  // namespace dspark

using namespace dspark;

extern "C" int dspark_token_logprobs(const dspark_score_args* p, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "token_logprobs: null argument");
  const dspark_score_args& a = *p;
  if (a.R < 0 || a.V <= 0 || a.top < 0)
    return fail(DSPARK_ERR_ARG, "token_logprobs: bad shape (%d rows, %d tokens, %d alternatives)", a.R, a.V, a.top);
  if (a.dtype != DSPARK_DTYPE_BF16 && a.dtype != DSPARK_DTYPE_F16 && a.dtype != DSPARK_DTYPE_F32)
    return fail(DSPARK_ERR_UNSUPPORTED, "token_logprobs: dtype %d (bf16 = 0, fp16 = 1, fp32 = 2)", a.dtype);
  if (a.top > score::MAX_TOP)
    return fail(DSPARK_ERR_UNSUPPORTED, "token_logprobs: %d alternatives (at most %d)", a.top, score::MAX_TOP);
  if (a.R > 0x7fffffff / score::MAX_CLUSTER)
    return fail(DSPARK_ERR_UNSUPPORTED, "token_logprobs: %d rows in one call", a.R);
  if (a.V > 0x7fffffff - 65536) return fail(DSPARK_ERR_UNSUPPORTED, "token_logprobs: %d tokens", a.V);
  if (a.R == 0) return DSPARK_OK;
  if (!a.logits || !a.tokens || !a.logprob || !a.entropy || !a.rank || (a.top && (!a.top_ids || !a.top_logprob)))
    return fail(DSPARK_ERR_ARG, "token_logprobs: null pointer");
  const int size = a.dtype == DSPARK_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a.logits) % size)
    return fail(DSPARK_ERR_UNSUPPORTED, "token_logprobs: logits must be aligned to their type");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  DSPARK_CUDA_TRY(a.dtype == DSPARK_DTYPE_BF16  ? score::launch<bf16>(a, s)
                  : a.dtype == DSPARK_DTYPE_F16 ? score::launch<__half>(a, s)
                                                : score::launch<float>(a, s),
                  "token_logprobs");
  return DSPARK_OK;
}
