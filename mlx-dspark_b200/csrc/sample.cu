// Verification of drafted tokens against the target's probabilities from given random numbers
// (dspark_sample_accept): two kernels chained by programmatic dependent launch.
//
// stat_kernel: (row, slice) blocks read each logits row that decides something (one with a child) once:
// running maximum and sum of exp2((l - m) log2e / T) in fp32, one (m, s, first largest) a slice. Rows
// without a child (a chain's last, a tree's leaves) are not read: the token after them needs no sum.
//
// pick_kernel: (request, slice) blocks join the slices' sums, walk the block or tree (every block of a
// request for itself, from a few hundred bytes), then read the one row that the next token comes from,
// with its noise and draft rows, once: the slice's best score and its place. The request's last block
// compares the slices in order (no result depends on timing) and writes the token.
//  * after a rejection with a draft distribution the score is max(p - q, 0) / e, with the row's sum;
//  * otherwise argmax p / e = argmax (l - ref) log2e / T - log2 e for any ref of the row: no sum, and
//    no rounding of p to zero. ref is the largest logit so far, so that scores stay near zero.
// Comparisons are made in 32 bits with the unit's exponential, logarithm and reciprocal, off by about 1e-6 of a
// probability: what lies closer than that may be decided either way.
// Bound: HBM (each deciding row once), or the two launches for a single block. Measured over 151,936
// tokens, 20 calls in a graph (a call of its own, host included): 256 chains of up to 16 rows 152 us (154 to
// 173; 0.90 to 0.79 of a plain copy), 16 trees of up to 61 nodes 36 us (39; 0.57: blocks of rows without a
// child and the walk's latency), five rows 12 us (17 to 22: the host).
#include <float.h>

#include <algorithm>

#include "elem.cuh"
#include "host_common.h"

namespace dspark {
namespace sample {

constexpr int THREADS = 256;
constexpr int MAX_ROWS = 1024;
constexpr int MAX_SLICE = 65536;   // values of one pick block (its bitmap: 8 KB)
constexpr float LOG2E = 1.4426950408889634f;

struct Stat {
  float m, s;  // largest logit, sum of exp((l - m) / T) of a slice
  int top;     // first place of the largest logit
  int pad;
};

struct Pick {  // a slice's best: score relative to ref, place (NONE: no token with mass may be kept)
  float ref, score;
  int place, pad;
};
constexpr int NONE = 0x7fffffff;

// A logit as the formulas take it: NaN has no mass, +inf is the largest finite value.
__device__ __forceinline__ float clean(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }
__device__ __forceinline__ bool greedy(float T) { return !(T > 0.f); }

// log2e / T, kept off zero and infinity, where the differences of -inf and equal logits would be lost.
__device__ __forceinline__ float slope(float T) { return fminf(fmaxf(LOG2E / T, FLT_MIN), 1e30f); }

// exp((l - m) / T), c = log2e / T. (-inf - -inf has no mass either.)
__device__ __forceinline__ float mass(float l, float m, float c) {
  return l == -INFINITY ? 0.f : ex2((l - m) * c);
}

__device__ __forceinline__ void better(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

// The larger of both halves of two words, NaN if one is.
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, bf16) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, float) {
  return __float_as_uint(max3(__uint_as_float(a), __uint_as_float(b), __uint_as_float(b)));
}

// Values of 16 bytes of a row.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  // The largest value of n vectors, NaN if there is one.
  static __device__ __forceinline__ float largest(const uint4* raw, int n) {
    uint32_t m = raw[0].x;
#pragma unroll
    for (int u = 0; u < n; ++u) {
      const uint32_t a = max2_nan(raw[u].x, raw[u].y, T()), b = max2_nan(raw[u].z, raw[u].w, T());
      m = max2_nan(m, max2_nan(a, b, T()), T());
    }
    if (sizeof(T) == 4) return __uint_as_float(m);
    const float2 f = Elem<T>::unpack(m);
    return max3(f.x, f.y, f.y);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = Elem<T>::unpack(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Whole 16-byte pieces of [p, p + bytes) into L2.
__device__ __forceinline__ void prefetch_l2(const void* p, int bytes) {
  const uintptr_t at = (reinterpret_cast<uintptr_t>(p) + 15) & ~uintptr_t(15);
  const int n = (bytes - int(at - reinterpret_cast<uintptr_t>(p))) & ~15;
  if (n > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(n) : "memory");
}

struct Running {
  float m = -INFINITY, s = 0.f;
  int top = 0x7fffffff;
};

// Joins two slices' maxima and sums.
__device__ __forceinline__ void join(Running& a, float m, float s, int top, float c, bool arg) {
  // (a maximum of -inf has no mass, whatever s says)
  if (arg) {
    better(a.m, a.top, m, top);
    return;
  }
  const float mn = fmaxf(a.m, m);
  a.s = a.s * mass(a.m, mn, c) + s * mass(m, mn, c);
  a.m = mn;
}

// The largest of a warp's values.
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// Joins a warp's maxima and sums, the same result in every lane.
__device__ __forceinline__ void warp_join(Running& a, float c, bool arg) {
  const float m = warp_max(a.m);
  if (arg) {
    a.top = __reduce_min_sync(0xffffffffu, a.m == m ? a.top : 0x7fffffff);
  } else {
    a.s *= mass(a.m, m, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
  }
  a.m = m;
}

// grid R * slices: block (r, slice). Also clears the requests' counts for the next kernel.
template <typename T>
__global__ void __launch_bounds__(THREADS) stat_kernel(const dspark_sample_args a, Stat* stat,
                                                       unsigned* done, const int slices) {
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  for (int b = blockIdx.x * THREADS + tid; b < a.B; b += gridDim.x * THREADS) done[b] = 0;
  const int r = blockIdx.x / slices, slice = blockIdx.x - r * slices;
  // the request of row r, and whether the row has a child
  __shared__ int s_b;
  if (tid == 0) s_b = -1;
  __syncthreads();
  for (int b = tid; b < a.B; b += THREADS)
    if (a.cu_rows[b] <= r && r < a.cu_rows[b + 1]) s_b = b;
  __syncthreads();
  const int b = s_b;
  if (b < 0) return;
  const int r0 = a.cu_rows[b], rows = min(a.cu_rows[b + 1], a.R) - r0;
  bool has = false;
  if (a.parent) {
    for (int j = r - r0 + 1 + tid; j < rows; j += THREADS) has |= a.parent[r0 + j] == r - r0;
  } else {
    has = r + 1 < r0 + rows;
  }
  if (!__syncthreads_or(has)) return;
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const bool arg = greedy(temp);
  const float c = arg ? 0.f : slope(temp);
  const T* row = static_cast<const T*>(a.logits) + int64_t(r) * a.ld_logits;
  constexpr int N = Vec<T>::N;
  // whole 16-byte vectors between the row's unaligned ends
  const int head = min(a.V, int((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / int(sizeof(T)));
  const int nv = (a.V - head) / N;
  const int v0 = int(int64_t(nv) * slice / slices), v1 = int(int64_t(nv) * (slice + 1) / slices);
  Running run;
  auto one = [&](int i) {
    const float x = clean(Elem<T>::to_f(row[i]));
    join(run, x, x == -INFINITY ? 0.f : 1.f, i, c, arg);
  };
  if (slice == 0 && tid < head) one(tid);
  if (slice == slices - 1 && tid < a.V - head - nv * N) one(head + nv * N + tid);
  const T* body = row + head;
  if (arg) {
    for (int v = v0 + tid; v < v1; v += THREADS) {
      float x[N];
      Vec<T>::unpack(ld_stream(body + int64_t(v) * N), x);
#pragma unroll
      for (int e = 0; e < N; ++e) better(run.m, run.top, clean(x[e]), head + v * N + e);
    }
  } else {
    // groups of G vectors under one maximum; the loop is bound by instructions as much as by HBM, so
    // values go in pairs, and only a group whose maximum is NaN or +inf is looked at one by one
    constexpr int G = sizeof(T) == 4 ? 4 : 2, U = 4;  // U vectors in flight a thread
    const f32x2 c2 = pack2(c, c);
    auto group = [&](const uint4* raw) {
      float mx = Vec<T>::largest(raw, G);
      if (!(mx < INFINITY)) {
        for (int u = 0; u < G; ++u) {
          float x[N];
          Vec<T>::unpack(raw[u], x);
#pragma unroll
          for (int e = 0; e < N; ++e) join(run, clean(x[e]), 1.f, 0, c, false);
        }
        return;
      }
      if (mx > run.m) {
        run.s *= mass(run.m, mx, c);
        run.m = mx;
      }
      if (run.m == -INFINITY) return;
      const f32x2 m2 = pack2(-run.m, -run.m);
      f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
      for (int u = 0; u < G; ++u) {
        float x[N];
        Vec<T>::unpack(raw[u], x);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          float p0, p1;
          unpack2(mul2(add2(pack2(x[e], x[e + 1]), m2), c2), p0, p1);
          sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pack2(ex2(p0), ex2(p1)));
        }
      }
      float s0, s1;
      unpack2(add2(sum[0], sum[1]), s0, s1);
      run.s += s0 + s1;
    };
    int v = v0 + tid;
    for (; v + (U - 1) * THREADS < v1; v += U * THREADS) {
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = ld_stream(body + int64_t(v + u * THREADS) * N);
#pragma unroll
      for (int u = 0; u < U; u += G) group(raw + u);
    }
    for (; v < v1; v += THREADS) {
      float x[N];
      Vec<T>::unpack(ld_stream(body + int64_t(v) * N), x);
#pragma unroll
      for (int e = 0; e < N; ++e) join(run, clean(x[e]), 1.f, 0, c, false);
    }
  }
  warp_join(run, c, arg);
  __shared__ Stat part[THREADS / 32];
  if ((tid & 31) == 0) part[tid >> 5] = Stat{run.m, run.s, run.top, 0};
  __syncthreads();
  if (tid < 32) {
    run = Running();
    if (tid < THREADS / 32) run.m = part[tid].m, run.s = part[tid].s, run.top = part[tid].top;
    warp_join(run, c, arg);
    if (tid == 0) stat[int64_t(r) * slices + slice] = Stat{run.m, run.s, run.top, 0};
  }
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// How the next token is scored.
enum Mode : int {
  kLargest,  // greedy: the logit
  kFree,     // any token, no sum known: (l - ref) c - log2 e
  kBarred,   // tokens tried are out, masses that are zero in 32 bits are none: the same, ref = m
  kRest      // max(p - q, 0) / e
};

struct Scorer {
  float m, c, inv;  // row's maximum and 1 / sum (kBarred, kRest), log2e / T
  float ref, best;
  int place;
  // places come in ascending order: the first of equal scores stays
  __device__ __forceinline__ void take(float score, int i) {
    if (score > best) {
      best = score;
      place = i;
    }
  }
  __device__ __forceinline__ void rebase(float mx) {  // kFree, before values up to mx
    if (!(mx > ref)) return;
    mx = fminf(mx, FLT_MAX);
    if (mx > ref) {
      best += ref == -INFINITY ? 0.f : (ref - mx) * c;
      ref = mx;
    }
  }
  template <Mode mode>
  __device__ __forceinline__ void look(float l, float q, float e, int i, bool barred) {
    if (mode == kRest) {
      const float p = ex2(fminf(fmaxf((l - m) * c, -INFINITY), 0.f)) * inv;
      take((p - q) * rcp(e), i);
    } else if (mode == kLargest) {
      if (!barred) take(clean(l), i);
    } else {
      l = clean(l);
      const float d = (l - ref) * c;
      if (!barred && l != -INFINITY && (mode == kFree || d >= -149.f)) take(d - lg2(e), i);
    }
  }
};

template <typename T, typename Q>
__global__ void __launch_bounds__(THREADS) pick_kernel(const dspark_sample_args a,
                                                       const int32_t* row_limit, const Stat* stat,
                                                       Pick* picks, unsigned* done, const int slices,
                                                       const int blocks) {
  pdl_launch_dependents();
  __shared__ float s_p[MAX_ROWS];           // p of each row's token given its parent
  __shared__ float s_m[MAX_ROWS], s_s[MAX_ROWS];
  __shared__ int s_up[MAX_ROWS], s_id[MAX_ROWS];  // a tree's parents and tokens
  __shared__ float s_u[MAX_ROWS];
  __shared__ int s_tried[MAX_ROWS];         // tokens tried at the last row
  __shared__ uint32_t s_map[MAX_SLICE / 32];  // those of them in this block's slice
  __shared__ int s_last, s_n, s_ntried, s_fail;
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / blocks, slice = blockIdx.x - b * blocks;
  const bool lead = slice == 0;  // this block writes what does not depend on the slice
  const int r0 = max(a.cu_rows[b], 0), rows = min(a.cu_rows[b + 1], a.R) - r0;
  if (rows <= 0) {
    if (lead && tid == 0) {
      a.n_accept[b] = 0;
      a.next_tok[b] = -1;
    }
    return;
  }
  int seen = min(rows, a.max_rows);  // rows that can be accepted
  if (row_limit) seen = min(seen, row_limit[b]);
  if (seen <= 0) {
    if (!lead) return;
    for (int i = tid; i < rows; i += THREADS) {
      if (a.path) a.path[r0 + i] = -1;
      if (a.prob) a.prob[r0 + i] = 0.f;
    }
    if (tid == 0) {
      a.n_accept[b] = 0;
      a.next_tok[b] = -1;
      if (a.lens) a.lens[b] = max(0, a.lens[b] - rows);
    }
    return;
  }
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const bool arg = greedy(temp);
  const float c = arg ? 0.f : slope(temp);
  const float* e = a.noise + int64_t(b) * a.ld_noise;
  // the slice: whole groups of eight values, dealt out evenly, so that no slice is wider than MAX_SLICE
  // (blocks_of: blocks * MAX_SLICE >= V, so blocks * (MAX_SLICE / 8) >= groups)
  const int groups = (a.V + 7) / 8;
  const int w0 = 8 * int(int64_t(groups) * slice / blocks);
  const int w1 = min(a.V, 8 * int(int64_t(groups) * (slice + 1) / blocks));
  if (!arg && tid == 0) prefetch_l2(e + w0, (w1 - w0) * 4);  // on its way to L2 beside the walk
  const T* logits = static_cast<const T*>(a.logits);
  const Q* draft = static_cast<const Q*>(a.draft);
  auto up = [&](int i) {
    const int u = a.parent ? a.parent[r0 + i] : i - 1;
    return u < i ? u : -1;  // a parent that is not before its child is none
  };

  // p of every row's token (beyond `seen` too: they are reported), and the sums of the rows that the
  // walk can end at; 4 to 32 lanes a row, all rows at once where there are up to 64. A chain's rows are
  // decided here.
  if (tid == 0) s_fail = MAX_ROWS;
  if (a.parent) {
    for (int i = tid; i < seen; i += THREADS) {
      s_up[i] = up(i);
      s_id[i] = a.ids[r0 + i];
      s_u[i] = a.u[r0 + i];
    }
  }
  __syncthreads();
  int span = 32;  // lanes a row
  while (span > 4 && rows * span > THREADS) span >>= 1;
  const int sub = tid & (span - 1);
  for (int i0 = tid / span; i0 < ((rows + 7) & ~7); i0 += THREADS / span) {
    const int u = i0 < rows ? up(i0) : -1;
    Running run;
    float l = -INFINITY, q = 1.f, chance = 0.f;
    int x = -1;
    if (u >= 0) {
      x = a.ids[r0 + i0];
      if (x >= 0 && x < a.V) {
        l = clean(Elem<T>::to_f(logits[int64_t(r0 + u) * a.ld_logits + x]));
        if (draft && !arg) q = Elem<Q>::to_f(draft[int64_t(r0 + u) * a.ld_draft + x]);
      }
      if (!a.parent) chance = a.u[r0 + u];
      for (int k = sub; k < slices; k += span) {
        const Stat st = stat[int64_t(r0 + u) * slices + k];
        join(run, st.m, st.s, st.top, c, arg);
      }
    }
    float m = run.m;
    for (int o = span / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (arg) {
      if (run.m != m) run.top = 0x7fffffff;
      for (int o = span / 2; o > 0; o >>= 1) run.top = min(run.top, __shfl_xor_sync(0xffffffffu, run.top, o));
    } else {
      run.s *= mass(run.m, m, c);
      for (int o = span / 2; o > 0; o >>= 1) run.s += __shfl_xor_sync(0xffffffffu, run.s, o);
    }
    run.m = m;
    if (sub == 0 && i0 < rows) {
      float p = 1.f;
      if (u >= 0) {
        if (arg) p = run.m != -INFINITY && x == run.top ? 1.f : 0.f;
        else p = run.s > 0.f ? mass(l, run.m, c) / run.s : 0.f;
      }
      if (lead && a.prob) a.prob[r0 + i0] = p;
      if (i0 < seen) {
        s_p[i0] = p;
        if (u >= 0) {  // every child of u writes the same
          s_m[u] = run.m;
          s_s[u] = run.s;
          if (!a.parent) {
            if (!(chance * q < p)) atomicMin(&s_fail, u);
            s_id[i0] = x;
          }
        }
      }
    }
  }
  __syncthreads();

  // the walk
  if (!a.parent) {
    const int stop = min(s_fail, seen - 1);
    if (tid == 0) {
      s_last = s_n = stop;
      s_ntried = stop + 1 < seen ? 1 : 0;
      if (s_ntried) s_tried[0] = s_id[stop + 1];
    }
    if (lead && a.path)
      for (int i = tid; i < rows; i += THREADS) a.path[r0 + i] = i <= stop ? i : -1;
  } else {
    if (warp == 0) {
      int cur = 0, n = 0, tried = 0;
      if (lead && a.path && lane == 0) a.path[r0] = 0;
      for (bool on = true; on;) {
        on = false;
        tried = 0;
        float run = 0.f;
        const float u = s_u[cur];
        for (int j0 = cur + 1; j0 < seen && !on; j0 += 32) {
          const int j = j0 + lane;
          const bool kid = j < seen && s_up[min(j, seen - 1)] == cur;
          const unsigned kids = __ballot_sync(0xffffffffu, kid);
          if (!kids) continue;
          int x = 0;
          float p = 0.f;
          bool twin = false;  // a token counts once
          if (kid) {
            x = s_id[j];
            p = s_p[j];
            twin = __match_any_sync(kids, x) & ((1u << lane) - 1u);
            for (int t = 0; t < tried; ++t) twin |= s_tried[t] == x;
          }
          unsigned fresh = __ballot_sync(0xffffffffu, kid && !twin);
          while (fresh) {
            const int l = __ffs(fresh) - 1;
            fresh &= fresh - 1;
            if (lane == l) s_tried[tried] = x;
            ++tried;
            run += __shfl_sync(0xffffffffu, p, l);
            if (u < run) {
              cur = j0 + l;
              ++n;
              if (lead && a.path && lane == 0) a.path[r0 + n] = cur;
              on = true;
              break;
            }
          }
          __syncwarp();
        }
      }
      if (lane == 0) {
        s_last = cur;
        s_n = n;
        s_ntried = tried;
      }
    }
  }
  __syncthreads();
  if (a.parent && lead && a.path)
    for (int i = s_n + 1 + tid; i < rows; i += THREADS) a.path[r0 + i] = -1;
  const int last = s_last, n = s_n, ntried = s_ntried;
  if (lead && tid == 0) {
    a.n_accept[b] = n;
    if (a.lens) a.lens[b] = max(0, a.lens[b] - (rows - 1 - n));
  }

  // the token after it
  const bool rest = draft && !arg && last + 1 < seen;  // a chain's rejection with a distribution
  const T* row = logits + int64_t(r0 + last) * a.ld_logits;
  const Q* qrow = rest ? draft + int64_t(r0 + last) * a.ld_draft : nullptr;
  const bool bar = !rest && ntried > 0;
  if (bar) {
    for (int i = tid; i < (w1 - w0 + 31) / 32; i += THREADS) s_map[i] = 0;
    __syncthreads();
    for (int t = tid; t < ntried; t += THREADS) {
      const int x = s_tried[t];
      if (x >= w0 && x < w1) atomicOr(&s_map[(x - w0) >> 5], 1u << ((x - w0) & 31));
    }
    __syncthreads();
  }
  auto out = [&](int i) { return bar && ((s_map[(i - w0) >> 5] >> ((i - w0) & 31)) & 1u); };
  Scorer sc;
  const Mode mode = rest ? kRest : arg ? kLargest : bar ? kBarred : kFree;
  sc.m = ntried ? s_m[last] : 0.f;
  sc.c = c;
  sc.inv = rest && s_s[last] > 0.f ? 1.f / s_s[last] : 0.f;
  sc.ref = mode == kBarred ? sc.m : mode == kFree ? -INFINITY : 0.f;
  sc.best = rest ? 0.f : -INFINITY;
  sc.place = NONE;
  const bool aligned = ((reinterpret_cast<uintptr_t>(row) | reinterpret_cast<uintptr_t>(e) |
                         reinterpret_cast<uintptr_t>(qrow)) & 15) == 0;
  auto scan = [&](auto mode_c) {
    constexpr Mode MODE = decltype(mode_c)::value;
    constexpr bool REST = MODE == kRest;
    auto single = [&](int i) {
      const float l = Elem<T>::to_f(row[i]);
      if (MODE == kFree) sc.rebase(l);
      sc.look<MODE>(l, REST ? Elem<Q>::to_f(qrow[i]) : 0.f, e[i], i, out(i));
    };
    if (!aligned) {
#pragma unroll 4
      for (int i = w0 + tid; i < w1; i += THREADS) single(i);
      return;
    }
    constexpr int U = 2;  // groups of eight values in flight a thread
    const int wv = w1 & ~7;
    for (int i0 = w0 + tid * 8; i0 < wv; i0 += U * THREADS * 8) {
      uint4 ez[U][2], xl[U][sizeof(T) / 2], ql[U][sizeof(Q) / 2];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * THREADS * 8;
        if (i >= wv) break;
        ez[k][0] = ld_stream(e + i);
        ez[k][1] = ld_stream(e + i + 4);
        xl[k][0] = ld_stream(row + i);
        if (sizeof(T) == 4) xl[k][sizeof(T) / 2 - 1] = ld_stream(row + i + 4);
        if (REST) {
          ql[k][0] = ld_stream(qrow + i);
          if (sizeof(Q) == 4) ql[k][sizeof(Q) / 2 - 1] = ld_stream(qrow + i + 4);
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * THREADS * 8;
        if (i >= wv) break;
        float x[8], q[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, z[8];
        Vec<float>::unpack(ez[k][0], z);
        Vec<float>::unpack(ez[k][1], z + 4);
        Vec<T>::unpack(xl[k][0], x);
        if (sizeof(T) == 4) Vec<T>::unpack(xl[k][sizeof(T) / 2 - 1], x + 4);
        if (REST) {
          Vec<Q>::unpack(ql[k][0], q);
          if (sizeof(Q) == 4) Vec<Q>::unpack(ql[k][sizeof(Q) / 2 - 1], q + 4);
        }
        if (MODE == kFree) {
          float mx = fmaxf(x[0], x[1]);
#pragma unroll
          for (int y = 2; y < 8; ++y) mx = fmaxf(mx, x[y]);
          sc.rebase(mx);
        }
        const uint32_t map = !REST && bar ? s_map[(i - w0) >> 5] >> ((i - w0) & 31) : 0u;
#pragma unroll
        for (int y = 0; y < 8; ++y) sc.look<MODE>(x[y], q[y], z[y], i + y, (map >> y) & 1u);
      }
    }
    for (int i = wv + tid; i < w1; i += THREADS) single(i);
  };
  if (mode == kRest) scan(std::integral_constant<Mode, kRest>());
  else if (mode == kLargest) scan(std::integral_constant<Mode, kLargest>());
  else if (mode == kBarred) scan(std::integral_constant<Mode, kBarred>());
  else scan(std::integral_constant<Mode, kFree>());

  // the best of the slice, then of the request's slices. Scores of different refs are put on the largest
  // of them first (the winner's own shift is small: less than log2 of the noise's range, so nothing is
  // lost in 32 bits; greedy and kRest: all refs are zero). Equal scores: the first place.
  __shared__ Pick s_pick[THREADS / 32];
  auto warp_best = [&](Pick x) {
    const bool any = x.place != NONE;
    const float ref = warp_max(any ? x.ref : -INFINITY);
    if (any && x.ref != ref) x.score += (x.ref - ref) * c;
    const float top = warp_max(any ? x.score : -INFINITY);
    x.place = __reduce_min_sync(0xffffffffu, any && x.score == top ? x.place : NONE);
    x.ref = ref;
    x.score = top;
    return x;
  };
  auto block_best = [&](Pick x) {
    x = warp_best(x);
    __syncthreads();
    if (lane == 0) s_pick[warp] = x;
    __syncthreads();
    x = Pick{0.f, 0.f, NONE, 0};
    if (lane < THREADS / 32) x = s_pick[lane];
    return warp_best(x);
  };
  const Pick mine = block_best(Pick{sc.ref, sc.best, sc.place, 0});
  __shared__ bool s_final;
  if (tid == 0) {
    picks[int64_t(b) * blocks + slice] = mine;
    __threadfence();
    s_final = atomicAdd(&done[b], 1u) + 1 == unsigned(blocks);
  }
  __syncthreads();
  if (!s_final) return;
  __threadfence();
  Pick win{0.f, 0.f, NONE, 0};
  for (int k = tid; k < blocks; k += THREADS) {
    const int4 raw = __ldcg(reinterpret_cast<const int4*>(&picks[int64_t(b) * blocks + k]));
    Pick x{__int_as_float(raw.x), __int_as_float(raw.y), raw.z, 0};
    if (x.place == NONE) continue;
    if (win.place != NONE) {  // (places ascend)
      const float ref = fmaxf(x.ref, win.ref);
      if (x.ref != ref) x.score += (x.ref - ref) * c;
      if (win.ref != ref) win.score += (win.ref - ref) * c;
      x.ref = win.ref = ref;
    }
    if (win.place == NONE || x.score > win.score) win = x;
  }
  win = block_best(win);
  if (win.place == NONE && (rest || bar)) {
    // nothing is left of the row's mass (only by rounding): the token is drawn from all of it
    Scorer all = sc;
    all.ref = arg ? 0.f : sc.m;
    all.best = -INFINITY;
    all.place = NONE;
    for (int i = tid; i < a.V; i += THREADS) {
      if (arg) all.look<kLargest>(Elem<T>::to_f(row[i]), 0.f, e[i], i, false);
      else all.look<kBarred>(Elem<T>::to_f(row[i]), 0.f, e[i], i, false);
    }
    win = block_best(Pick{all.ref, all.best, all.place, 0});
  }
  if (tid == 0) a.next_tok[b] = win.place == NONE ? -1 : win.place;
}

// Both rules by the mean of 35 mixes (1 to 96 requests; chains of 4 and 16 rows, trees of 16 and 61 nodes;
// 32000 to 200064 tokens, bf16 and fp32): 19.2 us a call with what stands here. In brackets what another
// value costs.
// Slices of a row for stat_kernel: of 128 KB, so that many rows do not end in a half-filled last round
// of blocks (64 KB 0.2 %, 256 KB nothing); with few rows more, blocks for eight an SM (four 3 %, twelve nothing,
// sixteen 1 %); at least 8192 values each (4096 2.5 %, 16384 4 %).
static int slices_of(int R, int V, int size, int sms) {
  const int want = (8 * sms + R - 1) / std::max(R, 1);
  return std::max(1, std::min(std::max(want, int(int64_t(V) * size / 131072)), V / 8192));
}
// Blocks of a request for pick_kernel: three an SM over all requests, which all run at once and walk
// side by side (two 2.5 %, four 5 %), but at least four a request (three to six nothing here, but 256 chains of
// up to 16 rows: three 160 us, four 152; eight 1 %), of at least 1024 values (512 1 %, 2048 1.5 %).
static int blocks_of(int B, int V, int sms) {
  const int want = std::max(4, (3 * sms + B - 1) / std::max(B, 1));
  return std::max((V + MAX_SLICE - 1) / MAX_SLICE, std::max(1, std::min(want, V / 1024)));
}

}  // namespace sample
}  // namespace dspark

using namespace dspark;

extern "C" {

size_t dspark_sample_workspace(int R, int B, int V) {
  if (R <= 0 || B <= 0 || V <= 0) return 0;
  const int sms = sm_count(current_device());
  return size_t(R) * sample::slices_of(R, V, 4, sms) * sizeof(sample::Stat) +
         size_t(B) * sample::blocks_of(B, V, sms) * sizeof(sample::Pick) + size_t(B) * sizeof(unsigned);
}

int dspark_sample_accept(const dspark_sample_args* p, void* stream) {
  return dspark_sample_accept_limited(p, nullptr, stream);
}

int dspark_sample_accept_limited(const dspark_sample_args* p, const int32_t* row_limit, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "sample_accept: null argument");
  const dspark_sample_args& a = *p;
  if (a.R < 0 || a.B < 0 || a.V <= 0) return fail(DSPARK_ERR_ARG, "sample_accept: bad shape");
  if (a.max_rows < 1 || a.max_rows > sample::MAX_ROWS)
    return fail(DSPARK_ERR_UNSUPPORTED, "sample_accept: max_rows %d (1..1024)", a.max_rows);
  if (a.dtype < DSPARK_DTYPE_BF16 || a.dtype > DSPARK_DTYPE_F32 ||
      (a.draft && (a.draft_dtype < DSPARK_DTYPE_BF16 || a.draft_dtype > DSPARK_DTYPE_F32)))
    return fail(DSPARK_ERR_UNSUPPORTED, "sample_accept: dtype %d / draft %d (bf16, fp16, fp32)", a.dtype,
                a.draft_dtype);
  if (a.B == 0) return DSPARK_OK;
  if (!a.cu_rows || !a.n_accept || !a.next_tok ||
      (a.R && (!a.logits || !a.ids || !a.u || !a.noise)))
    return fail(DSPARK_ERR_ARG, "sample_accept: null pointer");
  if (a.parent && a.draft)
    return fail(DSPARK_ERR_UNSUPPORTED, "sample_accept: a tree's proposals carry no draft distribution");
  // a stride of 0 is one row for all; anything else below V would overlap
  if (a.R && ((a.ld_logits && a.ld_logits < a.V) || (a.ld_noise && a.ld_noise < a.V) ||
              (a.draft && a.ld_draft && a.ld_draft < a.V)))
    return fail(DSPARK_ERR_ARG, "sample_accept: rows of %d values overlap", a.V);
  if (a.ws_bytes < dspark_sample_workspace(a.R, a.B, a.V) || (a.R && !a.workspace))
    return fail(DSPARK_ERR_ARG, "sample_accept: workspace of %zu bytes", a.ws_bytes);
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return fail(DSPARK_ERR_ARG, "sample_accept: the workspace must be 16-byte aligned");
  const int sms = sm_count(current_device());
  const int slices = sample::slices_of(a.R, a.V, a.dtype == DSPARK_DTYPE_F32 ? 4 : 2, sms);
  const int blocks = sample::blocks_of(a.B, a.V, sms);
  if (int64_t(a.R) * slices > 0x7fffffff || int64_t(a.B) * blocks > 0x7fffffff)
    return fail(DSPARK_ERR_UNSUPPORTED, "sample_accept: %d rows, %d requests", a.R, a.B);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  sample::Stat* st = static_cast<sample::Stat*>(a.workspace);
  sample::Pick* picks = reinterpret_cast<sample::Pick*>(st + int64_t(a.R) * slices);
  unsigned* done = reinterpret_cast<unsigned*>(picks + int64_t(a.B) * blocks);
#define DSPARK_STAT(T)                                                                             \
  DSPARK_CUDA_TRY(launch_ex(sample::stat_kernel<T>, dim3(a.R * slices), dim3(sample::THREADS), 0, s, 1, \
                            true, a, st, done, slices),                                            \
                  "sample_accept: sums")
#define DSPARK_PICK(T, Q)                                                                          \
  DSPARK_CUDA_TRY(launch_ex(sample::pick_kernel<T, Q>, dim3(a.B * blocks), dim3(sample::THREADS), 0, s, \
                            1, true, a, row_limit, (const sample::Stat*)st, picks, done, slices, blocks),            \
                  "sample_accept")
#define DSPARK_PICK_Q(T)                                                                           \
  do {                                                                                             \
    if (a.draft && a.draft_dtype == DSPARK_DTYPE_F32) DSPARK_PICK(T, float);                       \
    else if (a.draft && a.draft_dtype == DSPARK_DTYPE_F16) DSPARK_PICK(T, __half);                 \
    else DSPARK_PICK(T, bf16);                                                                     \
  } while (0)
  if (a.R) {
    if (a.dtype == DSPARK_DTYPE_BF16) DSPARK_STAT(bf16);
    else if (a.dtype == DSPARK_DTYPE_F16) DSPARK_STAT(__half);
    else DSPARK_STAT(float);
  }
  if (a.dtype == DSPARK_DTYPE_BF16) DSPARK_PICK_Q(bf16);
  else if (a.dtype == DSPARK_DTYPE_F16) DSPARK_PICK_Q(__half);
  else DSPARK_PICK_Q(float);
#undef DSPARK_STAT
#undef DSPARK_PICK
#undef DSPARK_PICK_Q
  return DSPARK_OK;
}

}  // extern "C"
