// Verification of drafted tokens against the target's probabilities from given random numbers
// (dspark_sample_accept).
//
// Simple form: one block a logits row for its maximum, sum and first largest logit; one block a
// request for the walk and the token after it.
#include <float.h>

#include "elem.cuh"
#include "host_common.h"

namespace dspark {
namespace sample {

// A logit as the formulas take it: NaN has no mass, +inf is the largest finite value.
__device__ __forceinline__ float clean(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }

struct RowStat {
  float m, s;  // largest logit, sum of exp((l - m) / T)
  int top;     // first place of the largest logit
  int pad;
};

// exp((l - m) / T); zero without mass (l = -inf, also where m is).
__device__ __forceinline__ float mass(float l, float m, float T) {
  return l == -INFINITY ? 0.f : expf((l - m) / T);
}

__device__ __forceinline__ bool greedy(float T) { return !(T > 0.f); }

template <typename T>
__device__ __forceinline__ float prob_at(const T* row, int v, int V, const RowStat& st, float temp) {
  if (v < 0 || v >= V || !(st.s > 0.f)) return 0.f;
  if (greedy(temp)) return v == st.top ? 1.f : 0.f;
  return mass(clean(Elem<T>::to_f(row[v])), st.m, temp) / st.s;
}

__device__ __forceinline__ int owner(const int32_t* cu, int B, int r) {
  if (r >= cu[B]) return -1;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void better(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

__device__ void block_best(float& v, int& i) {
  __shared__ float sv[32];
  __shared__ int si[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    better(v, i, ov, oi);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    sv[threadIdx.x >> 5] = v;
    si[threadIdx.x >> 5] = i;
  }
  __syncthreads();
  v = sv[0];
  i = si[0];
  for (int w = 1; w < int(blockDim.x >> 5); ++w) better(v, i, sv[w], si[w]);
}

template <typename T>
__global__ void __launch_bounds__(512) stat_simple_kernel(const dspark_sample_args a, RowStat* stat) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, b = owner(a.cu_rows, a.B, r);
  if (b < 0) return;
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const T* row = static_cast<const T*>(a.logits) + int64_t(r) * a.ld_logits;
  float m = -INFINITY;
  int top = 0x7fffffff;
  for (int v = threadIdx.x; v < a.V; v += blockDim.x) better(m, top, clean(Elem<T>::to_f(row[v])), v);
  block_best(m, top);
  float s = 0.f;
  if (greedy(temp)) {
    s = m == -INFINITY ? 0.f : 1.f;
  } else {
    for (int v = threadIdx.x; v < a.V; v += blockDim.x) s += mass(clean(Elem<T>::to_f(row[v])), m, temp);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __shared__ float ss[32];
    if ((threadIdx.x & 31) == 0) ss[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.f;
    for (int w = 0; w < int(blockDim.x >> 5); ++w) s += ss[w];
  }
  if (threadIdx.x == 0) stat[r] = RowStat{m, s, top, 0};
}

template <typename T, typename Q>
__global__ void __launch_bounds__(512) pick_simple_kernel(const dspark_sample_args a, const RowStat* stat) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const int r0 = a.cu_rows[b], rows = a.cu_rows[b + 1] - r0;
  if (rows <= 0) {
    if (threadIdx.x == 0) {
      a.n_accept[b] = 0;
      a.next_tok[b] = -1;
    }
    return;
  }
  const int seen = min(rows, a.max_rows);  // rows that can be accepted
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const T* logits = static_cast<const T*>(a.logits);
  const Q* draft = static_cast<const Q*>(a.draft);
  auto p = [&](int r, int v) { return prob_at(logits + int64_t(r) * a.ld_logits, v, a.V, stat[r], temp); };
  auto up = [&](int i) { return a.parent ? a.parent[r0 + i] : i - 1; };
  if (a.prob)
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
      const int u = up(i);
      a.prob[r0 + i] = u >= 0 && u < i ? p(r0 + u, a.ids[r0 + i]) : 1.f;
    }
  __shared__ int s_last, s_n;
  if (threadIdx.x == 0) {
    int cur = 0, n = 0;
    if (a.path) a.path[r0] = 0;
    for (bool more = true; more;) {
      more = false;
      float run = 0.f;
      for (int j = cur + 1; j < seen; ++j) {
        if (up(j) != cur) continue;
        const int x = a.ids[r0 + j];
        bool twin = false;
        for (int e = cur + 1; e < j; ++e) twin |= up(e) == cur && a.ids[r0 + e] == x;
        if (twin) continue;
        bool ok;
        const float px = p(r0 + cur, x);
        if (a.parent) {
          run += px;
          ok = a.u[r0 + cur] < run;
        } else {
          const float q = draft && !greedy(temp) && x >= 0 && x < a.V
                              ? Elem<Q>::to_f(draft[int64_t(r0 + cur) * a.ld_draft + x]) : 1.f;
          ok = a.u[r0 + cur] * q < px;
        }
        if (ok) {
          cur = j;
          ++n;
          if (a.path) a.path[r0 + n] = j;
          more = true;
          break;
        }
        if (!a.parent) break;
      }
    }
    s_last = cur;
    s_n = n;
    a.n_accept[b] = n;
    if (a.lens) a.lens[b] = max(0, a.lens[b] - (rows - 1 - n));
  }
  __syncthreads();
  const int last = s_last, n = s_n;
  if (a.path)
    for (int i = n + 1 + threadIdx.x; i < rows; i += blockDim.x) a.path[r0 + i] = -1;
  const RowStat st = stat[r0 + last];
  const bool rest = !a.parent && draft && !greedy(temp) && last + 1 < seen;
  const Q* qrow = draft ? draft + int64_t(r0 + last) * a.ld_draft : nullptr;
  const float* e = a.noise + int64_t(b) * a.ld_noise;
  float wv = 0.f, pv = 0.f;
  int wi = 0x7fffffff, pi = 0x7fffffff;
  for (int v = threadIdx.x; v < a.V; v += blockDim.x) {
    const float pr = p(r0 + last, v);
    float w = pr;
    if (rest) {
      w = fmaxf(pr - Elem<Q>::to_f(qrow[v]), 0.f);
    } else {
      for (int j = last + 1; j < seen; ++j)
        if (up(j) == last && a.ids[r0 + j] == v) w = 0.f;
    }
    if (w > 0.f) better(wv, wi, w / e[v], v);
    if (pr > 0.f) better(pv, pi, pr / e[v], v);
  }
  block_best(wv, wi);
  block_best(pv, pi);
  if (threadIdx.x == 0) a.next_tok[b] = !(st.s > 0.f) ? -1 : wi != 0x7fffffff ? wi : pi;
}

}  // namespace sample
}  // namespace dspark

using namespace dspark;

extern "C" {

size_t dspark_sample_workspace(int R, int B, int V) {
  (void)B; (void)V;
  return R > 0 ? size_t(R) * sizeof(sample::RowStat) : 0;
}

int dspark_sample_accept(const dspark_sample_args* p, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "sample_accept: null argument");
  const dspark_sample_args& a = *p;
  if (a.R < 0 || a.B < 0 || a.V <= 0) return fail(DSPARK_ERR_ARG, "sample_accept: bad shape");
  if (a.max_rows < 1 || a.max_rows > 1024)
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
  if (a.R && a.ld_logits < a.V) return fail(DSPARK_ERR_ARG, "sample_accept: logits rows overlap");
  if (a.ws_bytes < dspark_sample_workspace(a.R, a.B, a.V) || (a.R && !a.workspace))
    return fail(DSPARK_ERR_ARG, "sample_accept: workspace of %zu bytes", a.ws_bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  sample::RowStat* st = static_cast<sample::RowStat*>(a.workspace);
#define DSPARK_STAT(T)                                                                              \
  DSPARK_CUDA_TRY(launch_ex(sample::stat_simple_kernel<T>, dim3(a.R), dim3(512), 0, s, 1, true, a, st), \
                  "sample_accept")
#define DSPARK_PICK(T, Q)                                                                           \
  DSPARK_CUDA_TRY(launch_ex(sample::pick_simple_kernel<T, Q>, dim3(a.B), dim3(512), 0, s, 1, true, a, \
                            (const sample::RowStat*)st),                                            \
                  "sample_accept")
#define DSPARK_PICK_Q(T)                                                                            \
  do {                                                                                              \
    if (a.draft && a.draft_dtype == DSPARK_DTYPE_F32) DSPARK_PICK(T, float);                        \
    else if (a.draft && a.draft_dtype == DSPARK_DTYPE_F16) DSPARK_PICK(T, __half);                  \
    else DSPARK_PICK(T, bf16);                                                                      \
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
