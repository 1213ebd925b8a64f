// Attention of drafted trees over the cache (dspark_tree_attn): packed rows of ragged requests, each
// row seeing its request's cached prefix and its own ancestors.
//
// Simple form: one warp a (row, query head); 32 keys at a time, a lane a key for the scores
// (running maximum and sum in fp32), a lane D / 32 values of the output for the weighted sum.
#include "elem.cuh"
#include "host_common.h"

namespace dspark {
namespace tattn {

// The request that owns packed row r: the largest b with cu[b] <= r, or -1 past the last row.
__device__ __forceinline__ int owner(const int32_t* cu, int B, int r) {
  if (r >= cu[B]) return -1;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T, int D>
__global__ void __launch_bounds__(32) simple_kernel(const dspark_tree_attn_args a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int VPL = D / 32;
  const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int b = owner(a.cu_rows, a.B, r);
  if (b < 0) return;
  __shared__ float qs[D];
  const T* q = static_cast<const T*>(a.q) + r * a.q_strides[0] + h * a.q_strides[1];
  for (int d = lane; d < D; d += 32) qs[d] = Elem<T>::to_f(q[d]) * a.scale;
  __syncwarp();
  const int r0 = a.cu_rows[b], rows = a.cu_rows[b + 1] - r0, i = r - r0;
  const int start = a.kv_start ? a.kv_start[b] : 0;
  const int len = min(a.kv_len[b], a.cap - start), first = a.kv_len[b] - rows;
  const int hk = h / (a.Hq / a.Hk), kb = a.kv_batch == 1 ? 0 : b;
  const T* kp = static_cast<const T*>(a.k) + kb * a.k_strides[0] + hk * a.k_strides[1] +
                int64_t(start) * a.k_strides[2];
  const T* vp = static_cast<const T*>(a.v) + kb * a.v_strides[0] + hk * a.v_strides[1] +
                int64_t(start) * a.v_strides[2];
  float m = -INFINITY, l = 0.f, o[VPL];
#pragma unroll
  for (int e = 0; e < VPL; ++e) o[e] = 0.f;
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane, t = j - first;
    bool sees = j < len;
    if (sees && t >= 0)
      sees = a.anc ? t < 32 * a.anc_words &&
                         ((a.anc[int64_t(r) * a.anc_words + (t >> 5)] >> (t & 31)) & 1u)
                   : t <= i;
    float s = -INFINITY;
    if (sees) {
      s = 0.f;
      const T* kr = kp + int64_t(j) * a.k_strides[2];
      for (int d = 0; d < D; ++d) s += qs[d] * Elem<T>::to_f(kr[d]);
    }
    float mt = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
    const float mn = fmaxf(m, mt);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float keep = expf(m - base);
    const float p = sees ? expf(s - base) : 0.f;
    float ps = p;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, x);
    l = l * keep + ps;
    m = mn;
#pragma unroll
    for (int e = 0; e < VPL; ++e) o[e] *= keep;
    unsigned live = __ballot_sync(0xffffffffu, sees);
    while (live) {
      const int x = __ffs(live) - 1;
      live &= live - 1;
      const float px = __shfl_sync(0xffffffffu, p, x);
      const T* vr = vp + int64_t(j0 + x) * a.v_strides[2];
#pragma unroll
      for (int e = 0; e < VPL; ++e) o[e] += px * Elem<T>::to_f(vr[lane + 32 * e]);
    }
  }
  T* out = static_cast<T*>(a.out) + r * a.o_strides[0] + h * a.o_strides[1];
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < VPL; ++e) out[lane + 32 * e] = Elem<T>::from_f(o[e] * inv);
}

}  // namespace tattn
}  // namespace dspark

using namespace dspark;

extern "C" {

size_t dspark_tree_attn_workspace(int B, int Hq, int Hk, int D, int max_rows) {
  (void)B; (void)Hq; (void)Hk; (void)D; (void)max_rows;
  return 0;
}

int dspark_tree_attn(const dspark_tree_attn_args* p, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "tree_attn: null argument");
  const dspark_tree_attn_args& a = *p;
  if (a.R < 0 || a.B < 0 || a.Hq <= 0 || a.Hk <= 0 || a.Hq % a.Hk || a.cap < 0 || a.max_rows < 0)
    return fail(DSPARK_ERR_ARG, "tree_attn: bad shape (%d rows, %d requests, %d / %d heads)", a.R, a.B,
                a.Hq, a.Hk);
  if (a.dtype != DSPARK_DTYPE_BF16 && a.dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "tree_attn: dtype %d (bf16 = 0, fp16 = 1)", a.dtype);
  if (a.D != 64 && a.D != 128)
    return fail(DSPARK_ERR_UNSUPPORTED, "tree_attn: head_dim %d (64 or 128)", a.D);
  if (a.R == 0 || a.B == 0) return DSPARK_OK;
  if (a.kv_batch != 1 && a.kv_batch < a.B)
    return fail(DSPARK_ERR_ARG, "tree_attn: %d requests, %d cache entries", a.B, a.kv_batch);
  if (!a.q || !a.k || !a.v || !a.out || !a.cu_rows || !a.kv_len)
    return fail(DSPARK_ERR_ARG, "tree_attn: null pointer");
  if (a.anc && a.anc_words <= 0) return fail(DSPARK_ERR_ARG, "tree_attn: %d words a row", a.anc_words);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define DSPARK_TATTN(T, DD)                                                                        \
  DSPARK_CUDA_TRY(launch_ex(tattn::simple_kernel<T, DD>, dim3(a.R, a.Hq), dim3(32), 0, s, 1, true, a), \
                  "tree_attn")
  if (a.dtype == DSPARK_DTYPE_BF16) {
    if (a.D == 128) DSPARK_TATTN(bf16, 128); else DSPARK_TATTN(bf16, 64);
  } else {
    if (a.D == 128) DSPARK_TATTN(__half, 128); else DSPARK_TATTN(__half, 64);
  }
#undef DSPARK_TATTN
  return DSPARK_OK;
}

}  // extern "C"
