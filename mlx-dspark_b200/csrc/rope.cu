// Rotary positions of packed q / k rows fused with the K/V append of a drafted tree
// (dspark_rope_append): the standalone form for targets whose rotary layout, rotated part,
// frequencies or cache slots the projection's epilogue does not serve.
//
// Simple form: one block a row, a thread a pair.
#include "elem.cuh"
#include "host_common.h"

namespace dspark {
namespace rope {

// cos and sin of pos * f for a frequency in 64-bit fixed-point turns: the product wraps at whole
// turns, so the phase is exact to 2^-32 of a turn at any position.
__device__ __forceinline__ void phase(int pos, uint64_t f, float& c, float& s) {
  const uint64_t t = uint64_t(int64_t(pos)) * f;
  const float half_turns = float(int32_t(uint32_t(t >> 32))) * 4.656612873077393e-10f;  // 2^-31
  sincospif(half_turns, &s, &c);
}

template <typename T>
__global__ void __launch_bounds__(256) rope_simple_kernel(const dspark_rope_args a, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int pos = a.row_pos[r];
  const int req = a.row_req ? a.row_req[r] : 0;
  const int slot = a.Hk ? a.row_slot[r] : 0;
  const bool fits = slot >= 0 && slot < a.cap && req >= 0 && req < a.batch;
  if (a.Hk && !fits && threadIdx.x == 0) report_error(status, 0x203);
  const int D = a.D, rot = a.rot;
  for (int h = warp; h < a.Hq + 2 * a.Hk; h += nw) {
    const T* src;
    T* dst;
    const T* w = nullptr;
    const bool is_v = h >= a.Hq + a.Hk;
    if (h < a.Hq) {
      src = static_cast<const T*>(a.q) + r * a.q_strides[0] + h * a.q_strides[1];
      dst = static_cast<T*>(a.q_out) + r * a.qo_strides[0] + h * a.qo_strides[1];
      w = static_cast<const T*>(a.q_norm);
    } else if (!is_v) {
      const int hh = h - a.Hq;
      if (!fits) continue;
      src = static_cast<const T*>(a.k) + r * a.k_strides[0] + hh * a.k_strides[1];
      dst = static_cast<T*>(a.k_cache) + req * a.kc_strides[0] + hh * a.kc_strides[1] +
            int64_t(slot) * a.kc_strides[2];
      w = static_cast<const T*>(a.k_norm);
    } else {
      const int hh = h - a.Hq - a.Hk;
      if (!fits) continue;
      src = static_cast<const T*>(a.v) + r * a.v_strides[0] + hh * a.v_strides[1];
      dst = static_cast<T*>(a.v_cache) + req * a.vc_strides[0] + hh * a.vc_strides[1] +
            int64_t(slot) * a.vc_strides[2];
    }
    if (is_v) {
      for (int d = lane; d < D; d += 32) dst[d] = src[d];
      continue;
    }
    float rs = 1.f;
    if (w) {
      float ss = 0.f;
      for (int d = lane; d < D; d += 32) {
        const float x = Elem<T>::to_f(src[d]);
        ss += x * x;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rs = rsqrtf(ss / float(D) + a.eps);
    }
    for (int i = lane; i < rot / 2; i += 32) {
      const int i0 = a.layout == DSPARK_ROPE_HALF ? i : 2 * i;
      const int i1 = a.layout == DSPARK_ROPE_HALF ? i + rot / 2 : 2 * i + 1;
      float x0 = Elem<T>::to_f(src[i0]), x1 = Elem<T>::to_f(src[i1]);
      if (w) {
        x0 *= rs * Elem<T>::to_f(w[i0]);
        x1 *= rs * Elem<T>::to_f(w[i1]);
      }
      float c, s;
      phase(pos, a.freq[i], c, s);
      c *= a.mscale;
      s *= a.mscale;
      dst[i0] = Elem<T>::from_f(x0 * c - x1 * s);
      dst[i1] = Elem<T>::from_f(x1 * c + x0 * s);
    }
    for (int d = rot + lane; d < D; d += 32) {
      float x = Elem<T>::to_f(src[d]);
      if (w) x *= rs * Elem<T>::to_f(w[d]);
      dst[d] = Elem<T>::from_f(x);
    }
  }
}

}  // namespace rope
}  // namespace dspark

using namespace dspark;

extern "C" int dspark_rope_append(const dspark_rope_args* p, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "rope_append: null argument");
  const dspark_rope_args& a = *p;
  if (a.R < 0 || a.Hq < 0 || a.Hk < 0 || a.Hq + a.Hk == 0)
    return fail(DSPARK_ERR_ARG, "rope_append: bad shape (%d rows, %d / %d heads)", a.R, a.Hq, a.Hk);
  if (a.dtype != DSPARK_DTYPE_BF16 && a.dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "rope_append: dtype %d (bf16 = 0, fp16 = 1)", a.dtype);
  if (a.layout != DSPARK_ROPE_HALF && a.layout != DSPARK_ROPE_INTERLEAVED)
    return fail(DSPARK_ERR_ARG, "rope_append: layout %d", a.layout);
  if (a.D <= 0 || a.D % 16 || a.D > 512)
    return fail(DSPARK_ERR_UNSUPPORTED, "rope_append: head_dim %d (a multiple of 16, at most 512)", a.D);
  if (a.rot <= 0 || a.rot % 16 || a.rot > a.D)
    return fail(DSPARK_ERR_UNSUPPORTED, "rope_append: rotary dim %d of %d (a multiple of 16)", a.rot, a.D);
  if (a.R == 0) return DSPARK_OK;
  if (!a.freq || !a.row_pos || (a.Hq && (!a.q || !a.q_out)))
    return fail(DSPARK_ERR_ARG, "rope_append: null pointer");
  if (a.Hk && (!a.k || !a.v || !a.k_cache || !a.v_cache || !a.row_slot))
    return fail(DSPARK_ERR_ARG, "rope_append: k needs v, both caches and row_slot");
  if (a.Hk && (a.cap <= 0 || a.batch <= 0)) return fail(DSPARK_ERR_ARG, "rope_append: empty cache");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int* st = status_word(current_device());
  if (a.dtype == DSPARK_DTYPE_BF16)
    DSPARK_CUDA_TRY(launch_ex(rope::rope_simple_kernel<bf16>, dim3(a.R), dim3(256), 0, s, 1, true, a, st),
                    "rope_append");
  else
    DSPARK_CUDA_TRY(launch_ex(rope::rope_simple_kernel<__half>, dim3(a.R), dim3(256), 0, s, 1, true, a, st),
                    "rope_append");
  return DSPARK_OK;
}
