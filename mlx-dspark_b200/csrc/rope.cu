// Rotary positions of packed q / k rows fused with the K/V append of a drafted tree
// (dspark_rope_append): the standalone form for targets whose rotary layout, rotated part,
// frequencies or cache slots the projection's epilogue does not serve.
//
// One pass over q, k and v: each value is read and written once (bound: HBM; a few rows: the launch).
// A lane owns 16 values of a head as two 16-byte chunks that hold whole pairs (half layout: chunk i
// and its partner half the rotated part away; interleaved: 16 neighbours), so a rotation needs no other
// lane, and a head's RMS norm only a sum over its lanes. A lane meets the same pairs in every head of
// its row: cosines and sines are computed once a row and lane.
// Measured: 16,389 rows of 32/8 heads of 128 69.1 us (5.8 TB/s, 0.89 of a plain copy); one row 2.4 us in
// a graph.
#include <algorithm>

#include "elem.cuh"
#include "host_common.h"

namespace dspark {
namespace rope {

// cos and sin of pos * f for a frequency in 64-bit fixed-point turns: the product wraps at whole
// turns, so the phase is exact to 2^-32 of a turn at any position. The reduced angle is within half a
// turn, where the special-function unit's cosine and sine are off by less than 1e-6: nothing beside
// the rounding to 16 bits.
__device__ __forceinline__ void phase(int pos, uint64_t f, float& c, float& s) {
  const uint64_t t = uint64_t(int64_t(pos)) * f;
  const float a = float(int32_t(uint32_t(t >> 32))) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  c = __cosf(a);
  s = __sinf(a);
}

constexpr int THREADS = 128;
constexpr int U = 4;  // heads in flight a lane

// Eight values at p.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, uint32_t* w) {
  if (VEC) {
    const uint4 v = ldcg_v4(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = uint32_t(h[2 * i]) | uint32_t(h[2 * i + 1]) << 16;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const uint32_t* w) {
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[2 * i] = uint16_t(w[i]);
      h[2 * i + 1] = uint16_t(w[i] >> 16);
    }
  }
}

// Warp w of the grid: row w / warps, heads of part w % warps (4 heads at a time with head_dim 128).
// lanes: lanes of a head, the next power of two of D / 16.
template <typename T, bool VEC, bool HALF>
__global__ void __launch_bounds__(THREADS) rope_kernel(const dspark_rope_args a, const int lanes,
                                                       const int warps, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int gw = int((blockIdx.x * unsigned(THREADS) + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  const int r = gw / warps, part = gw - r * warps;
  if (r >= a.R) return;
  const int per = 32 / lanes, group = lane / lanes, li = lane - group * lanes;
  const int D = a.D, turned = a.rot / 16;  // lanes that rotate
  const bool live = li < D / 16, turns = li < turned;
  const int c0 = turns && HALF ? 8 * li : 16 * li;
  const int c1 = turns && HALF ? a.rot / 2 + 8 * li : c0 + 8;
  const int pos = a.row_pos[r];
  const int req = a.row_req ? a.row_req[r] : 0;
  const int slot = a.Hk ? a.row_slot[r] : 0;
  const bool fits = slot >= 0 && slot < a.cap && req >= 0 && req < a.batch;
  if (a.Hk && !fits && req != -1 && lane == 0) report_error(status, 0x203);
  const int heads = a.Hq + (fits ? 2 * a.Hk : 0);

  auto source = [&](int h) {
    const T* p = h < a.Hq ? static_cast<const T*>(a.q) + r * a.q_strides[0] + h * a.q_strides[1]
                 : h < a.Hq + a.Hk
                     ? static_cast<const T*>(a.k) + r * a.k_strides[0] + (h - a.Hq) * a.k_strides[1]
                     : static_cast<const T*>(a.v) + r * a.v_strides[0] + (h - a.Hq - a.Hk) * a.v_strides[1];
    return p;
  };
  auto target = [&](int h) {
    T* p = h < a.Hq ? static_cast<T*>(a.q_out) + r * a.qo_strides[0] + h * a.qo_strides[1]
           : h < a.Hq + a.Hk ? static_cast<T*>(a.k_cache) + req * a.kc_strides[0] +
                                   (h - a.Hq) * a.kc_strides[1] + int64_t(slot) * a.kc_strides[2]
                             : static_cast<T*>(a.v_cache) + req * a.vc_strides[0] +
                                   (h - a.Hq - a.Hk) * a.vc_strides[1] + int64_t(slot) * a.vc_strides[2];
    return p;
  };
  const int h0 = part * per + group, step = warps * per;
  uint32_t raw[U][8];
  auto fetch = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (live && h + u * step < heads) {
        const T* p = source(h + u * step);
        load8<T, VEC>(p + c0, raw[u]);
        load8<T, VEC>(p + c1, raw[u] + 4);
      }
    }
  };
  fetch(h0);  // under way while the phases are computed
  float cs[8], sn[8];
  if (turns) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      phase(pos, a.freq[8 * li + i], cs[i], sn[i]);
      cs[i] *= a.mscale;
      sn[i] *= a.mscale;
    }
  }
  // a warp's groups leave the loop together (the norm's sum is over the warp)
  for (int hb = part * per; hb < heads; hb += U * step) {
    const int h = hb + group;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = h + u * step;
      if (hb + u * step >= heads) break;
      const bool mine = live && hh < heads;
      float x[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = Elem<T>::unpack(raw[u][i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
      const T* w = static_cast<const T*>(hh < a.Hq ? a.q_norm : hh < a.Hq + a.Hk ? a.k_norm : nullptr);
      if (a.q_norm || a.k_norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss += mine ? x[i] * x[i] : 0.f;
        for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && mine) {
          const float rs = rsqrtf(ss / float(D) + a.eps);
          uint32_t ww[8];
          load8<T, false>(w + c0, ww);
          load8<T, false>(w + c1, ww + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 f = Elem<T>::unpack(ww[i]);
            x[2 * i] *= rs * f.x;
            x[2 * i + 1] *= rs * f.y;
          }
        }
      }
      if (!mine) continue;
      uint32_t y[8];
      if (turns && hh < a.Hq + a.Hk) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int i0 = HALF ? i : 2 * i, i1 = HALF ? 8 + i : 2 * i + 1;
          const float p = x[i0], q = x[i1];
          x[i0] = p * cs[i] - q * sn[i];
          x[i1] = q * cs[i] + p * sn[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = Elem<T>::pack(x[2 * i], x[2 * i + 1]);
      } else if (w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = Elem<T>::pack(x[2 * i], x[2 * i + 1]);
      } else {  // copied as it is, bit by bit
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = raw[u][i];
      }
      T* p = target(hh);
      store8<T, VEC>(p + c0, y);
      store8<T, VEC>(p + c1, y + 4);
    }
    if (hb + U * step < heads) fetch(h + U * step);
  }
}

template <typename T, bool VEC>
static cudaError_t launch(const dspark_rope_args& a, cudaStream_t s) {
  int lanes = 1;
  while (lanes < a.D / 16) lanes *= 2;
  // warps a row: one, unless that leaves less than 32 warps an SM (then as many as take U heads a lane)
  const int sms = sm_count(current_device()), heads = a.Hq + 2 * a.Hk, per = 32 / lanes;
  const int most = (heads + per - 1) / per, want = (32 * sms + a.R - 1) / a.R;
  const int warps = std::max(1, std::min(want, most));
  const int64_t blocks = (int64_t(a.R) * warps * 32 + THREADS - 1) / THREADS;
  int* st = status_word(current_device());
  return a.layout == DSPARK_ROPE_HALF
             ? launch_ex(rope_kernel<T, VEC, true>, dim3(unsigned(blocks)), dim3(THREADS), 0, s, 1, true, a,
                         lanes, warps, st)
             : launch_ex(rope_kernel<T, VEC, false>, dim3(unsigned(blocks)), dim3(THREADS), 0, s, 1, true, a,
                         lanes, warps, st);
}

// Whether every head of every row starts on a 16-byte boundary.
static bool aligned16(const dspark_rope_args& a) {
  auto ok = [](const void* p, const int64_t* st, int n) {
    bool r = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int i = 0; i < n; ++i) r &= st[i] % 8 == 0;
    return r;
  };
  bool r = !a.Hq || (ok(a.q, a.q_strides, 2) && ok(a.q_out, a.qo_strides, 2));
  if (a.Hk)
    r &= ok(a.k, a.k_strides, 2) && ok(a.v, a.v_strides, 2) && ok(a.k_cache, a.kc_strides, 3) &&
         ok(a.v_cache, a.vc_strides, 3);
  return r;
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
  const bool vec = rope::aligned16(a);
  DSPARK_CUDA_TRY(a.dtype == DSPARK_DTYPE_BF16
                      ? (vec ? rope::launch<bf16, true>(a, s) : rope::launch<bf16, false>(a, s))
                      : (vec ? rope::launch<__half, true>(a, s) : rope::launch<__half, false>(a, s)),
                  "rope_append");
  return DSPARK_OK;
}
