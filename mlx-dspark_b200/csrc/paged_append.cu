// Rotary positions of packed q and k rows with the append of k and v to pages of 8-bit values
// (dspark_paged_append).
//
// A page holds `page` tokens of every head; the value of a code is e4m3(code) * scale, one scale a page and head:
// the smallest power of two with which the page's largest value is at most 448. Powers of two, because an append
// to a page that holds tokens may raise its scale: the old codes are then multiplied by a power of two, which
// changes none of them but those that end below e4m3's normal range (2^-6), so that a page filled token by token
// is all but one filled at once. Rotation, norm and the division by the scale are fp32 and rounded once.
//
// Blocks: first those of the cache, one a (page that the call writes to, group of heads, k or v): a page's largest
// value is then known inside a block, which holds a head's new values in registers meanwhile. Then those of q, a warp or more a
// row. Which page a block has is found from cu_rows without a sum over the requests: request b's pages
// start at unit cu_rows[b] / page + 2 b, which leaves room for every page that n rows can touch (n / page + 2).
// Bound: HBM and instructions for prompts (each value is read and written once; 16,389 rows of 32/8 heads of 128 79 us, 0.71
// of the measured rate; 84 with operations on single values instead of pairs), the launch for few rows (one row 3.2 us).
#include <algorithm>

#include "host_common.h"
#include "paged.cuh"

namespace dspark {
namespace paged {

constexpr int U = 4;  // heads of q in flight a lane

// cos and sin of pos * f, f in 64-bit fixed-point turns (the product wraps at whole turns: any position keeps its
// phase to 2^-32 of a turn), to a little more than half an fp32 step: not the special-function unit's, which are off by
// up to 1e-6, for every error sends its share of values to the other side of a border between two codes. The angle
// from the nearest quarter turn, up to pi / 4, is a + d, d what is lost in fp32: its first 23 bits a product with its
// rounding, the others' product. Taylor series to the 9th and 10th power (off by 2e-9 and 1e-10), d by their derivatives,
// the largest term added last.
__device__ __forceinline__ void phase(int pos, uint64_t f, float& c, float& s) {
  constexpr float K = 0x1.921fb60000000p-30f, K_LOW = -0x1.777a5c0000000p-55f;  // 2 pi / 2^32, and what fp32 leaves of it
  const uint32_t t = uint32_t((uint64_t(int64_t(pos)) * f) >> 32), quarter = (t + 0x20000000u) >> 30;
  const int r = int(t - (quarter << 30));
  const float hi = float(r & ~127), a = hi * K, z = a * a;
  const float d = fmaf(float(r & 127), K, fmaf(hi, K_LOW, fmaf(hi, K, -a)));
  const float p = fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6);
  const float q = fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f);
  const float sn = a + fmaf(a * z, p, d * fmaf(z, q, 1.f)), cs = 1.f + fmaf(z, q, -d * a);
  const float x = quarter & 1 ? sn : cs, y = quarter & 1 ? cs : sn;
  c = __uint_as_float(__float_as_uint(x) ^ ((quarter + 1) & 2) << 30);
  s = __uint_as_float(__float_as_uint(y) ^ (quarter & 2) << 30);
}

// Sixteen values of a row: eight at p + c0 and eight at p + c1.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* p, int c0, int c1, uint32_t* w) {
  if (VEC) {
    const uint4 a = ldcg_v4(p + c0), b = ldcg_v4(p + c1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = i < 4 ? c0 + 2 * i : c1 + 2 * (i - 4);
      w[i] = uint32_t(h[at]) | uint32_t(h[at + 1]) << 16;
    }
  }
}

// A lane's sixteen values in pairs: p[j] has those of rotary pairs 2 j and 2 j + 1 that come first, q[j] their partners (in the
// half layout values 2 j, 2 j + 1 and 8 + 2 j, 9 + 2 j, else 4 j, 4 j + 2 and 4 j + 1, 4 j + 3).
struct Vals {
  f32x2 p[4], q[4];
};

template <typename T, bool HALF>
__device__ __forceinline__ Vals unpack16(const uint32_t* w) {
  Vals x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = Elem<T>::unpack(w[HALF ? j : 2 * j]), b = Elem<T>::unpack(w[HALF ? 4 + j : 2 * j + 1]);
    x.p[j] = HALF ? pack2(a.x, a.y) : pack2(a.x, b.x);
    x.q[j] = HALF ? pack2(b.x, b.y) : pack2(a.y, b.y);
  }
  return x;
}

// The values in their order.
template <bool HALF>
__device__ __forceinline__ void in_order(const Vals& v, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unpack2(v.p[j], x[HALF ? 2 * j : 4 * j], x[HALF ? 2 * j + 1 : 4 * j + 2]);
    unpack2(v.q[j], x[HALF ? 8 + 2 * j : 4 * j + 1], x[HALF ? 9 + 2 * j : 4 * j + 3]);
  }
}

// RMS norm of a head whose 16-value parts are on `lanes` neighbouring lanes, then the rotation of the lane's part. cs, sn: two
// pairs' cosines and sines.
template <typename T, bool HALF>
__device__ __forceinline__ void norm_turn(Vals& x, const uint32_t* weight, bool norm, int lanes, float inv_d, float eps,
                                          bool turns, const f32x2* cs, const f32x2* sn) {
  if (norm) {
    f32x2 s2 = mul2(x.p[0], x.p[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) s2 = fma2(x.p[j], x.p[j], s2);
#pragma unroll
    for (int j = 0; j < 4; ++j) s2 = fma2(x.q[j], x.q[j], s2);
    float ss, other;
    unpack2(s2, ss, other);
    ss += other;
    for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float rs = rsqrtf(ss * inv_d + eps);
    const Vals w = unpack16<T, HALF>(weight);
    const f32x2 r2 = pack2(rs, rs);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x.p[j] = mul2(x.p[j], mul2(r2, w.p[j]));
      x.q[j] = mul2(x.q[j], mul2(r2, w.q[j]));
    }
  }
  if (turns) {
    const f32x2 minus = pack2(-1.f, -1.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 p = x.p[j], q = x.q[j];
      x.p[j] = fma2(q, mul2(sn[j], minus), mul2(p, cs[j]));
      x.q[j] = fma2(p, sn[j], mul2(q, cs[j]));
    }
  }
}

// cos and sin of two neighbouring pairs, times mscale.
__device__ __forceinline__ void two_phases(int pos, const uint64_t* f, float mscale, f32x2& cs, f32x2& sn) {
  float c0, s0, c1, s1;
  phase(pos, f[0], c0, s0);
  phase(pos, f[1], c1, s1);
  cs = pack2(c0 * mscale, c1 * mscale);
  sn = pack2(s0 * mscale, s1 * mscale);
}

// One (page, some heads, k or v). PASS rounds of 16 values a thread. Cosines and sines
// are the same for all heads: they wait in shared memory, where each thread reads its own.
template <typename T, bool VEC, bool HALF, int PASS, int THREADS>
__device__ void append_page(const dspark_paged_append_args& a, int unit, int groups, int* status) {
  extern __shared__ ulonglong2 s_turn[];  // [PASS][4][THREADS]: two pairs' cosines, their sines
  __shared__ uint32_t s_max[2][THREADS / 32];
  const int tid = threadIdx.x, D = a.D, lanes = D / 16, li = tid % lanes;
  const int kv = unit & 1, hu = unit >> 1, u = hu / groups, group = hu - u * groups;
  const int shift = 31 - __clz(a.page);
  const int b = last_at_most(a.B, u, [&](int i) { return (first_row(a.cu_rows, i, a.R) >> shift) + 2 * i; });
  const int r0 = first_row(a.cu_rows, b, a.R), n = max(first_row(a.cu_rows, b + 1, a.R) - r0, 0);
  const int j = u - (r0 >> shift) - 2 * b;
  const int64_t len = max(a.kv_len[b], 0), room = int64_t(a.max_pages) << shift;
  if (j < 0) return;
  if (j == 0 && group == 0 && kv == 0 && tid == 0 && a.len_out) a.len_out[b] = int32_t(min(len + n, max(room, len)));
  const int64_t pi = (len >> shift) + j;
  if (n == 0 || pi > (len + n - 1) >> shift) return;
  const int begin = j == 0 ? int(len & (a.page - 1)) : 0;       // tokens that the page has
  const int place0 = int((pi << shift) + begin - len);          // the first new one's place in the request
  const int count = min(a.page - begin, n - place0);
  const int h0 = int(int64_t(a.Hk) * group / groups), h1 = int(int64_t(a.Hk) * (group + 1) / groups);
  const int64_t row_stride = kv ? a.v_strides[0] : a.k_strides[0], head_stride = kv ? a.v_strides[1] : a.k_strides[1];
  const bool turns = !kv && li < a.rot / 16, half = turns && HALF;
  const int c0 = half ? 8 * li : 16 * li, c1 = half ? a.rot / 2 + 8 * li : c0 + 8;
  constexpr int W = THREADS * 16;  // values a round
  static_assert(PASS <= 2, "a head's rows and the next one's in registers");
  const int per = W / D, first = tid / lanes;
  const T* src = static_cast<const T*>(kv ? a.v : a.k) + (r0 + place0 + first) * row_stride;
  uint32_t raw[PASS][8];
  auto fetch = [&](int h) {
#pragma unroll
    for (int z = 0; z < PASS; ++z)
      if (z * per + first < count) load16<T, VEC>(src + z * per * row_stride + h * head_stride, c0, c1, raw[z]);
  };
  if (count <= PASS * per) fetch(h0);  // under way while the page is looked up
  const int pid = pi < a.max_pages ? a.page_table[int64_t(b) * a.table_stride + pi] : -1;
  if (pid < 0 || pid >= a.n_pages) {
    if (tid == 0) report_error(status, kErrAppendPage);
    return;
  }
  const int64_t ts = kv ? a.vp_strides[2] : a.kp_strides[2], hs = kv ? a.vp_strides[1] : a.kp_strides[1];
  uint8_t* page = static_cast<uint8_t*>(kv ? a.v_pages : a.k_pages) + pid * (kv ? a.vp_strides[0] : a.kp_strides[0]);
  float* scales = (kv ? a.v_scale : a.k_scale) + pid * a.scale_strides[0];
  float old = begin ? scales[h0 * a.scale_strides[1]] : 0.f;
  const bool norm = !kv && a.k_norm;
  uint32_t weight[8];
  if (norm) load16<T, false>(static_cast<const T*>(a.k_norm), c0, c1, weight);
  // The codes of 16 values of the page's new row t.
  auto put = [&](uint8_t* codes, int t, const Vals& v, float inv) {
    const f32x2 i2 = pack2(inv, inv);
    Vals z;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      z.p[j] = mul2(v.p[j], i2);
      z.q[j] = mul2(v.q[j], i2);
    }
    float x[16];
    in_order<HALF>(z, x);
    uint32_t y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = f32_to_e4m3(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    uint8_t* p = codes + (begin + t) * ts;
    if (half) {
      *reinterpret_cast<uint2*>(p + c0) = make_uint2(y[0], y[1]);
      *reinterpret_cast<uint2*>(p + c1) = make_uint2(y[2], y[3]);
    } else {
      *reinterpret_cast<uint4*>(p + c0) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  };
  auto larger = [](float top, const Vals& v) {  // the largest finite value (NaN: 0)
    float x[16], m = top;
    in_order<HALF>(v, x);
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = max3(m, fabsf(x[i]), fabsf(x[i + 1]));
    if (m < INFINITY) return m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // rare
      const float y = fabsf(x[i]);
      top = fmaxf(top, y < INFINITY ? y : 0.f);
    }
    return top;
  };
  // The head's scale, from the threads' largest values; its page's old codes are rounded to it. Returns its inverse.
  auto settle = [&](int h, float top, float before) {
    const uint32_t wm = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if ((tid & 31) == 0) s_max[h & 1][tid >> 5] = wm;
    __syncthreads();
    uint32_t m = s_max[h & 1][0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) m = max(m, s_max[h & 1][i]);
    const int e = scale_exponent(__uint_as_float(m));
    const float need = pow2(e);
    const float now = before > need ? before : need;  // (what is no scale gives way)
    uint8_t* codes = page + h * hs;
    if (begin && now != before) {
      const float f = before == before ? before / now : 0.f;  // (a scale of zero or NaN: the page's tokens are zeros)
      for (int i = tid; i < begin * lanes; i += THREADS) {
        uint4* p = reinterpret_cast<uint4*>(codes + (i / lanes) * ts + (i % lanes) * 16);
        uint4 w = *p;
        uint32_t* y = &w.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t l2 = e4m3_to_f16(y[k]), h2 = e4m3_to_f16_hi(y[k]);
          const float2 lo = Elem<__half>::unpack(l2), hi = Elem<__half>::unpack(h2);
          y[k] = f32_to_e4m3(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
        }
        *p = w;
      }
    }
    if (tid == 0 && now != before) scales[h * a.scale_strides[1]] = now;
    return before > need ? 1.f / before : pow2(-e);
  };
  if (count > PASS * per) {  // more rows than the block holds: they are made twice, for the scale and for the codes
    for (int h = h0; h < h1; ++h) {
      const float before = begin ? scales[h * a.scale_strides[1]] : 0.f;
      float top = 0.f, inv = 0.f;
#pragma unroll 1
      for (int turn = 0; turn < 2; ++turn) {
#pragma unroll 1
        for (int t0 = 0; t0 < count; t0 += per) {
          const int t = min(t0 + first, count - 1), r = r0 + place0 + t;
          uint32_t w[8];
          load16<T, VEC>(src + (t - first) * row_stride + h * head_stride, c0, c1, w);
          Vals x = unpack16<T, HALF>(w);
          f32x2 cs[4], sn[4];
          if (turns) {
            const int pos = a.row_pos ? a.row_pos[r] : int(len + place0 + t);
#pragma unroll
            for (int j = 0; j < 4; ++j) two_phases(pos, a.freq + 8 * li + 2 * j, a.mscale, cs[j], sn[j]);
          }
          norm_turn<T, HALF>(x, weight, norm, lanes, 1.f / D, a.eps, turns, cs, sn);
          if (turn == 0) top = larger(top, x);
          else if (t0 + first < count) put(page + h * hs, t, x, inv);
        }
        if (turn == 0) inv = settle(h, top, before);
      }
    }
    return;
  }
  if (turns) {
#pragma unroll 1
    for (int z = 0; z < PASS; ++z) {
      const int t = z * per + first;
      if (t >= count) break;
      const int r = r0 + place0 + t, pos = a.row_pos ? a.row_pos[r] : int(len + place0 + t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ulonglong2 y;
        two_phases(pos, a.freq + 8 * li + 2 * i, a.mscale, y.x, y.y);
        s_turn[(z * 4 + i) * THREADS + tid] = y;
      }
    }
  }
  for (int h = h0; h < h1; ++h) {
    Vals x[PASS];
#pragma unroll
    for (int z = 0; z < PASS; ++z) x[z] = unpack16<T, HALF>(raw[z]);
    const float before = old;
    if (h + 1 < h1) {  // the next head under this one's work
      fetch(h + 1);
      old = begin ? scales[(h + 1) * a.scale_strides[1]] : 0.f;
    }
    float top = 0.f;
#pragma unroll
    for (int z = 0; z < PASS; ++z) {
      const int t = z * per + first;
      if (z * per >= count) break;  // (a norm's lanes leave together)
      f32x2 cs[4], sn[4];
      if (turns && t < count) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const ulonglong2 y = s_turn[(z * 4 + i) * THREADS + tid];
          cs[i] = y.x;
          sn[i] = y.y;
        }
      }
      norm_turn<T, HALF>(x[z], weight, norm, lanes, 1.f / D, a.eps, turns && t < count, cs, sn);
      if (t < count) top = larger(top, x[z]);
    }
    const float inv = settle(h, top, before);
#pragma unroll
    for (int z = 0; z < PASS; ++z)
      if (z * per + first < count) put(page + h * hs, z * per + first, x[z], inv);
  }
}

// Warp w: row w / warps, the heads of part w % warps.
template <typename T, bool VEC, bool HALF>
__device__ void turn_q(const dspark_paged_append_args& a, int w, int warps) {
  const int lane = threadIdx.x & 31, D = a.D, lanes = D / 16, per = 32 / lanes;
  const int r = w / warps, part = w - r * warps;
  if (r >= a.R) return;
  const int group = lane / lanes, li = lane % lanes;
  const bool turns = li < a.rot / 16, half = turns && HALF;
  const int c0 = half ? 8 * li : 16 * li, c1 = half ? a.rot / 2 + 8 * li : c0 + 8;
  const int step = warps * per;
  const T* src = static_cast<const T*>(a.q) + r * a.q_strides[0];
  T* dst = static_cast<T*>(a.q_out) + r * a.qo_strides[0];
  uint32_t raw[U][8];
  auto fetch = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (h + u * step < a.Hq) load16<T, VEC>(src + (h + u * step) * a.q_strides[1], c0, c1, raw[u]);
  };
  fetch(part * per + group);  // under way while the request is looked for
  int pos = 0;
  const int b = last_at_most(a.B, r, [&](int i) { return first_row(a.cu_rows, i, a.R); });
  const int r0 = first_row(a.cu_rows, b, a.R);
  if (r < r0 || r >= first_row(a.cu_rows, b + 1, a.R)) return;  // a row of no request
  pos = a.row_pos ? a.row_pos[r] : max(a.kv_len[b], 0) + r - r0;
  f32x2 cs[4], sn[4];
  if (turns) {
#pragma unroll
    for (int j = 0; j < 4; ++j) two_phases(pos, a.freq + 8 * li + 2 * j, a.mscale, cs[j], sn[j]);
  }
  const bool norm = a.q_norm;
  uint32_t weight[8];
  if (norm) load16<T, false>(static_cast<const T*>(a.q_norm), c0, c1, weight);
  for (int hb = part * per; hb < a.Hq; hb += U * step) {
    const int h = hb + group;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = h + u * step;
      if (hb + u * step >= a.Hq) break;
      Vals v = unpack16<T, HALF>(raw[u]);
      norm_turn<T, HALF>(v, weight, norm, lanes, 1.f / D, a.eps, turns, cs, sn);
      if (hh >= a.Hq) continue;
      float x[16];
      in_order<HALF>(v, x);
      uint32_t y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = turns || norm ? Elem<T>::pack(x[2 * i], x[2 * i + 1]) : raw[u][i];
      T* p = dst + hh * a.qo_strides[1];
      if (VEC) {
        *reinterpret_cast<uint4*>(p + c0) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(p + c1) = make_uint4(y[4], y[5], y[6], y[7]);
      } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = i < 4 ? c0 + 2 * i : c1 + 2 * (i - 4);
          o[at] = uint16_t(y[i]);
          o[at + 1] = uint16_t(y[i] >> 16);
        }
      }
    }
    if (hb + U * step < a.Hq) fetch(h + U * step);
  }
}

template <typename T, bool VEC, bool HALF, int PASS, int THREADS, int MIN_BLOCKS>
__global__ void __launch_bounds__(THREADS, MIN_BLOCKS) append_kernel(const dspark_paged_append_args a, const int page_blocks, const int groups,
                                                         const int warps, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  if (int(blockIdx.x) < page_blocks)
    append_page<T, VEC, HALF, PASS, THREADS>(a, int(blockIdx.x), groups, status);
  else
    turn_q<T, VEC, HALF>(a, int((blockIdx.x - page_blocks) * (THREADS / 32) + (threadIdx.x >> 5)), warps);
}

template <typename T, bool VEC, bool HALF, int PASS, int THREADS, int MIN_BLOCKS>
static cudaError_t launch_as(const dspark_paged_append_args& a, cudaStream_t s) {
  const int64_t units = int64_t(a.R) / a.page + 2 * int64_t(a.B);
  // groups of heads: as few as leave a round of blocks (a page that is not written ends its block at once)
  const int64_t least = int64_t(MIN_BLOCKS) * sm_count(current_device());
  const int groups = int(std::min<int64_t>(a.Hk, std::max<int64_t>(1, (least + 2 * units - 1) / (2 * units))));
  const int64_t page_blocks = units * groups * 2;
  // warps a row of q: one, unless that leaves less than 16 warps an SM (then as many as take U heads a lane)
  const int sms = sm_count(current_device()), per = 32 / (a.D / 16);
  const int most = (a.Hq + per - 1) / per, want = (16 * sms + a.R - 1) / std::max(a.R, 1);
  const int warps = std::max(1, std::min(want, most));
  const int64_t q_blocks = (int64_t(a.R) * warps + THREADS / 32 - 1) / (THREADS / 32);
  if (page_blocks + q_blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  constexpr int SMEM = PASS * 4 * THREADS * 16;
  auto kernel = append_kernel<T, VEC, HALF, PASS, THREADS, MIN_BLOCKS>;
  const cudaError_t e = configure_once((const void*)kernel, SMEM, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  });
  if (e != cudaSuccess) return e;
  return launch_ex(kernel, dim3(unsigned(page_blocks + q_blocks)), dim3(THREADS), SMEM, s, 1, true, a, int(page_blocks), groups,
                   warps, status_word(current_device()));
}

template <typename T, bool VEC, bool HALF>
static cudaError_t launch_page(const dspark_paged_append_args& a, cudaStream_t s) {
  // Threads by the rows that a page gets on average (a page with more than its block holds is made twice): in registers
  // 64 * 16 values of few rows, else the whole page. 200 requests of 1 to 16 rows 13.2 us with 128 threads, a prompt's
  // 16,389 rows in pages of 64 79 with 256 threads of two rows (4 rows a thread: 94 beside 81, in an earlier form).
  const int64_t rows = std::min<int64_t>(a.page, (int64_t(a.R) + a.B - 1) / a.B), parts = rows * a.D / 16;
  if (parts <= 32) return launch_as<T, VEC, HALF, 1, 64, 10>(a, s);
  if (parts <= 128) return launch_as<T, VEC, HALF, 1, 128, 5>(a, s);
  if (parts <= 256) return launch_as<T, VEC, HALF, 2, 128, 5>(a, s);
  if (parts <= 512) return launch_as<T, VEC, HALF, 2, 256, 2>(a, s);
  return launch_as<T, VEC, HALF, 2, 512, 1>(a, s);
}

template <typename T>
static cudaError_t launch(const dspark_paged_append_args& a, bool vec, cudaStream_t s) {
  const bool half = a.layout == DSPARK_ROPE_HALF;
  if (vec) return half ? launch_page<T, true, true>(a, s) : launch_page<T, true, false>(a, s);
  return half ? launch_page<T, false, true>(a, s) : launch_page<T, false, false>(a, s);
}

}  // namespace paged
}  // namespace dspark

using namespace dspark;

extern "C" int dspark_paged_append(const dspark_paged_append_args* p, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "paged_append: null argument");
  const dspark_paged_append_args& a = *p;
  if (a.R < 0 || a.B < 0 || a.Hq <= 0 || a.Hk <= 0 || a.n_pages < 0 || a.max_pages < 0)
    return fail(DSPARK_ERR_ARG, "paged_append: bad shape (%d rows, %d requests, %d / %d heads, %d pages)", a.R, a.B,
                a.Hq, a.Hk, a.n_pages);
  if (a.dtype != DSPARK_DTYPE_BF16 && a.dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_append: dtype %d (bf16 = 0, fp16 = 1)", a.dtype);
  if (a.layout != DSPARK_ROPE_HALF && a.layout != DSPARK_ROPE_INTERLEAVED)
    return fail(DSPARK_ERR_ARG, "paged_append: layout %d", a.layout);
  if (a.D != 64 && a.D != 128) return fail(DSPARK_ERR_UNSUPPORTED, "paged_append: head_dim %d (64 or 128)", a.D);
  if (a.page != 16 && a.page != 32 && a.page != 64 && a.page != 128)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_append: pages of %d tokens (16, 32, 64 or 128)", a.page);
  if (a.rot <= 0 || a.rot % 16 || a.rot > a.D)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_append: rotary dim %d of %d (a multiple of 16)", a.rot, a.D);
  if (a.B == 0) return DSPARK_OK;
  if (!a.freq || !a.cu_rows || !a.kv_len || (a.max_pages && !a.page_table))
    return fail(DSPARK_ERR_ARG, "paged_append: null pointer");
  if (a.R && (!a.q || !a.q_out || !a.k || !a.v || !a.k_pages || !a.v_pages || !a.k_scale || !a.v_scale))
    return fail(DSPARK_ERR_ARG, "paged_append: null pointer");
  // blocks of one launch read these while another writes the new lengths
  auto apart = [&](const int32_t* x, int64_t n) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(x), out = reinterpret_cast<uintptr_t>(a.len_out);
    return !x || at + n * sizeof(int32_t) <= out || out + a.B * sizeof(int32_t) <= at;
  };
  if (a.len_out && !(apart(a.kv_len, a.B) && apart(a.cu_rows, int64_t(a.B) + 1) && apart(a.row_pos, a.R) &&
                     (a.max_pages == 0 || apart(a.page_table, (a.B - 1) * a.table_stride + a.max_pages))))
    return fail(DSPARK_ERR_ARG, "paged_append: len_out overlaps kv_len, cu_rows, row_pos or page_table");
  bool codes = true;
  for (const void* x : {a.k_pages, a.v_pages}) codes &= reinterpret_cast<uintptr_t>(x) % 16 == 0;
  for (int i = 0; i < 3; ++i) codes &= a.kp_strides[i] % 16 == 0 && a.vp_strides[i] % 16 == 0;
  if (!codes) return fail(DSPARK_ERR_UNSUPPORTED, "paged_append: the pages' rows must be 16-byte aligned");
  // what is written has a place of its own: blocks write pages, heads, keys and values at the same time
  bool own = a.k_pages != a.v_pages && a.k_scale != a.v_scale;
  for (const int64_t* st : {a.kp_strides, a.vp_strides})
    own &= (st[0] || a.n_pages <= 1) && (st[1] || a.Hk == 1) && st[2];
  own &= (a.scale_strides[0] || a.n_pages <= 1) && (a.scale_strides[1] || a.Hk == 1);
  if (a.R && !own) return fail(DSPARK_ERR_ARG, "paged_append: pages or scales share their memory");
  bool vec = true;
  for (const void* x : {a.q, a.k, a.v, (const void*)a.q_out}) vec &= reinterpret_cast<uintptr_t>(x) % 16 == 0;
  for (int i = 0; i < 2; ++i)
    vec &= a.q_strides[i] % 8 == 0 && a.k_strides[i] % 8 == 0 && a.v_strides[i] % 8 == 0 && a.qo_strides[i] % 8 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  DSPARK_CUDA_TRY(a.dtype == DSPARK_DTYPE_BF16 ? paged::launch<bf16>(a, vec, s) : paged::launch<__half>(a, vec, s),
                  "paged_append");
  return DSPARK_OK;
}
