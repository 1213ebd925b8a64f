// Attention over pages of 8-bit values for blocks of many rows (verify blocks, prompts' chunks), on the 5th-generation
// tensor cores. The formulas, the cache and the shares are paged_attn.cu's; here an item is up to 256 rows of one
// (request, kv head).
//
// Block (one an SM): two slots of 128 rows (TMEM lanes), each with a softmax warpgroup, a score tile S (TMEM, overwritten
// by the 16-bit weights P) and an output accumulator O (TMEM).
//  * items of more than 128 rows: the slots are the two halves of the rows and share each K/V tile;
//  * items of up to 128 rows: the slots take the even and the odd key tiles and are joined at the segment's end.
// Either way one slot's softmax runs under the other slot's products.
//  * One warp asks for the codes' tiles by TMA, a box a page (ids read two windows of four tiles ahead), 128 keys x D. Four
//    converting warps write them as fp16, which holds every e4m3 value, into the ring that the products read: 128-byte
//    swizzle, K as it is multiplied (K-major) and V as it lies (N-major). A row is converted once for up to 256 rows of
//    q; neither scale is multiplied in. Beside a K tile go its 16-key groups' factors.
//  * One thread issues the products: S = Q K^T (both from shared memory), O += P V (P from tensor memory).
//  * A thread of a softmax warpgroup owns a row: no shuffles. It writes the row's q as fp16 (bf16: scaled by a power of two,
//    exact). x = f s + log2(vs), f = log2(e) scale 2^e ks, of each group;
//    the maximum in use is only raised when a tile exceeds it by more than 2^8; weights are 2^7 times as large.
//
// Rounding: weights are rounded to fp16 for the product with V (their sum is not); scores, maxima, sums and O are fp32.
//
// Bound: softmax and products in turn (two chunks of 509 rows over 16k keys, 64/8 heads of 128: 515 to 550 us in a graph of such
// calls, 0.6 of the products' measured rate, 2.06 us a 256 x 128 tile, 562 to 576 in calls one by one); for slots of few rows
// the latency of the four converting warps (24 blocks of 1 to 16 rows over 256 to 16k keys, 32/8 heads: 93 us, about 1.3 a tile
// of K and V, with no unit above a third of its rate).
#include <algorithm>

#include "host_common.h"
#include "paged_share.cuh"
#include "tcgen05.cuh"

namespace dspark {
namespace paged {
namespace wide {

constexpr int ROWS = 128;            // rows a slot
constexpr int RB = 2 * ROWS;         // rows an item
constexpr int NTHR = 512;            // two softmax warpgroups, one of the products, loads and segments, one that converts
constexpr int WARP_MMA = 8, WARP_LOAD = 9, WARP_PREP = 10, WARP_CONV = 12;
// Cost of a segment, in tiles of up to 128 rows. Mean of 12 mixes (1 to 60 requests of 16 to 509 rows over 3k to 30k
// keys), us: 4 121.5, 7 117.9, 10 118.5, 14 121.1, 20 124.9.
constexpr int SEG = 7;
constexpr int NB = 3;                // tiles in the ring
constexpr int NC = 3;                // tiles of codes on their way or waiting to be converted
constexpr int NSC = 8;               // tiles whose factors are kept: K of tile t + 5 is asked for after V of tile t is read
                                     // (it is NB + NC loads behind it)

template <int D>
struct Lay {
  static constexpr int TILE = BN * D * 2;         // a K or V tile (and a slot's Q)
  static constexpr int HALF = BN * 128;           // 64 values of 128 rows, 128-byte swizzled
  static constexpr int CODES = BN * D;            // a K or V tile's codes
  static constexpr int Q = 0;
  static constexpr int RING = 2 * TILE;
  static constexpr int STAGE = RING + NB * TILE;
  static constexpr int ML = STAGE + NC * CODES;       // [slot][row] (m, l) at the segment's end
  static constexpr int RF = ML + 2 * ROWS * 8;        // [row] the rows' powers of two, for the other slot
  static constexpr int SC = RF + ROWS * 4;          // [tile % NSC][16-key group] (ks, log2 vs, 1 / vs)
  static constexpr int FLAG = SC + NSC * 8 * 16;
  static constexpr int SEGS = FLAG + 16;              // two segments for the softmax threads
  static constexpr int NOTE = SEGS + 2 * 64;          // what a tile of codes is (Note)
  static constexpr int BARS = NOTE + NC * 8;
  static constexpr int NBAR = 2 * NB + 2 * NC + 2 * 7 + NSC + 1;
  static constexpr int MISC = BARS + NBAR * 8;        // tensor memory's address; 17 pairs of find_share
  static constexpr int TOTAL = MISC + 8 + 17 * 8;
  static_assert(TOTAL <= 232448, "shared memory of one SM");
  static_assert(CODES % 1024 == 0 && BARS % 8 == 0, "alignment");
};

__device__ __forceinline__ void st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void ld_x32(uint32_t taddr, float* d) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
      "[%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) d[i] = __uint_as_float(r[i]);
}

// D[tmem] (+)= A[smem] . B[smem]^T
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 128-byte-swizzled operand: K-major (lbo unused, 8-row groups 1024 bytes apart) or MN-major (lbo between 64-value
// blocks of MN, 8-row groups of K 1024 bytes apart). Only the low word (address, lbo) varies.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return ((addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}
__device__ __forceinline__ uint64_t desc_sw128(uint32_t lo) {
  constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // sbo, version, 128-byte swizzle
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(HI));
  return d;
}

__device__ __forceinline__ void named_sync(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}

// named_sync that tells all its threads whether `ok` held in every one of them.
__device__ __forceinline__ bool named_all(int id, int n, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(ok)), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}

// kind: 0 K, 1 V, - segment: V with keys that not every row sees (its NaN codes are taken out), 2: no more tiles; left: rows
// that are keys.
struct Note {
  int kind, left;
};

// A segment as the walking warp hands it to the softmax threads.
struct Handed {
  Segment s;
  int more;
};
static_assert(sizeof(Handed) <= 64, "Lay::SEGS");

__device__ __forceinline__ bool is_pair(const Segment& s) { return s.live > ROWS; }

// Keys that the item's first row sees, and with it all of them.
__device__ __forceinline__ int seen_by_all(const dspark_paged_attn_args& a, const Segment& s) {
  return a.causal ? min(s.len, s.before + s.row_base / (a.Hq / a.Hk) + 1) : s.len;
}

// Load u of a segment of n tiles, in the order that the products take them: K0 V0 K1 V1 .. (pair) or K0 K1 V0 K2 V1 ..
// (tiles alternate between the slots). Returns the tile; `value`: V.
__device__ __forceinline__ int load_of(bool pair, int u, int n, bool& value) {
  if (pair) {
    value = u & 1;
    return u >> 1;
  }
  if (u == 2 * n - 1) {
    value = true;
    return n - 1;
  }
  value = u > 0 && !(u & 1);
  return value ? (u - 2) >> 1 : (u + 1) >> 1;
}

// Use of the ring (within the segment) by the V tile of tile t.
__device__ __forceinline__ int v_use(bool pair, int t, int n) {
  return pair ? 2 * t + 1 : t == n - 1 ? 2 * n - 1 : 2 * t + 2;
}

// A group's factor, 1e-35 at least (of a negative rf too): -inf stays that, and NaN.
__device__ __forceinline__ float factor_of(float rf, float ks) {
  const float f = rf * ks;
  return f < 1e-35f ? 1e-35f : f;
}

// The NaN codes that were taken out of the segment's V tiles, added to what a row that sees them has stored (`out`: the
// output, or `part`: the fp32 part). They are taken out of whole tiles, those that not all rows of the item see whole: two or
// three, however many rows the request has.
template <typename T>
__device__ __noinline__ void add_hidden(const dspark_paged_attn_args& a, const Segment& s, int lim, int d0, int d1, T* out,
                                        float* part) {
  const int k0 = max(s.t0 * BN, max(seen_by_all(a, s), 0) / BN * BN), k1 = min(min(s.t1 * BN, s.len), lim);
  for (int k = k0; k < k1; ++k) {
    const int id = a.page_table[int64_t(s.b) * a.table_stride + k / a.page];
    if (id < 0 || id >= a.n_pages) continue;
    const int64_t sc = id * a.scale_strides[0] + s.h * a.scale_strides[1];
    if (!(a.k_scale[sc] > 0.f && a.v_scale[sc] > 0.f)) continue;
    const uint8_t* v = static_cast<const uint8_t*>(a.v_pages) + id * a.vp_strides[0] + s.h * a.vp_strides[1] +
                       (k % a.page) * a.vp_strides[2];
    for (int d = d0; d < d1; ++d) {
      if ((v[d] & 0x7f) != 0x7f) continue;
      if (part) part[d * RB] = NAN;
      else out[d] = Elem<T>::from_f(NAN);
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(NTHR, 1) attn_kernel(const __grid_constant__ CUtensorMap kmap,
                                                       const __grid_constant__ CUtensorMap vmap,
                                                       const dspark_paged_attn_args a, const float c_log2,
                                                       const uint32_t q_sign, int* status) {
  typedef Lay<D> L;
  constexpr uint32_t ID_QK = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(ROWS >> 4) << 24);  // fp16, fp32 sums
  constexpr uint32_t ID_PV = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(ROWS >> 4) << 24);
  constexpr uint32_t O_COL = 256;
  constexpr float LIFT = 7.f, SLACK = 8.f;  // weights are at most 2^15
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + L::RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty = full + NB;
  uint64_t* c_full = empty + NB;
  uint64_t* c_empty = c_full + NC;
  uint64_t* q_full = c_empty + NC;
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* p_part = p_full + 2;
  uint64_t* o_full = p_part + 2;
  uint64_t* seg_full = o_full + 2;
  uint64_t* seg_empty = seg_full + 2;
  uint64_t* sc_full = seg_empty + 2;
  uint64_t* fin = sc_full + NSC;
  float2* ml = reinterpret_cast<float2*>(smem + L::ML);
  float* rowf = reinterpret_cast<float*>(smem + L::RF);
  float4* factors = reinterpret_cast<float4*>(smem + L::SC);
  int* flag = reinterpret_cast<int*>(smem + L::FLAG);
  Note* notes = reinterpret_cast<Note*>(smem + L::NOTE);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  uint2* pairs = reinterpret_cast<uint2*>(smem + L::MISC + 8);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles need it; never seen without static arrays
    pdl_wait();
    if (tid == 0) {
      report_error(status, kErrAlign);
      static_cast<Cut*>(a.workspace)[blockIdx.x] = Cut{0, 0, 0, 0, 0, {0, 0, 0}};
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(&full[i], 4);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {  // p_*, q_full and seg_empty count warps
      mbar_init(&q_full[i], 4);
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], 8);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_part[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) flag[i] = 0;
    for (int i = 0; i < NC; ++i) {
      mbar_init(&c_full[i], 1);
      mbar_init(&c_empty[i], 4);
    }
    for (int i = 0; i < NSC; ++i) mbar_init(&sc_full[i], 1);
    mbar_init(fin, 1);
    fence_mbar_init();
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  if (warp == WARP_MMA) tcg::tmem_alloc(tmem_slot, 512);
  pdl_launch_dependents();
  pdl_wait();
  Plan<RB> plan{a, 0};
  Walker<RB> wk;
  const Deal deal = find_share<RB, NTHR>(plan, SEG, wk, pairs, pairs + 16);
  tcg::tc_fence_before();
  __syncthreads();
  tcg::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int G = a.Hq / a.Hk;
  bool ok = true;

  if (warp < WARP_MMA) {
    // ------------------------------------------- softmax: slot = warpgroup, row = TMEM lane
    // (registers: 256 * 184 + 256 * 72 = 512 * 128, what the block was launched with)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    const int slot = warp >> 2, row = tid & 127;
    const uint32_t t_s = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(slot * 128);
    const uint32_t t_o = t_s + O_COL;
    uint32_t n_s = 0;              // completed phases of s_full
    uint32_t n_o0 = 0, n_o1 = 0;   // of o_full
    int use0 = 0, tiles0 = 0;      // ring uses and tiles before this segment
    auto arrive = [&](uint64_t* bar) {  // this warp's stores to tensor memory are done
      tcg::tmem_wait_st();
      tcg::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // flag[seg & 3] == seg: a hidden NaN in segment `seg`. The converting warps are two segments ahead at most: beyond the
    // first product of the next one, which needs no weights, they have room for NB tiles.
    for (int seg = 1;; ++seg) {
      const int hand = (seg - 1) & 1;
      const Handed& sh = *reinterpret_cast<const Handed*>(smem + L::SEGS + 64 * hand);
      if (ok) ok = mbar_wait(&seg_full[hand], uint32_t((seg - 1) >> 1) & 1u, status, kErrWaitPeer);
      // after a wait that ran out all leave together: the barriers below count all of them
      ok = named_all(3, 256, ok);
      if (!ok || !sh.more) break;
      const Segment& s = sh.s;
      const int n = s.t1 - s.t0;
      const bool pair = is_pair(s);
      const int steps = pair ? n : (n - slot + 1) >> 1;
      const int my = s.row_base + (pair ? slot * ROWS : 0) + row;  // (node, head) row of this thread
      const bool alive = my < s.rows * G;
      const bool warp_alive = s.row_base + (pair ? slot * ROWS : 0) + (warp & 3) * 32 < s.rows * G;
      const int place = alive ? my / G : 0;
      const int lim = a.causal ? min(s.len, s.before + place + 1) : s.len;  // keys that the row sees
      const int edge0 = seen_by_all(a, s) - BN;  // later: hidden keys
      // ---- Q as fp16, a row a thread (the first slot's for both where there are up to 128). The products that read the
      // last segment's are done: their O has been waited for.
      float rf = 1.f;
      if (n > 0 && (pair || slot == 0)) {
        if (alive) {
          const T* q = static_cast<const T*>(a.q) + int64_t(s.r0 + place) * a.q_strides[0] +
                       (s.h * G + my - place * G) * a.q_strides[1];
          uint4 v[D / 8];
#pragma unroll
          for (int c = 0; c < D / 8; ++c) v[c] = ldcg_v4(q + 8 * c);
          constexpr uint32_t SHIFT = std::is_same<T, bf16>::value ? 7 : 10, ONES = std::is_same<T, bf16>::value ? 0xff : 0x1f;
          uint32_t e = 0;  // the largest exponent; all ones: infinite or NaN (its factor is negative then, its q zeros)
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint32_t* y = &v[c].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) e = max(e, max((y[i] >> SHIFT) & ONES, (y[i] >> (SHIFT + 16)) & ONES));
          }
          float inv = 1.f;
          if (std::is_same<T, bf16>::value) {
            const int up = int(e) - 141;  // values below 2^15
            inv = pow2(max(min(-up, 126), -126));
            rf = pow2(max(min(up, 126), -126));
          }
          rf = e == ONES ? -1.f : rf * c_log2;
          uint8_t* dst = smem + L::Q + slot * L::TILE + row * 128;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            uint32_t* y = &v[c].x;
            if (std::is_same<T, bf16>::value) {
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = Elem<__half>::pack(bf16_lo(y[i]) * inv, bf16_hi(y[i]) * inv);
            }
            if (e == ONES) y[0] = y[1] = y[2] = y[3] = 0u;
            *reinterpret_cast<uint4*>(dst + (c >> 3) * L::HALF + (((c & 7) ^ (row & 7)) << 4)) =
                make_uint4(y[0] ^ q_sign, y[1] ^ q_sign, y[2] ^ q_sign, y[3] ^ q_sign);
          }
        }
        if (!pair) rowf[row] = rf;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[slot]);
      }
      if (!pair) {
        named_sync(3, 256);
        rf = rowf[row];
      }
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < steps; ++j) {
        const int t = pair ? j : 2 * j + slot, k0 = (s.t0 + t) * BN, tile = tiles0 + t;
        const bool edge = k0 > edge0;
        if (ok) ok = mbar_wait(&sc_full[tile % NSC], uint32_t(tile / NSC) & 1u, status, kErrWaitKV);
        if (ok) ok = mbar_wait(&s_full[slot], n_s & 1, status, kErrWaitMma);
        ++n_s;
        tcg::tc_fence_after();
        if (edge && (slot == 0 || !pair)) {
          // NaN codes have been taken out of V and noted. Not before the scores: they are made of K(t), and the previous use
          // of V(t)'s buffer was loaded before K(t) or is K(t) itself, so the parity waited for here cannot
          // be that of an earlier, still missing load
          const int g = use0 + v_use(pair, t, n);
          if (ok) ok = mbar_wait(&full[g % NB], uint32_t(g / NB) & 1u, status, kErrWaitKV);
        }
        if (warp_alive) {
          float x[128];
#pragma unroll
          for (int i = 0; i < 4; ++i) ld_x32(t_s + uint32_t(32 * i), x + 32 * i);
          const float4* fa = factors + (tile % NSC) * 8;
          tcg::tmem_wait_ld();
          if (edge) {
            const int left = lim - k0;
#pragma unroll
            for (int i = 0; i < 128; ++i) x[i] = i < left ? x[i] : -INFINITY;
          }
          // (the factors are positive: a group's largest score is that of its largest product)
          float mt = -INFINITY;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float* y = x + 16 * g;
            const float mg = max3(max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), max3(y[6], y[7], y[8])),
                                  max3(y[9], y[10], y[11]), max3(max3(y[12], y[13], y[14]), y[15], y[15]));
            mt = max3(mt, fmaf(mg, factor_of(rf, fa[g].x), fa[g].y), mt);
          }
          if (!(mt < INFINITY)) m = NAN;  // a visible score of +inf or NaN: the row is NaN
          const bool up = mt - m > SLACK;
          if (__any_sync(0xffffffffu, up)) {
            const float mn = up ? mt : m;
            const float f = up ? ex2(m - mn) : 1.f;
            m = mn;
            l *= f;
            if (j > 0) {
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                float o[16];
                tcg::tmem_ld16(t_o + uint32_t(16 * i), o);
                tcg::tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= f;
                st_x16(t_o + uint32_t(16 * i), reinterpret_cast<const uint32_t*>(o));
              }
            }
          }
          const float ref = LIFT - (m == -INFINITY ? 0.f : m);
          // pair by pair, sums and packing LAG pairs behind the exponentials: the special-function unit (8 clocks a warp
          // instruction) then never waits for them
          constexpr int LAG = 4;
          f32x2 e[64], sum = pack2(0.f, 0.f), f2 = sum, l2 = sum;
          uint32_t p[64];
#pragma unroll
          for (int i = 0; i < 64 + LAG; ++i) {
            if (i < 64) {
              if ((i & 7) == 0) {
                const float4 y = fa[i >> 3];
                const float f = factor_of(rf, y.x), lv = y.y + ref;
                f2 = pack2(f, f);
                l2 = pack2(lv, lv);
              }
              float e0, e1;
              unpack2(fma2(pack2(x[2 * i], x[2 * i + 1]), f2, l2), e0, e1);
              e[i] = pack2(ex2(e0), ex2(e1));
            }
            const int z = i - LAG;
            if (z >= 0) {
              float e0, e1;
              unpack2(e[z], e0, e1);
              sum = (z & 7) == 0 ? e[z] : add2(sum, e[z]);
              p[z] = Elem<__half>::pack(e0, e1);
              if ((z & 7) == 7) {
                unpack2(sum, e0, e1);
                l = fmaf(e0 + e1, fa[z >> 3].z, l);
              }
              if ((z & 15) == 15) st_x16(t_s + uint32_t(z - 15), p + z - 15);
              if (z == 47) arrive(&p_part[slot]);  // three quarters' products may start
            }
          }
        } else {
          arrive(&p_part[slot]);
        }
        arrive(&p_full[slot]);
      }
      use0 += 2 * n;
      tiles0 += n;
      // ---- end of the segment: with one row block, both slots' O of half of the values
      const bool both = !pair && n > 1;
      if (n > 0) {
        if (ok && steps > 0) ok = mbar_wait(&o_full[slot], (slot ? n_o1 : n_o0) & 1, status, kErrWaitMma);
        if (ok && both) ok = mbar_wait(&o_full[slot ^ 1], (slot ? n_o0 : n_o1) & 1, status, kErrWaitMma);
        if (!pair && slot == 1 && n == 1 && ok) ok = mbar_wait(&o_full[0], n_o0 & 1, status, kErrWaitMma);
        ++n_o0;
        n_o1 += pair || n > 1;
      }
      tcg::tc_fence_after();
      const bool whole = s.parts == 1;
      float f0 = 1.f, f1 = 0.f;
      if (!pair) {
        ml[slot * ROWS + row] = make_float2(m, l);
        named_sync(3, 256);
        const float2 a0 = ml[row], a1 = ml[ROWS + row];
        // (a NaN in either is the row's: fmaxf would lose it)
        const float mn = a0.x != a0.x || a1.x != a1.x ? NAN : fmaxf(a0.x, a1.x), ref = mn == -INFINITY ? 0.f : mn;
        f0 = ex2(a0.x - ref);
        f1 = ex2(a1.x - ref);
        l = a0.y * f0 + a1.y * f1;
        m = mn;
      }
      if (rf < 0.f && l > 0.f) l = NAN;  // an infinite or NaN q: NaN whatever the codes are, where the row sees a key
      const bool hidden = *reinterpret_cast<volatile int*>(&flag[seg & 3]) == seg;
      if (warp_alive) {
        const int hq = s.h * G + my - place * G;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int prow = (pair ? slot * ROWS : 0) + row;
        float* pp = whole ? nullptr : part_of<D, RB>(a.workspace, blockIdx.x, int(blockIdx.x) == s.first);
        // 32-value chunks: all of the slot's own, or every second one of both slots'
        const int i0 = pair ? 0 : slot * (D / 64), i1 = pair ? D / 32 : i0 + D / 64;
        const uint32_t t_0 = pair ? t_o : tmem + (uint32_t((warp & 3) * 32) << 16) + O_COL;
        T* out = static_cast<T*>(a.out) + int64_t(s.r0 + place) * a.o_strides[0] + hq * a.o_strides[1];
        if (!whole && alive && (pair || slot == 0)) pp[RB * D + prow] = l == 0.f ? -INFINITY : m + lg2(l);
        if (n > 0) {
#pragma unroll 1
          for (int i = i0; i < i1; ++i) {
            float o[32];
            ld_x32(t_0 + uint32_t(32 * i), o);
            tcg::tmem_wait_ld();
            if (both) {
              float o1[32];
              ld_x32(t_0 + 128u + uint32_t(32 * i), o1);
              tcg::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = o[e] * f0 + o1[e] * f1;
            }
            if (alive && !whole) {
#pragma unroll
              for (int e = 0; e < 32; ++e) pp[(32 * i + e) * RB + prow] = l == 0.f ? 0.f : o[e] * inv;
            } else if (alive) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint4 v;
                v.x = Elem<T>::pack(o[e] * inv, o[e + 1] * inv);
                v.y = Elem<T>::pack(o[e + 2] * inv, o[e + 3] * inv);
                v.z = Elem<T>::pack(o[e + 4] * inv, o[e + 5] * inv);
                v.w = Elem<T>::pack(o[e + 6] * inv, o[e + 7] * inv);
                *reinterpret_cast<uint4*>(out + 32 * i + e) = l == 0.f ? make_uint4(0u, 0u, 0u, 0u) : v;
              }
            }
          }
          if (hidden && alive) add_hidden<T>(a, s, lim, 32 * i0, 32 * i1, out, whole ? nullptr : pp + prow);
        }
      }
      tcg::tc_fence_before();
      if (!pair) named_sync(3, 256);  // both have read both: the next weights may be given
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[hand]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    Segment s{};
    if (warp >= WARP_CONV) {
      // -------------------------------------------------------------- codes to fp16 tiles
      constexpr int CH = D / 16, RPI = 32 / CH, ROUNDS = 32 / RPI;  // 16-byte chunks a row, rows a round, rounds a warp
      // A lane's chunk and row of a round. D = 128: eight lanes that go together have four chunks of one 64-value half of rows
      // r and r ^ 5, whose places differ in both swizzles: no two on one bank, reading or writing.
      const int w = warp - WARP_CONV, c = D == 128 ? (lane & 3) + (lane >> 4) * 4 : lane & 3;
      auto row_of = [&](int z) {
        const int q = (lane >> 2) & 3;
        return w * 32 + (D == 128 ? 8 * (z >> 1) + ((2 * (z & 1) + (q >> 1)) ^ ((q & 1) * 5)) : z * RPI + (lane >> 2));
      };
      int st = 0, st_phase = 0, x = 0, use = 0;
      while (true) {
        ok = mbar_wait(&c_full[st], uint32_t(st_phase), status, kErrWaitKV);
        if (!__all_sync(0xffffffffu, ok)) break;
        const Note note = notes[st];
        if (note.kind == 2) break;  // no more
        if (use > 0) {
          ok = mbar_wait(&empty[x], uint32_t(use - 1) & 1u, status, kErrWaitKVEmpty);
          if (!__all_sync(0xffffffffu, ok)) break;
        }
        const uint8_t* codes = smem + L::STAGE + st * L::CODES;
        uint8_t* base = ring + x * L::TILE + (c >> 2) * L::HALF;
        auto get = [&](int z) {
          const int row = row_of(z), sw = D == 128 ? row & 7 : (row >> 1) & 3;
          return *reinterpret_cast<const uint4*>(codes + row * D + ((c ^ sw) << 4));
        };
        auto put = [&](int z, uint4 v) {
          const uint4 h0 = make_uint4(e4m3_to_f16(v.x), e4m3_to_f16_hi(v.x), e4m3_to_f16(v.y), e4m3_to_f16_hi(v.y));
          const uint4 h1 = make_uint4(e4m3_to_f16(v.z), e4m3_to_f16_hi(v.z), e4m3_to_f16(v.w), e4m3_to_f16_hi(v.w));
          const int row = row_of(z), at = (c & 3) * 2, sw = row & 7;
          *reinterpret_cast<uint4*>(base + row * 128 + ((at ^ sw) << 4)) = h0;
          *reinterpret_cast<uint4*>(base + row * 128 + (((at + 1) ^ sw) << 4)) = h1;
        };
        if (note.kind >= 0 && note.left >= BN) {
#pragma unroll
          for (int z0 = 0; z0 < ROUNDS; z0 += 4) {  // four in flight
            uint4 v[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) v[z] = get(z0 + z);
#pragma unroll
            for (int z = 0; z < 4; ++z) put(z0 + z, v[z]);
          }
        } else {
#pragma unroll 1
          for (int z = 0; z < ROUNDS; ++z) {
            uint4 v = get(z);
            if (row_of(z) >= note.left) v = make_uint4(0u, 0u, 0u, 0u);  // no key: whatever the page holds there
            if (note.kind < 0) {
              uint32_t* y = &v.x;
              uint32_t any = 0;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t nan = (((y[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                any |= nan;
                y[k] &= ~(nan * 0xffu);
              }
              if (any) *reinterpret_cast<volatile int*>(&flag[(-note.kind) & 3]) = -note.kind;
            }
            put(z, v);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&c_empty[st]);
          mbar_arrive(&full[x]);
        }
        if (++st == NC) {
          st = 0;
          st_phase ^= 1;
        }
        if (++x == NB) {
          x = 0;
          ++use;
        }
      }
      __syncwarp();
    } else if (warp == WARP_LOAD) {
      // -------------------------------------------------------------- codes, by TMA from the pages
      // A lane has one 16-key group of four tiles (a window): page ids are read two windows ahead, scales one.
      const int shift = 31 - __clz(a.page), boxes = BN >> shift;
      int load = 0, tiles0 = 0, seg = 0;
      auto wait_free = [&]() {  // the next stage
        const int st = load % NC;
        if (load >= NC && ok) ok = mbar_wait(&c_empty[st], uint32_t(load / NC - 1) & 1u, status, kErrWaitKVEmpty);
        ok = __all_sync(0xffffffffu, ok);
        return st;
      };
      while (ok && wk.next(plan, deal, s)) {
        ++seg;
        const int n = s.t1 - s.t0;
        const bool pair = is_pair(s);
        const int edge0 = seen_by_all(a, s) - BN;
        const int32_t* table = a.page_table + int64_t(s.b) * a.table_stride;
        auto page_ids = [&](int window) {
          int id = -1;
          const int t = window * 4 + (lane >> 3), key = (s.t0 + t) * BN + (lane & 7) * 16;
          if (t < n && key < s.len) {
            id = table[key >> shift];
            if (id < 0 || id >= a.n_pages) {
              report_error(status, kErrAttnPage);
              id = -1;
            }
          }
          return id;
        };
        auto scales = [&](int id) {
          float2 y = make_float2(0.f, 0.f);
          if (id >= 0) {
            const int64_t at = id * a.scale_strides[0] + s.h * a.scale_strides[1];
            y = make_float2(a.k_scale[at], a.v_scale[at]);
          }
          return y;
        };
        // ids: of the window in work (-1: not seen), `before` of the one before (V is up to two tiles behind K)
        int window = -1, ids = -1, before = -1, ids1 = n > 0 ? page_ids(0) : -1, ids2 = n > 0 ? page_ids(1) : -1;
        float2 sc = make_float2(0.f, 0.f), sc1 = scales(ids1);
        for (int u = 0; u < 2 * n && ok; ++u) {
          bool value;
          const int t = load_of(pair, u, n, value);
          if (!value && (t >> 2) != window) {
            window = t >> 2;
            before = ids;
            sc = sc1;
            ids = sc.x > 0.f && sc.y > 0.f ? ids1 : -1;  // a page without a positive scale is not seen
            ids1 = ids2;
            sc1 = scales(ids1);
            ids2 = page_ids(window + 2);
          }
          const int st = wait_free();
          if (!ok) break;
          // lane i: the page of the tile's i-th box
          const int id = __shfl_sync(0xffffffffu, (t >> 2) != window ? before : ids, (t & 3) * 8 + ((lane << (shift - 4)) & 7));
          const int key0 = (s.t0 + t) * BN;
          if (!value && (lane >> 3) == (t & 3))
            factors[((tiles0 + t) % NSC) * 8 + (lane & 7)] =
                ids >= 0 ? make_float4(sc.x, lg2(sc.y), 1.f / sc.y, 0.f) : make_float4(1.f, -INFINITY, 0.f, 0.f);
          if (lane == 0) {
            notes[st] = Note{!value ? 0 : key0 > edge0 ? -seg : 1, s.len - key0};
            mbar_arrive_expect_tx(&c_full[st], L::CODES);
          }
          __syncwarp();
          if (lane == 0 && !value) mbar_arrive(&sc_full[(tiles0 + t) % NSC]);
          if (lane < boxes)  // a page that is not seen: past the last one, where the copy writes zeros
            tma_load_4d(smem + L::STAGE + st * L::CODES + lane * a.page * D, value ? &vmap : &kmap, &c_full[st], 0, 0, s.h,
                        id < 0 ? a.n_pages : id);
          ++load;
        }
        tiles0 += n;
      }
      // no copy may still be in flight when the block exits (under the default limit, whatever is set); before the
      // end is told, which is one more phase of its stage
      if (lane == 0)
        for (int i = max(0, load - NC); i < load; ++i) mbar_wait(&c_full[i % NC], uint32_t(i / NC) & 1u, nullptr, 0);
      __syncwarp();
      const int end = wait_free();
      if (ok && lane == 0) {
        notes[end] = Note{2, 0};
        mbar_arrive(&c_full[end]);
      }
      __syncwarp();
    } else if (warp == WARP_PREP) {
      // -------------------------------------------------------------- segments, one ahead
      Cut cut{0, 0, 0, 0, 0, {0, 0, 0}};
      for (int k = 0;; ++k) {
        const bool more = __all_sync(0xffffffffu, ok) && wk.next(plan, deal, s);
        const int hand = k & 1;
        if (k >= 2 && ok) ok = mbar_wait(&seg_empty[hand], uint32_t((k >> 1) - 1) & 1u, status, kErrWaitPeer);
        if (lane == 0) {
          Handed* h = reinterpret_cast<Handed*>(smem + L::SEGS + 64 * hand);
          if (more) {
            h->s = s;
            if (s.parts > 1 && int(blockIdx.x) == s.first) cut = Cut{s.parts, s.r0, s.live, s.row_base, s.h, {0, 0, 0}};
          }
          h->more = more;
          mbar_arrive(&seg_full[hand]);
        }
        if (!more) break;
      }
      if (lane == 0) static_cast<Cut*>(a.workspace)[blockIdx.x] = cut;
      __syncwarp();
    } else if (warp == WARP_MMA) {
      // -------------------------------------------------------------- products
      // The whole warp walks and waits; one lane issues.
      const uint32_t leader = tcg::elect_one() ? 1u : 0u;
      const uint32_t q_lo = desc_lo(smem_u32(smem + L::Q), 16), ring_a = smem_u32(ring);
      int x_ring = 0, g_phase = 0;
      uint32_t n_q[2] = {0, 0}, n_p[2] = {0, 0};
      bool issued = false;
      auto take = [&]() {  // the next ring buffer, filled
        const int x = x_ring;
        if (ok) ok = mbar_wait(&full[x], uint32_t(g_phase), status, kErrWaitKV);
        tcg::tc_fence_after();
        if (++x_ring == NB) {
          x_ring = 0;
          g_phase ^= 1;
        }
        return x;
      };
      auto commit = [&](uint64_t* bar) {
        if (leader) tcg::umma_commit(bar);
      };
      auto scores = [&](int slot, int qt, int x) {  // qt: the tile of Q
        if (!ok) return;
        const uint32_t qd = q_lo + uint32_t(qt) * (L::TILE >> 4);
        const uint32_t kd = desc_lo(ring_a + uint32_t(x) * L::TILE, 16);
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t((k >> 2) * (L::HALF >> 4) + (k & 3) * 2);
            umma_ss(tmem + uint32_t(slot * 128), desc_sw128(qd + off), desc_sw128(kd + off), ID_QK, k ? 1u : 0u);
          }
          tcg::umma_commit(&s_full[slot]);
        }
        issued = true;
      };
      auto values = [&](int slot, int x, bool first) {
        const uint32_t vd = desc_lo(ring_a + uint32_t(x) * L::TILE, L::HALF);
        const uint32_t ph = n_p[slot]++ & 1u;
        const uint32_t d = tmem + O_COL + uint32_t(slot * 128), p = tmem + uint32_t(slot * 128);
        if (ok) ok = mbar_wait(&p_part[slot], ph, status, kErrWaitMma);
        if (!ok) return;
        tcg::tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = 0; k < 6; ++k)
            tcg::umma_ts(d, p + uint32_t(8 * k), desc_sw128(vd + uint32_t(k * (2048 >> 4))), ID_PV, first && k == 0 ? 0u : 1u);
        }
        ok = mbar_wait(&p_full[slot], ph, status, kErrWaitMma);
        if (!ok) return;
        tcg::tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = 6; k < BN / 16; ++k)
            tcg::umma_ts(d, p + uint32_t(8 * k), desc_sw128(vd + uint32_t(k * (2048 >> 4))), ID_PV, 1u);
        }
      };
      auto release = [&](int x) {
        if (ok) commit(&empty[x]);
      };
      auto q_ready = [&](int slot) {
        if (ok) ok = mbar_wait(&q_full[slot], n_q[slot]++ & 1u, status, kErrWaitMma);
        tcg::tc_fence_after();
      };
      while (__all_sync(0xffffffffu, ok) && wk.next(plan, deal, s)) {
        const int n = __shfl_sync(0xffffffffu, s.t1 - s.t0, 0);
        const bool pair = __shfl_sync(0xffffffffu, int(is_pair(s)), 0);
        if (n <= 0) continue;
        if (pair) {
          int x = take();
          q_ready(0);
          scores(0, 0, x);
          q_ready(1);
          scores(1, 1, x);
          release(x);
          for (int t = 0; t < n; ++t) {
            const int v = take();
            const bool more = t + 1 < n;
            values(0, v, t == 0);
            if (more) {
              x = take();
              scores(0, 0, x);
            } else if (ok) {
              commit(&o_full[0]);
            }
            values(1, v, t == 0);
            release(v);
            if (more) {
              scores(1, 1, x);
              release(x);
            } else if (ok) {
              commit(&o_full[1]);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
          }
        } else {
          for (int z = 0; z < min(n, 2); ++z) {
            const int x = take();
            if (z == 0) q_ready(0);
            scores(z, 0, x);
            release(x);
          }
          for (int t = 0; t < n; ++t) {
            const int v = take(), z = t & 1;
            values(z, v, t < 2);
            release(v);
            if (t + 2 < n) {
              const int x = take();
              scores(z, 0, x);
              release(x);
            } else if (ok) {
              commit(&o_full[z]);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
          }
        }
      }
      if (issued) {  // nothing may write tensor memory after the block releases it
        commit(fin);
        mbar_wait(fin, 0, nullptr, 0);  // (under the default limit)
      }
      __syncwarp();
    }
  }
  tcg::tc_fence_before();
  __syncthreads();
  tcg::tc_fence_after();
  if (warp == WARP_MMA) tcg::tmem_dealloc(tmem, 512);
}

// A block: 32 rows (lanes) of a cut item, a warp D / 4 of their values; the parts in order. The parts' values lie with
// the row innermost, as a warp of 32 rows writes them.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_wide_kernel(const dspark_paged_attn_args a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int N = D / 4, HELD = 4;  // values a thread, parts under way together
  const int cta = blockIdx.x, r = blockIdx.y * 32 + (threadIdx.x & 31), d0 = (threadIdx.x >> 5) * N;
  const Cut c = static_cast<const Cut*>(a.workspace)[cta];
  if (r >= c.live || c.parts == 0) return;
  auto at = [&](int x) { return part_of<D, RB>(a.workspace, cta + x, x == 0); };
  float m = -INFINITY;
  for (int x0 = 0; x0 < c.parts; x0 += HELD) {
    float y[HELD];
#pragma unroll
    for (int x = 0; x < HELD; ++x) y[x] = __ldcg(at(min(x0 + x, c.parts - 1)) + RB * D + r);
#pragma unroll
    for (int x = 0; x < HELD; ++x) m = fmaxf(m, y[x]);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f, v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int x = 0; x < c.parts; ++x) {
    const float* p = at(x) + d0 * RB + r;
    const float y = __ldcg(at(x) + RB * D + r);
    float u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = __ldcg(p + i * RB);
    if (y == -INFINITY) continue;  // a part that saw nothing
    const float f = ex2(y - ref);
    sum += f;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fmaf(u[i], f, v[i]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int G = a.Hq / a.Hk, node = (c.row_base + r) / G, hq = c.h * G + c.row_base + r - node * G;
  T* out = static_cast<T*>(a.out) + int64_t(c.r0 + node) * a.o_strides[0] + hq * a.o_strides[1] + d0;
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    uint4 w;
    w.x = Elem<T>::pack(v[i] * inv, v[i + 1] * inv);
    w.y = Elem<T>::pack(v[i + 2] * inv, v[i + 3] * inv);
    w.z = Elem<T>::pack(v[i + 4] * inv, v[i + 5] * inv);
    w.w = Elem<T>::pack(v[i + 6] * inv, v[i + 7] * inv);
    *reinterpret_cast<uint4*>(out + i) = w;
  }
}

template <typename T, int D>
static int launch(const dspark_paged_attn_args& a, cudaStream_t s) {
  constexpr int TOTAL = Lay<D>::TOTAL;
  const int dev = current_device(), n = std::min(sm_count(dev), MAX_CTA);
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? a.vp_strides : a.kp_strides;
    // (a dimension of one entry is never stepped: any valid stride does)
    const uint64_t dims[4] = {uint64_t(D), uint64_t(a.page), uint64_t(a.Hk), uint64_t(a.n_pages)};
    const uint64_t strides[3] = {uint64_t(st[2]), uint64_t(a.Hk > 1 ? st[1] : D), uint64_t(a.n_pages > 1 ? st[0] : D)};
    const uint32_t box[4] = {uint32_t(D), uint32_t(a.page), 1, 1};
    if (!encode_tmap_nd(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, i ? a.v_pages : a.k_pages, dims, strides, box,
                        D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return NO_MAP;
  }
  DSPARK_CUDA_TRY(configure_once((const void*)attn_kernel<T, D>, TOTAL,
                                 [&] {
                                   // setmaxnreg.inc waits for registers that the block was launched with
                                   cudaFuncAttributes f;
                                   const cudaError_t e = cudaFuncGetAttributes(&f, attn_kernel<T, D>);
                                   if (e != cudaSuccess) return e;
                                   if (f.numRegs * NTHR < 256 * (184 + 72)) return cudaErrorLaunchOutOfResources;
                                   return cudaFuncSetAttribute(attn_kernel<T, D>,
                                                               cudaFuncAttributeMaxDynamicSharedMemorySize, TOTAL);
                                 }),
                  "paged_attn: shared memory");
  const float c = fabsf(a.scale) * 1.4426950408889634f;
  DSPARK_CUDA_TRY(launch_ex(attn_kernel<T, D>, dim3(n), dim3(NTHR), TOTAL, s, 1, true, maps[0], maps[1], a, c,
                            a.scale < 0.f ? 0x80008000u : 0u, status_word(dev)),
                  "paged_attn");
  DSPARK_CUDA_TRY(launch_ex(join_wide_kernel<T, D>, dim3(n, RB / 32), dim3(128), 0, s, 1, true, a), "paged_attn: join");
  return DSPARK_OK;
}

}  // namespace wide

size_t wide_workspace(int D) {
  return MAX_CTA * sizeof(Cut) + size_t(std::min(sm_count(current_device()), MAX_CTA)) * 2 * wide::RB * (D + 1) * sizeof(float);
}

int launch_wide(const dspark_paged_attn_args& a, cudaStream_t s) {
  if (a.dtype == DSPARK_DTYPE_BF16) return a.D == 128 ? wide::launch<bf16, 128>(a, s) : wide::launch<bf16, 64>(a, s);
  return a.D == 128 ? wide::launch<__half, 128>(a, s) : wide::launch<__half, 64>(a, s);
}

}  // namespace paged
}  // namespace dspark
