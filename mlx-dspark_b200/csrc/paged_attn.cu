// Attention of packed rows over pages of 8-bit values with a scale a page and head (dspark_paged_attn).
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(scale q_i.k_j - m_i), k_j = code * ks(page of j), v_j = code * vs.
// Neither scale is ever multiplied into a code: with x_ij = log2(e) scale ks (q_i.code_j) + log2(vs) and
// p'_ij = 2^(x_ij - max x), the sum over p' code_v is the numerator and the sum over p' / vs the denominator. The
// codes go to the tensor core as fp16, which holds every e4m3 value, converted in registers on the way.
//
// Rows and items. The G = Hq / Hk heads of a kv head share its keys: row node * G + g of a product. An item is RB = 16
// or 32 rows of one (request, kv head), its work the key tiles (128 keys) that its last row sees. All items' costs
// lie in one line (requests in order, a request's heads, a head's row blocks), which is cut into equal shares, one a
// block of a resident grid, from the lengths on the device (shares, Walker). A block that has a whole item writes the
// output; of a cut item each block leaves an fp32 part, and a second launch joins the parts in order. Where a call has few
// items, each is a cluster of blocks instead, which join their parts through shared memory.
//
// Block: four warps, each on its own: a warp takes every fourth subtile of 32 keys of the segment, with a ring of
// its own in shared memory that it fills itself (16-byte cp.async, no block-wide wait in the loop), its own running
// maximum and its own O in registers; they are joined at the segment's end.
// mma.m16n8k16: S = Q K^T with the head's values dealt to the four lanes of a key so that a lane reads 16 codes at a
// time, O += P V with V transposed by ldmatrix in pairs of values.
//
// Rounding: q is used as fp16, bf16 rows scaled by a power of two (exact); weights p' are rounded to fp16, 2^11 times
// as large, so that what a long tail loses is below 2^-36 of the largest a key; scores, sums and O are fp32.
//
// Bound: HBM for decoded tokens (96 requests over 256 to 16k keys, 32/8 heads of 128, pages of 16: 128 us in a graph of such
// calls, 138 to 149 in calls one by one, 111.5 of them the bytes at the measured rate), latency for one (2k keys 8.8 us). fp16
// products, because the 8-bit form of this instruction is as slow as a conversion of its operands and needs q and the weights
// in parts: 313 us.
#include <algorithm>

#include "host_common.h"
#include "paged_share.cuh"

namespace dspark {
namespace paged {

constexpr int SUB = 32;      // keys a warp's subtile
constexpr int WARPS = 4;
constexpr int NTHR = WARPS * 32;
// Cost of a segment, in tiles. Us for 2, 3, 4, 5: 96 decoded tokens over 256 to 16k keys 131, 128, 131, 133, 200 over 256 to 4k
// 113, 114, 117, 121, 64 blocks of 1 to 8 rows over 256 to 2k 63, 61, 62, 62.
constexpr int SEG = 3;
constexpr float LIFT = 11.f; // weights are 2^11 times as large in fp16 ...
constexpr float SLACK = 4.f; // ... and the maximum in use may be 2^4 too low

template <int D, int RT>
struct Lay {
  static constexpr int RB = 16 * RT;
  static constexpr int PER_SM = 2;      // blocks an SM
  static constexpr int NS = 3;          // ring buffers a warp
  static constexpr int TILE = SUB * D;                // a subtile's K or V codes
  static constexpr int STAGE = 2 * TILE + 32;         // K, V, two pages' scales
  static constexpr int RING = NS * STAGE;             // a warp's
  static constexpr int Q = 0;                         // fragments [rt][step][lane] of 16 bytes
  static constexpr int QF = Q + RB * D * 2;           // the rows' powers of two
  static constexpr int ML = QF + RB * 4;              // (m, l) [warp][row]
  static constexpr int BUF = ML + WARPS * RB * 8;
  static constexpr int AHEAD = NS - RT;               // loads of the next segment while a warp's O [row][D] is in the other buffers
  static constexpr int O = AHEAD * STAGE;             // ... in its ring, from here
  static constexpr int TOTAL = BUF + WARPS * RING;
  static_assert(BUF % 16 == 0 && STAGE % 16 == 0, "16-byte copies");
  static_assert(O + RB * D * 4 <= RING, "O");
};

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return Elem<__half>::pack(a, b); }

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// 16-byte chunk c of a subtile's row, swizzled so that the eight rows of an ldmatrix and the eight lanes of a 16-byte
// load meet different banks.
template <int D>
__device__ __forceinline__ uint32_t at_chunk(int row, int c) {
  return uint32_t(row * D + ((D == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) << 4));
}

// ------------------------------------------------------------------ the kernel

// Item i of the line as one segment, for up to 32 requests. A warp together.
template <int RB>
__device__ __forceinline__ bool find_item(const Plan<RB>& p, int i, Segment& g) {
  const dspark_paged_attn_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int n = lane < a.B ? p.shape(lane).M * a.Hk : 0;
  int to = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, to, o);
    if (lane >= o) to += y;
  }
  const unsigned past = __ballot_sync(0xffffffffu, i < to);
  if (past == 0) return false;
  const int b = __ffs(past) - 1;
  i -= __shfl_sync(0xffffffffu, to - n, b);
  const Shape s = p.shape(b);
  const int h = i / s.M, m = i - h * s.M;
  g = Segment{b, h, s.r0, s.rows, s.len, s.before, m * RB, min(s.rows * (a.Hq / a.Hk) - m * RB, RB), 0, p.tiles(s, m), 0, 1};
  return true;
}

// CL = 1: a block takes its share of the line. CL > 1: a cluster an item, its warps in turn through the subtiles; the
// blocks' parts are joined through their shared memory.
template <typename T, int D, int RT, int CL>
__global__ void __launch_bounds__(NTHR, 2) attn_kernel(const dspark_paged_attn_args a, const float c_log2,
                                                       const uint32_t q_sign, int* status) {
  typedef Lay<D, RT> L;
  constexpr int RB = L::RB, KS = D / 16, CH = D / 16;  // k steps of the scores, 16-byte chunks a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint2 s_cost[WARPS], s_req;
  __shared__ float s_lse[RB];  // (CL > 1)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, qd = lane & 3;  // row (or key) and quarter of an mma fragment
  pdl_launch_dependents();
  pdl_wait();
  Plan<RB> plan{a, 0};
  Walker<RB> wk;
  Deal deal(0, 1);
  if (CL == 1) deal = find_share<RB, NTHR>(plan, SEG, wk, s_cost, &s_req);
  Cut cut{0, 0, 0, 0, 0, {0, 0, 0}};

  const int G = a.Hq / a.Hk, shift = 31 - __clz(a.page);
  uint8_t* ring = smem + L::BUF + warp * L::RING;
  const uint32_t ring_a = smem_u32(ring);
  const uint32_t q_a = smem_u32(smem + L::Q) + lane * 16;
  float* rowf = reinterpret_cast<float*>(smem + L::QF);
  float2* ml = reinterpret_cast<float2*>(smem + L::ML);
  // float4 d / 4 of row r of a warp's O
  auto merge = [&](int w, int r, int d) {
    return reinterpret_cast<float4*>(smem + L::BUF + w * L::RING + L::O) + (r * (D / 4) + (d / 4 ^ (r & 1) << 2));
  };

  constexpr int RPI = 32 / CH, ROUNDS = SUB / RPI;  // tokens a round of 16-byte copies, rounds a subtile
  const int kts = int(a.kp_strides[2]), vts = int(a.vp_strides[2]);
  const bool packed = kts == D && vts == D;
  const uint32_t sw0 = at_chunk<D>(lane / CH, lane % CH), sw1 = at_chunk<D>(RPI + lane / CH, lane % CH) - RPI * D;

  constexpr int STEP = CL * WARPS;  // subtiles between a warp's
  // The segment whose subtiles are on their way: the one in work, from its end on the next one.
  int sub0 = 0, n = 0, len = 0, ids = -1, later = -1;
  const int32_t* table = nullptr;
  const uint8_t *kp = nullptr, *vp = nullptr;
  const float *ksc = nullptr, *vsc = nullptr;
  // The pages of 16 subtiles' halves, a half a lane (-1 where there is none to read): read 16 subtiles ahead.
  auto page_ids = [&](int i0) {
    int id = -1;
    const int i = i0 + (lane >> 1), key = (sub0 + i * STEP) * SUB + (lane & 1) * 16;
    if (i < n && key < len) {
      id = table[key >> shift];
      if (id < 0 || id >= a.n_pages) {
        report_error(status, kErrAttnPage);
        id = -1;
      }
    }
    return id;
  };
  auto issue = [&](int i) {
    if (i < n) {
      if (i > 0 && (i & 15) == 0) {
        ids = later;
        later = page_ids(i + 16);
      }
      const uint32_t dst = ring_a + (i % L::NS) * L::STAGE;
      const int key0 = (sub0 + i * STEP) * SUB;
      const int id0 = __shfl_sync(0xffffffffu, ids, (i & 15) * 2), id1 = __shfl_sync(0xffffffffu, ids, (i & 15) * 2 + 1);
      if (lane < 2) {
        const int mine = lane ? id1 : id0;
        const int64_t at_s = mine < 0 ? 0 : int64_t(mine) * a.scale_strides[0];
        const uint32_t to = dst + 2 * L::TILE + lane * 8;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(ksc + at_s), "r"(mine < 0 ? 0 : 4)
                     : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4), "l"(vsc + at_s),
                     "r"(mine < 0 ? 0 : 4)
                     : "memory");
      }
      const int mask = a.page - 1;
      const uint8_t* k0 = kp + (id0 * a.kp_strides[0] + (key0 & mask) * a.kp_strides[2]);
      const uint8_t* v0 = vp + (id0 * a.vp_strides[0] + (key0 & mask) * a.vp_strides[2]);
      const uint8_t* k1 = kp + (id1 * a.kp_strides[0] + ((key0 + 16) & mask) * a.kp_strides[2]);
      const uint8_t* v1 = vp + (id1 * a.vp_strides[0] + ((key0 + 16) & mask) * a.vp_strides[2]);
      const bool whole = key0 + SUB <= len && id0 >= 0 && id1 >= 0;
      if (whole && packed) {  // the usual case: no address arithmetic a copy
#pragma unroll
        for (int z = 0; z < ROUNDS; ++z) {
          const uint32_t to = dst + z * RPI * D + (z & 1 ? sw1 : sw0);
          cp_async_16(to, (z < ROUNDS / 2 ? k0 : k1) + z % (ROUNDS / 2) * RPI * D);
          cp_async_16(to + L::TILE, (z < ROUNDS / 2 ? v0 : v1) + z % (ROUNDS / 2) * RPI * D);
        }
      } else {
#pragma unroll 1
        for (int z = 0; z < ROUNDS; ++z) {
          const uint32_t to = dst + z * RPI * D + (z & 1 ? sw1 : sw0);
          const int y = z % (ROUNDS / 2) * RPI;
          const uint8_t* k = (z < ROUNDS / 2 ? k0 : k1) + y * kts;
          const uint8_t* v = (z < ROUNDS / 2 ? v0 : v1) + y * vts;
          const bool there = whole || ((z < ROUNDS / 2 ? id0 : id1) >= 0 && key0 + z * RPI + lane / CH < len);
          cp_async_16_zfill(to, there ? k : kp, there);
          cp_async_16_zfill(to + L::TILE, there ? v : vp, there);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto start = [&](const Segment& g) {
    sub0 = g.t0 * (BN / SUB) + (CL == 1 ? 0 : int(blockIdx.x) % CL * WARPS) + warp;
    const int sub1 = min(g.t1 * (BN / SUB), (g.len + SUB - 1) / SUB);
    n = sub0 < sub1 ? (sub1 - sub0 + STEP - 1) / STEP : 0;
    len = g.len;
    table = a.page_table + int64_t(g.b) * a.table_stride;
    // the lane's first 16 bytes of a subtile; the next are RPI tokens on
    kp = static_cast<const uint8_t*>(a.k_pages) + g.h * a.kp_strides[1] + lane / CH * kts + lane % CH * 16;
    vp = static_cast<const uint8_t*>(a.v_pages) + g.h * a.vp_strides[1] + lane / CH * vts + lane % CH * 16;
    ksc = a.k_scale + g.h * a.scale_strides[1];
    vsc = a.v_scale + g.h * a.scale_strides[1];
    ids = page_ids(0);
    later = page_ids(16);
    __syncwarp();  // the last segment's buffers have been read
#pragma unroll
    for (int i = 0; i < L::AHEAD; ++i) issue(i);
  };

  // 16 neighbouring values of a row of Q a thread and round; of 16 rows a segment ahead (of 32 the registers are not there:
  // 62.4 us for 61.3).
  constexpr bool Q_AHEAD = RT == 1;
  constexpr int PER = D / 16, Q_ROUNDS = (RB * PER + NTHR - 1) / NTHR;  // threads a row
  uint4 q0[Q_ROUNDS], q1[Q_ROUNDS];
  auto fetch_q = [&](const Segment& g) {
#pragma unroll
    for (int z = 0; z < Q_ROUNDS; ++z) {
      const int r = (z * NTHR + tid) / PER, p = tid % PER;
      q0[z] = q1[z] = make_uint4(0u, 0u, 0u, 0u);
      if (r < min(g.live, RB)) {
        const int node = (g.row_base + r) / G, hq = g.h * G + g.row_base + r - node * G;
        const T* q = static_cast<const T*>(a.q) + int64_t(g.r0 + node) * a.q_strides[0] + hq * a.q_strides[1] + p * 16;
        q0[z] = ldcg_v4(q);
        q1[z] = ldcg_v4(q + 8);
      }
    }
  };

  Segment s;
  bool more = CL == 1 ? wk.next(plan, deal, s) : find_item(plan, int(blockIdx.x) / CL, s);
  if (more) {
    start(s);
    if (Q_AHEAD) fetch_q(s);
  }
  while (more) {
#pragma unroll
    for (int i = L::AHEAD; i < L::NS - 1; ++i) issue(i);

    // ---- Q as fp16 fragments
    if (!Q_AHEAD) fetch_q(s);
    {
#pragma unroll
      for (int z = 0; z < Q_ROUNDS; ++z) {
        const int r = (z * NTHR + tid) / PER, p = tid % PER;
        uint32_t w[8] = {q0[z].x, q0[z].y, q0[z].z, q0[z].w, q1[z].x, q1[z].y, q1[z].z, q1[z].w};
        float f = 1.f;
        bool bad = false;
        if (std::is_same<T, bf16>::value) {  // largest exponent of the row; 255: infinite or NaN
          uint32_t e = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) e = max(e, max((w[i] >> 7) & 0xffu, (w[i] >> 23) & 0xffu));
#pragma unroll
          for (int o = 1; o < PER; o <<= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, o));
          // values below 2^15: the row divided by 2^(e - 127 - 14); in two steps, where that is no fp32 value
          const int up = int(e) - 141;
          const float inv = pow2(max(min(-up, 126), -126));
          bad = e == 255;
          f = bad ? 1.f : pow2(max(min(up, 126), -126));
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = pack_f16(bf16_lo(w[i]) * inv, bf16_hi(w[i]) * inv);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) bad |= (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
          uint32_t any = bad;
#pragma unroll
          for (int o = 1; o < PER; o <<= 1) any |= __shfl_xor_sync(0xffffffffu, any, o);
          bad = any;
        }
        if (bad) {  // an infinite q makes its row NaN whatever the codes are: by its scores, of which those of hidden keys are dropped
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = 0x7fff7fffu;
        }
        if (r < RB) {
          if (p == 0) rowf[r] = f * c_log2;
          // value d = quarter * D / 4 + step * 4 + j
          const int quarter = p * 16 / (D / 4), step0 = (p * 16 % (D / 4)) / 4, rt = r >> 4, rr = r & 15;
          uint32_t* to = reinterpret_cast<uint32_t*>(smem + L::Q) + (rr >> 3);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int f0 = ((rt * KS + step0 + i) * 32 + (rr & 7) * 4 + quarter) * 4;
            to[f0] = w[2 * i] ^ q_sign;
            to[f0 + 2] = w[2 * i + 1] ^ q_sign;
          }
        }
      }
    }
    __syncthreads();

    float o[RT][D / 8][4], m[RT][2], l[RT][2], rf[RT][2];
    int lim[RT][2];  // keys that the thread's rows see
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int x = 0; x < D / 8; ++x) o[rt][x][0] = o[rt][x][1] = o[rt][x][2] = o[rt][x][3] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = rt * 16 + i * 8 + g;
        m[rt][i] = -INFINITY;
        l[rt][i] = 0.f;
        rf[rt][i] = rowf[r];
        const int place = min((s.row_base + r) / G, s.rows - 1);
        lim[rt][i] = a.causal ? min(s.len, s.before + place + 1) : s.len;
      }
    }
    const int edge0 = (a.causal ? min(s.len, s.before + s.row_base / G + 1) : s.len) - SUB;  // later: hidden keys

    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::NS - 2) : "memory");
      __syncwarp();
      issue(i + L::NS - 1);
      const int key0 = (sub0 + i * STEP) * SUB;
      const uint32_t kt = ring_a + (i % L::NS) * L::STAGE, vt = kt + L::TILE;
      const float2 sc0 = *reinterpret_cast<const float2*>(ring + (i % L::NS) * L::STAGE + 2 * L::TILE);
      const float2 sc1 = *reinterpret_cast<const float2*>(ring + (i % L::NS) * L::STAGE + 2 * L::TILE + 8);
      // pages without a positive scale (absent ones have 0) are not seen
      const bool ok0 = sc0.x > 0.f && sc0.y > 0.f, ok1 = sc1.x > 0.f && sc1.y > 0.f;
      const bool edge = key0 > edge0 || !ok0 || !ok1;

      // ---- scores
      float x[RT][4][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int t = 0; t < 4; ++t) x[rt][t][0] = x[rt][t][1] = x[rt][t][2] = x[rt][t][3] = 0.f;
#pragma unroll
      for (int half = 0; half < KS / 4; ++half) {  // 16 codes of a key, four steps
        uint4 kw[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          kw[t] = lds128(kt + at_chunk<D>(t * 8 + g, qd * (KS / 4) + half));
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          uint32_t qf[RT][4];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const uint4 y = lds128(q_a + ((rt * KS + half * 4 + st) * 32) * 16);
            qf[rt][0] = y.x; qf[rt][1] = y.y; qf[rt][2] = y.z; qf[rt][3] = y.w;
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t w = st == 0 ? kw[t].x : st == 1 ? kw[t].y : st == 2 ? kw[t].z : kw[t].w;
            const uint32_t b0 = e4m3_to_f16(w), b1 = e4m3_to_f16_hi(w);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma_f16(x[rt][t], qf[rt], b0, b1);
          }
        }
      }

      // ---- weights
      if (edge) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(key0 + t * 8 + 2 * qd + (e & 1) < lim[rt][e >> 1] && (t < 2 ? ok0 : ok1))) x[rt][t][e] = -INFINITY;
      }
      const float ks[2] = {ok0 ? sc0.x : 1.f, ok1 ? sc1.x : 1.f}, lv[2] = {ok0 ? lg2(sc0.y) : 0.f, ok1 ? lg2(sc1.y) : 0.f};
      const float iv[2] = {ex2(-lv[0]), ex2(-lv[1])};
      uint32_t pw[RT][4][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float f[2][2], mx[2];  // [row][page]: the factor of its scores; at least 1e-35, so that -inf stays that
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f[k][0] = rf[rt][k] * ks[0];
          f[k][1] = rf[rt][k] * ks[1];
          f[k][0] = f[k][0] < 1e-35f ? 1e-35f : f[k][0];
          f[k][1] = f[k][1] < 1e-35f ? 1e-35f : f[k][1];
          const float m0 = fmaxf(fmaxf(x[rt][0][2 * k], x[rt][0][2 * k + 1]), fmaxf(x[rt][1][2 * k], x[rt][1][2 * k + 1]));
          const float m1 = fmaxf(fmaxf(x[rt][2][2 * k], x[rt][2][2 * k + 1]), fmaxf(x[rt][3][2 * k], x[rt][3][2 * k + 1]));
          mx[k] = fmaxf(fmaf(m0, f[k][0], lv[0]), fmaf(m1, f[k][1], lv[1]));
        }
        const bool up = mx[0] > m[rt][0] + SLACK || mx[1] > m[rt][1] + SLACK;
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float y = mx[k];
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
            if (y > m[rt][k]) {
              const float g = ex2(m[rt][k] - y);  // (0 at first)
              m[rt][k] = y;
              l[rt][k] *= g;
#pragma unroll
              for (int z = 0; z < D / 8; ++z) {
                o[rt][z][2 * k] *= g;
                o[rt][z][2 * k + 1] *= g;
              }
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float ref = LIFT - (m[rt][k] == -INFINITY ? 0.f : m[rt][k]);
#pragma unroll
          for (int page = 0; page < 2; ++page) {
            const float add = lv[page] + ref;
            float sum = 0.f;
#pragma unroll
            for (int t = 2 * page; t < 2 * page + 2; ++t) {
              const float e0 = ex2(fmaf(x[rt][t][2 * k], f[k][page], add));
              const float e1 = ex2(fmaf(x[rt][t][2 * k + 1], f[k][page], add));
              sum += e0 + e1;
              pw[rt][t][k] = pack_f16(e0, e1);
            }
            l[rt][k] = fmaf(sum, iv[page], l[rt][k]);
          }
        }
      }

      // ---- O += P V
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // 16 keys
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          uint32_t w[4];
          const int row = j * 16 + (lane & 15), ch = c + (lane >> 4);
          ldmatrix_x4_trans(vt + at_chunk<D>(row, ch), w[0], w[1], w[2], w[3]);
          if (edge) {
            // A NaN code reaches only the rows that see its key: it is taken out, and its place counted.
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) bad |= (((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
            if (__any_sync(0xffffffffu, bad)) {
              uint32_t is[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t nan = (((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                is[k] = nan * 0x38u;    // e4m3's 1
                w[k] &= ~(nan * 0xffu);
              }
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) {
                uint32_t see[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int t = 2 * j + (k >> 1), key = key0 + t * 8 + 2 * qd, li = lim[rt][k & 1];
                  const bool ok = t < 2 ? ok0 : ok1;
                  see[k] = (ok && key < li ? 0x3c00u : 0u) | (ok && key + 1 < li ? 0x3c000000u : 0u);
                }
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                  const uint32_t y0 = __byte_perm(is[2 * cc], 0, 0x3120), y1 = __byte_perm(is[2 * cc + 1], 0, 0x3120);
                  float n0[4] = {0.f, 0.f, 0.f, 0.f}, n1[4] = {0.f, 0.f, 0.f, 0.f};
                  mma_f16(n0, see, e4m3_to_f16(y0), e4m3_to_f16(y1));
                  mma_f16(n1, see, e4m3_to_f16_hi(y0), e4m3_to_f16_hi(y1));
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    if (n0[e] > 0.f) o[rt][2 * (c + cc)][e] = NAN;
                    if (n1[e] > 0.f) o[rt][2 * (c + cc) + 1][e] = NAN;
                  }
                }
              }
            }
          }
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const uint32_t y0 = __byte_perm(w[2 * cc], 0, 0x3120), y1 = __byte_perm(w[2 * cc + 1], 0, 0x3120);
            const uint32_t a0 = e4m3_to_f16(y0), a1 = e4m3_to_f16(y1);
            const uint32_t b0 = e4m3_to_f16_hi(y0), b1 = e4m3_to_f16_hi(y1);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const uint32_t p[4] = {pw[rt][2 * j][0], pw[rt][2 * j][1], pw[rt][2 * j + 1][0], pw[rt][2 * j + 1][1]};
              mma_f16(o[rt][2 * (c + cc)], p, a0, a1);      // values 16 c + 2 n
              mma_f16(o[rt][2 * (c + cc) + 1], p, b0, b1);  // values 16 c + 2 n + 1
            }
          }
        }
      }
    }

    // ---- the warps' parts joined, the next segment's first subtiles on their way
    Segment next;
    const bool again = CL == 1 && wk.next(plan, deal, next);
    if (again) {
      start(next);
      if (Q_AHEAD) fetch_q(next);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y = l[rt][k];
        y += __shfl_xor_sync(0xffffffffu, y, 1);
        y += __shfl_xor_sync(0xffffffffu, y, 2);
        const int r = rt * 16 + k * 8 + g;
        if (qd == 0) ml[warp * RB + r] = make_float2(m[rt][k], y);
#pragma unroll
        for (int c = 0; c < CH; ++c)
          *merge(warp, r, 16 * c + 4 * qd) = make_float4(o[rt][2 * c][2 * k], o[rt][2 * c + 1][2 * k],
                                                         o[rt][2 * c][2 * k + 1], o[rt][2 * c + 1][2 * k + 1]);
      }
    }
    __syncthreads();
    const bool whole = CL == 1 && s.parts == 1;
    const int which = int(blockIdx.x) == s.first;
    float* part = CL > 1 || whole ? nullptr : part_of<D, RB>(a.workspace, blockIdx.x, which);
    if (CL == 1 && !whole && which) cut = Cut{s.parts, s.r0, s.live, s.row_base, s.h, {0, 0, 0}};
#pragma unroll 4
    for (int z = tid; z < RB * (D / 4); z += NTHR) {
      const int r = z / (D / 4), d = z % (D / 4) * 4;
      if (r >= s.live) break;
      float2 y[WARPS];
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        y[w] = ml[w * RB + r];
        mx = fmaxf(mx, y[w].x);
      }
      const float ref = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = ex2(y[w].x - ref);
        const float4 u = *merge(w, r, d);
        sum += y[w].y * f;
        v.x += u.x * f;
        v.y += u.y * f;
        v.z += u.z * f;
        v.w += u.w * f;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (nothing seen: v is zero)
      v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      if (whole) {
        const int node = (s.row_base + r) / G, hq = s.h * G + s.row_base + r - node * G;
        T* out = static_cast<T*>(a.out) + int64_t(s.r0 + node) * a.o_strides[0] + hq * a.o_strides[1] + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack(v.x, v.y), Elem<T>::pack(v.z, v.w));
      } else if (CL > 1) {  // in the place of the first warp's
        *merge(0, r, d) = v;
        if (d == 0) s_lse[r] = sum == 0.f ? -INFINITY : ref + lg2(sum);
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = v;
        if (d == 0) part[RB * D + r] = sum == 0.f ? -INFINITY : ref + lg2(sum);
      }
    }
    if (CL > 1) {
      cluster_sync_all();
#pragma unroll
      for (int z0 = 0; z0 < RB * (D / 4); z0 += CL * NTHR) {
        const int z = z0 + int(blockIdx.x) % CL * NTHR + tid, r = z / (D / 4), d = z % (D / 4) * 4;
        if (r >= min(s.live, RB)) break;
        float y[CL], top = -INFINITY, sum = 0.f;
        float4 u[CL], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < CL; ++q) {
          y[q] = ld_dsmem_f32(mapa_shared(smem_u32(s_lse + r), q));
          u[q] = ld_dsmem_f4(mapa_shared(smem_u32(merge(0, r, d)), q));
        }
#pragma unroll
        for (int q = 0; q < CL; ++q) top = fmaxf(top, y[q]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int q = 0; q < CL; ++q) {
          const float f = ex2(y[q] - ref);  // (a part that saw nothing: 0, and its values are)
          sum += f;
          v.x = fmaf(u[q].x, f, v.x);
          v.y = fmaf(u[q].y, f, v.y);
          v.z = fmaf(u[q].z, f, v.z);
          v.w = fmaf(u[q].w, f, v.w);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int node = (s.row_base + r) / G, hq = s.h * G + s.row_base + r - node * G;
        T* out = static_cast<T*>(a.out) + int64_t(s.r0 + node) * a.o_strides[0] + hq * a.o_strides[1] + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack(v.x * inv, v.y * inv), Elem<T>::pack(v.z * inv, v.w * inv));
      }
      cluster_sync_all();  // the others have read this block's part
    } else {
      __syncthreads();  // the buffers of O and Q are free again
    }
    more = again;
    if (again) s = next;
  }
  if (CL == 1 && tid == 0) static_cast<Cut*>(a.workspace)[blockIdx.x] = cut;
}

static int grid_of(int device, int per_sm) { return std::min(per_sm * sm_count(device), MAX_CTA); }

// Items of a call at most.
static int64_t most_items(const dspark_paged_attn_args& a, int rb) {
  return (int64_t(a.R) * (a.Hq / a.Hk) + int64_t(a.B) * (rb - 1)) / rb * a.Hk;
}

template <typename T, int D, int RT, int CL>
static int launch(const dspark_paged_attn_args& a, cudaStream_t s) {
  typedef Lay<D, RT> L;
  const int dev = current_device(), n = CL > 1 ? int(most_items(a, L::RB)) * CL : grid_of(dev, L::PER_SM);
  auto kernel = attn_kernel<T, D, RT, CL>;
  DSPARK_CUDA_TRY(configure_once((const void*)kernel, L::TOTAL,
                                 [&] {
                                   if (CL > 8) {
                                     const cudaError_t e =
                                         cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
                                     if (e != cudaSuccess) return e;
                                   }
                                   return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
                                 }),
                  "paged_attn: shared memory");
  // the running maximum needs a positive factor: a negative scale goes into q (none is below 1e-35, with which all weights
  // are equal)
  const float c = fabsf(a.scale) * 1.4426950408889634f;
  DSPARK_CUDA_TRY(launch_ex(kernel, dim3(n), dim3(NTHR), L::TOTAL, s, CL, true, a, c, a.scale < 0.f ? 0x80008000u : 0u,
                            status_word(dev)),
                  "paged_attn");
  if (CL == 1)
    DSPARK_CUDA_TRY(launch_ex(join_kernel<T, D, L::RB>, dim3(n, L::RB / 4), dim3(128), 0, s, 1, true, a), "paged_attn: join");
  return DSPARK_OK;
}

// Which calls go to clusters, without a second launch: those whose items (a request's rows taken as the average) all run at
// once, over keys that a cluster is done with soon. Clusters of 16 begin a microsecond later, and more than
// a block an SM of them not all at once (16 items over 1k keys 13.7): for few items with more than three subtiles a warp in
// clusters of 8. One launch and a join / clusters of
// 8 / of 16, us, 32/8 heads of 128: one row over 1k keys 9.1 / 6.6 / 7.9, 2049 11.0 / 9.2 / 9.5, 4k 12.0 / 10.5 / 9.6, 8k 15.7 /
// 15.5 / 12.6, 16k 19.8 / 24.9 / 19.2; 4 requests of 8 rows over 2k 22.6 / 16.0, 16k 51.3 / 45.6, 32k 78.8 / 78.2.
constexpr int CLUSTER_KEYS = 8192;
template <typename T, int D, int RT>
static int launch_few(const dspark_paged_attn_args& a, cudaStream_t s) {
  const int64_t sms = sm_count(current_device()), rows = (int64_t(a.R) * (a.Hq / a.Hk) + a.B - 1) / a.B;
  const int64_t items = (rows + 16 * RT - 1) / (16 * RT) * a.B * a.Hk, keys = int64_t(a.max_pages) * a.page;
  if (a.B <= 32) {
    if (items * 16 <= sms && keys > 3 * 8 * WARPS * SUB && keys <= 2 * CLUSTER_KEYS) return launch<T, D, RT, 16>(a, s);
    if (items * 8 <= 2 * sms && keys <= (items * 8 > sms ? 4 : 1) * CLUSTER_KEYS) return launch<T, D, RT, 8>(a, s);
  }
  return launch<T, D, RT, 1>(a, s);
}

// Which calls go to the 5th-generation tensor cores (paged_wide.cu): those with more than 32 rows a request and kv head on
// average and with work enough, in tiles of 32 rows by 128 keys (the table's width stands for the lengths, which are
// on the device). Measured, this kernel / the other, us, 32/8 heads of 128: 16 rows over 4k keys, 1 request (528 of
// such tiles with their 64 rows a head) 17 / 28, 4 requests (2112) 34 / 29, 8 (4224) 51 / 41, 16 84 / 62; one request of 64 rows
// over 4k (2112) 33 / 37, of 16 over 16k (2064) 35 / 38, of 32 over 16k (4128) 43 / 39; 64 requests over 4k, 8 rows (32 a head)
// 150 / 182, 16 rows 281 / 194.
// Not where a request may have more than 2^25 keys: a wait there can last a segment, which has to end within the limit.
constexpr int FEW_ROWS = 32, WIDE_TILES = 3000, LONGEST = 1 << 25;
static bool has_many_rows(int R, int B, int Hq, int Hk) { return int64_t(R) * (Hq / Hk) > int64_t(FEW_ROWS) * B; }
static bool is_wide(const dspark_paged_attn_args& a) {
  const int64_t blocks = (int64_t(a.R) * (a.Hq / a.Hk) + FEW_ROWS - 1) / FEW_ROWS * a.Hk, keys = int64_t(a.max_pages) * a.page;
  return has_many_rows(a.R, a.B, a.Hq, a.Hk) && blocks * (keys / BN + 1) > WIDE_TILES &&
         keys <= LONGEST && a.n_pages > 0;
}

template <typename T, int D>
static int launch_rows(const dspark_paged_attn_args& a, cudaStream_t s) {
  if (is_wide(a)) {
    const int rc = launch_wide(a, s);
    if (rc != NO_MAP) return rc;  // (the workspace is enough for either)
  }
  // rows of a product: 16 where requests have no more on average
  return int64_t(a.R) * (a.Hq / a.Hk) <= int64_t(16) * a.B ? launch_few<T, D, 1>(a, s) : launch_few<T, D, 2>(a, s);
}

}  // namespace paged
}  // namespace dspark

using namespace dspark;

extern "C" {

size_t dspark_paged_attn_workspace(int R, int B, int Hq, int Hk, int D) {
  if (R <= 0 || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || D <= 0) return 0;
  if (paged::has_many_rows(R, B, Hq, Hk)) return paged::wide_workspace(D);
  return paged::MAX_CTA * sizeof(paged::Cut) +
         size_t(paged::grid_of(current_device(), 2)) * 2 * 32 * (D + 1) * sizeof(float);
}

int dspark_paged_attn(const dspark_paged_attn_args* p, void* stream) {
  if (!p) return fail(DSPARK_ERR_ARG, "paged_attn: null argument");
  const dspark_paged_attn_args& a = *p;
  if (a.R < 0 || a.B < 0 || a.Hq <= 0 || a.Hk <= 0 || a.Hq % a.Hk || a.n_pages < 0 || a.max_pages < 0)
    return fail(DSPARK_ERR_ARG, "paged_attn: bad shape (%d rows, %d requests, %d / %d heads, %d pages)", a.R, a.B, a.Hq,
                a.Hk, a.n_pages);
  if (a.dtype != DSPARK_DTYPE_BF16 && a.dtype != DSPARK_DTYPE_F16)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: dtype %d (bf16 = 0, fp16 = 1)", a.dtype);
  if (a.D != 64 && a.D != 128) return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: head_dim %d (64 or 128)", a.D);
  if (a.page != 16 && a.page != 32 && a.page != 64 && a.page != 128)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: pages of %d tokens (16, 32, 64 or 128)", a.page);
  if (int64_t(a.max_pages) * a.page > 0x3fffffff)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: %d pages of %d tokens a request", a.max_pages, a.page);
  if (int64_t(a.R) * (a.Hq / a.Hk) > 0x3fffffff || (int64_t(a.R) * (a.Hq / a.Hk) / 16 + 1) * a.Hk > 0x3fffffff)
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: %d rows of %d heads in one call", a.R, a.Hq);
  // costs are summed in 32 bits
  if ((int64_t(a.R) * (a.Hq / a.Hk) / 16 + a.B) * a.Hk > 0x7fffffff / (int64_t(a.max_pages) * a.page / paged::BN + paged::SEG + 2))
    return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: %d rows over %d pages a request in one call", a.R, a.max_pages);
  if (a.R == 0 || a.B == 0) return DSPARK_OK;
  if (!a.q || !a.out || !a.cu_rows || !a.kv_len || (a.max_pages && !a.page_table) ||
      (a.n_pages && (!a.k_pages || !a.v_pages || !a.k_scale || !a.v_scale)))
    return fail(DSPARK_ERR_ARG, "paged_attn: null pointer");
  bool aligned = true;
  for (const void* x : {a.q, a.k_pages, a.v_pages, (const void*)a.out}) aligned &= reinterpret_cast<uintptr_t>(x) % 16 == 0;
  for (int i = 0; i < 2; ++i) aligned &= a.q_strides[i] % 8 == 0 && a.o_strides[i] % 8 == 0;
  for (int i = 0; i < 3; ++i) aligned &= a.kp_strides[i] % 16 == 0 && a.vp_strides[i] % 16 == 0;
  if (!aligned) return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: rows must be 16-byte aligned");
  for (int64_t t : {a.kp_strides[2], a.vp_strides[2]})
    if (t < 0 || t > 1 << 24) return fail(DSPARK_ERR_UNSUPPORTED, "paged_attn: %lld bytes between tokens", (long long)t);
  if (!a.workspace || a.ws_bytes < dspark_paged_attn_workspace(a.R, a.B, a.Hq, a.Hk, a.D))
    return fail(DSPARK_ERR_ARG, "paged_attn: workspace of %zu bytes", a.ws_bytes);
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return fail(DSPARK_ERR_ARG, "paged_attn: the workspace must be 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a.dtype == DSPARK_DTYPE_BF16)
    return a.D == 128 ? paged::launch_rows<bf16, 128>(a, s) : paged::launch_rows<bf16, 64>(a, s);
  return a.D == 128 ? paged::launch_rows<__half, 128>(a, s) : paged::launch_rows<__half, 64>(a, s);
}

}  // extern "C"
