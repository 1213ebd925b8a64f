// Attention of drafted trees over the cache (dspark_tree_attn): packed rows of ragged requests, each
// row seeing its request's cached prefix and its own ancestors, on the 5th-generation tensor cores.
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(scale q_i.k_j - m_i): one pass over the keys with a
// running maximum m_i and sum (fp32). The G = Hq / Hk query heads of a kv head share its keys, so
// the rows of one product are (node, head of the group): node * G + g.
//
// Items and segments. An item is up to 256 rows of one (request, kv head), its work a run of tiles of 128
// keys. The work of the call, in order (request, head, rows, keys), is cut into contiguous shares, one
// a CTA (one CTA per SM), from the lengths on the device: requests of any mix of lengths load the SMs
// evenly without the host knowing them (locate). A CTA walks its share as segments (a run of tiles of
// one item). A segment that covers its item writes the output; else it leaves an
// fp32 part (O and the logarithm of its sum) in the workspace, at most two a CTA; when all parts of an item
// are there, each of its CTAs joins a share of the rows, the parts in order (so results do not depend
// on timing). They wait for one another, so the launch is cooperative: all CTAs run at once.
//
// CTA: two slots of 128 rows (TMEM lanes), each with a softmax warpgroup, a score tile S (TMEM,
// overwritten by the 16-bit weights P) and an output accumulator O (TMEM).
//  * items of more than 128 rows: the slots are the two halves of the rows and share each K/V tile;
//  * items of up to 128 rows: the slots take the even and the odd key tiles of the segment and
//    are joined at its end (each warpgroup reads half of both slots' O: their rows have the same
//    lanes).
// Either way one slot's softmax runs under the other slot's products. One producer thread streams
// K and V tiles by TMA through a ring (the order the products use them); two preparing warps walk ahead
// and load the next segment's Q as soon as the last scores have read the old one, under the end of the
// softmax and the output of the old segment; one thread issues the products: S = Q K^T (both from shared memory, K-major), O += P V (P from tensor memory, V from
// shared memory as it lies, keys along K, so N-major). A thread of a softmax warpgroup owns a row:
// no shuffles. The maximum in use is only raised when a tile exceeds it by more than 2^8: the
// weights then stay within fp16 / fp32 range and O is rarely rescaled. (That, and starting the second product at
// three quarters of the weights, are known from published attention kernels for this architecture.)
//
// Rounding: the weights are rounded to the input's type for the product with V, as the tensor core takes them;
// scores, maxima, sums and O are fp32. Against 64 bits the mean error of a result is 1.3 to 1.4 times that of
// fp32 weights (bf16 0.0023 for 0.0017, fp16 0.00029 for 0.00021, most of both the result's own rounding).
//
// Bound: HBM up to about 200 rows an item, above that the chain of softmax and products, a chain of latencies
// for few tiles. Measured, 20 calls in a graph (a call of its own among others' work, host included):
// 64 ragged requests of 256 to 16k keys 195-236 us (196-236; 0.76 to 0.63 of a plain copy's rate, lowest when
// the GPU is at its power cap); two trees of 384 nodes, 64/8 heads, 32k keys 846-994 us (890-995; 975 to 830
// TFLOP/s at the power cap: 3750 clocks a tile of 256 x 128, 2048 of them products); one token over 2k keys
// 13.6 us (16); 61 nodes over 16k keys 35 us (37-39).
//
// Keys that a row does not see take no part whatever they hold: scores are replaced by -inf, V rows
// past the request's keys are zeroed in shared memory, and a non-finite V among the tree's own keys
// is taken out of the tile and added only to the rows that see it (fix_values / add_hidden).
#include <algorithm>
#include <atomic>
#include <chrono>

#include "elem.cuh"
#include "host_common.h"
#include "tcgen05.cuh"

namespace dspark {
namespace tattn {

constexpr int BN = 128;       // keys a tile
constexpr int ROWS = 128;     // rows a slot
constexpr int NTHR = 384;     // two softmax warpgroups; producer, MMA and two preparing warps
constexpr int WARP_TMA = 8, WARP_MMA = 9, WARP_PREP = 10;

template <int D>
struct Lay {
  static constexpr int TILE = BN * D * 2;         // a K or V tile (and a slot's Q)
  static constexpr int HALF = BN * 128;           // 64 values of 128 rows, 128-byte swizzled
  static constexpr int NB = D == 128 ? 5 : 10;    // ring buffers
  static constexpr int Q = 0;
  static constexpr int RING = 2 * TILE;
  static constexpr int ML = RING + NB * TILE;     // [slot][row] (m, l) at the segment's end
  static constexpr int FLAG = ML + 2 * ROWS * 8;
  static constexpr int SEGS = FLAG + 16;            // two segments for the softmax threads
  static constexpr int CUTS = SEGS + 2 * 64;        // the CTA's parts of cut items
  static constexpr int BARS = CUTS + 2 * 32 + 16;
  static constexpr int NBAR = 2 * NB + 2 * 8 + 1;
  static constexpr int TOTAL = BARS + NBAR * 8;
  static_assert(TOTAL <= 232448, "shared memory of one SM");
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
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 128-byte-swizzled operand: K-major (lbo unused, 8-row groups 1024 bytes apart) or MN-major (lbo
// between 64-value blocks of MN, 8-row groups of K 1024 bytes apart).
// Only the low word (address, lbo) varies: steps along the tile are added to it.
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

// ------------------------------------------------------------------ units, ranges, segments

__device__ __forceinline__ int rows_of(const dspark_tree_attn_args& a, int b, int& r0) {
  r0 = min(max(a.cu_rows[b], 0), a.R);
  return min(max(a.cu_rows[b + 1] - r0, 0), a.R - r0);
}

__device__ __forceinline__ int start_of(const dspark_tree_attn_args& a, int b) {
  return a.kv_start ? min(max(a.kv_start[b], 0), a.cap) : 0;
}

// Row blocks and key tiles of request b (a request of rows but no keys has one tile, all hidden), and
// what a tile of the last row block costs.
struct Shape {
  int M, T, wl;
};

// Costs in half microseconds, fitted to CTA times over ragged batches: a tile of one row block 1 us
// (more when HBM holds it: 64 KB take 1.5 us with all SMs at it), one of two row blocks 2 us, and a
// segment 7 us (its Q, its pipeline's fill, its O, its share of the joins). Mean of 47 mixes (1 to 250 requests
// of 1 to 100 nodes over 64 to 32k keys, groups of 1 to 8, two runs each) by a segment's cost: 8 98.4 us,
// 10 97.7, 12 96.8, 14 96.9, 16 97.0: flat from 12 to 16, the middle of it stands.
constexpr int ONE = 2, PAIR = 4, SEG = 14;

__device__ __forceinline__ Shape shape_of(const dspark_tree_attn_args& a, int b) {
  int r0;
  const int rows = rows_of(a, b, r0) * (a.Hq / a.Hk);
  Shape s;
  s.M = (rows + 2 * ROWS - 1) / (2 * ROWS);
  s.T = max(1, (min(a.kv_len[b], a.cap - start_of(a, b)) + BN - 1) / BN);
  s.wl = rows - (s.M - 1) * 2 * ROWS > ROWS ? PAIR : ONE;
  return s;
}

// Cost of all row blocks of one head.
__device__ __forceinline__ int cost_of(const Shape& s) {
  return s.M ? (s.M - 1) * (SEG + PAIR * s.T) + SEG + s.wl * s.T : 0;
}

// A CTA's work: either an equal share [x, end) of the summed cost of all items, which may cross from
// item to item, or (parts > 0) tiles [t0, t1) of one item that has CTAs of its own.
struct Range {
  int x, end;         // in costs
  int b, base;        // request of x (or of the item), the request's first cost
  int im, t0, t1;     // own: item of the request, its tiles
  int first, parts;   // own: the item's first CTA, how many
  int total, n;       // summed cost, CTAs that share it
  __device__ __forceinline__ int dealt(int c) const {
    const int q = n ? total / n : 0;
    return c < n ? c * q + min(c, total - q * n) : total;
  }
};

// CTAs of one item among n when items have their own: one each, and the others by the tiles.
__device__ __forceinline__ int ctas_of(int T, int n, int items, int tiles) {
  return min(T, 1 + int(uint32_t(T) * uint32_t(n - items) / uint32_t(tiles)));  // T < 2^24: one cache
}

// Every warp for itself, no barrier. Items get their own CTAs unless the longest range then has OWN
// tiles more than an equal deal: what a second segment costs is about that many tiles: 61 rows over
// 16k keys, 8 items: 40 us for the CTAs with two segments of together 7 tiles, 24 us for those with
// one.
constexpr int OWN = 8;
__device__ Range locate(const dspark_tree_attn_args& a, int cta, int n_cta) {
  const int lane = threadIdx.x & 31;
  auto scan = [&](int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    return v;
  };
  Shape mine{0, 1, ONE};  // the lane's own request of the first 32
  if (lane < a.B) mine = shape_of(a, lane);
  auto shape = [&](int b) { return b < 32 ? mine : b < a.B ? shape_of(a, b) : Shape{0, 1, ONE}; };
  int items = 0, tiles = 0, total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const Shape s = shape(b0 + lane);
    items += s.M * a.Hk;
    tiles += s.M * s.T * a.Hk;
    total += cost_of(s) * a.Hk;
  }
  items = __reduce_add_sync(0xffffffffu, items);
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  total = __reduce_add_sync(0xffffffffu, total);
  // shares are wider than any tile's cost, so that an item's parts lie in neighbouring CTAs
  Range r{0, 0, a.B, 0, 0, 0, 0, 0, 0, total, min(n_cta, max(1, total / (2 * PAIR)))};
  if (tiles == 0) return r;
  bool own = items <= n_cta;
  if (own) {
    int longest = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const Shape s = shape(b0 + lane);
      const int c = ctas_of(s.T, n_cta, items, tiles);
      if (s.M) longest = max(longest, (s.T + c - 1) / c);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    own = longest <= (tiles + n_cta - 1) / n_cta + OWN;
  }
  const int want = own ? cta : r.dealt(cta);  // in CTAs or in costs
  if (!own && want >= total) return r;
  int at = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const Shape s = shape(b0 + lane);
    const int c = ctas_of(s.T, n_cta, items, tiles);
    const int v = own ? s.M * a.Hk * c : cost_of(s) * a.Hk, x = scan(v);
    const unsigned hit = __ballot_sync(0xffffffffu, v > 0 && want < at + x && want >= at + x - v);
    if (hit) {
      const int k = __ffs(hit) - 1;
      r.b = b0 + k;
      r.base = at + __shfl_sync(0xffffffffu, x - v, k);
      if (own) {
        const int ck = __shfl_sync(0xffffffffu, c, k), Tk = __shfl_sync(0xffffffffu, s.T, k);
        const int local = want - r.base, im = local / ck, part = local - im * ck;
        r.im = im;
        r.t0 = Tk * part / ck;
        r.t1 = Tk * (part + 1) / ck;
        r.first = cta - part;
        r.parts = ck;
      } else {
        r.x = want;
        r.end = r.dealt(cta + 1);
      }
      return r;
    }
    at += __shfl_sync(0xffffffffu, x, 31);
  }
  return r;
}

// One run of key tiles of one item.
struct Segment {
  int b, h, rows, r0;   // request, kv head, its packed rows
  int row_base, live;   // first (node, head) row of the item, its rows (<= 256)
  int t0, t1, T;        // tiles [t0, t1) of T
  int len, first;       // keys, keys before the tree
  int start, kb;        // cache position and batch entry
  bool pair;
};

struct Walker {
  int x, end, base, b;        // next cost, end of the share, first cost of request b
  int start, w;               // of the item last given: its first cost, a tile's cost
  int im, t0, t1;             // own: the one segment (t1 0: given)
  __device__ __forceinline__ Walker(const Range& r)
      : x(r.x), end(r.end), base(r.base), b(r.b), start(0), w(ONE), im(r.im), t0(r.t0), t1(r.t1) {}

  // First tile of the item at or after a cost.
  static __device__ __forceinline__ int tile_at(int y, int start, int w, int T) {
    const int d = y - start - SEG;
    return d <= 0 ? 0 : min(T, (d + w - 1) / w);
  }
  __device__ __forceinline__ void fill(const dspark_tree_attn_args& a, Segment& s, const Shape& sh, int im_,
                                       int t0_, int t1_) {
    const int G = a.Hq / a.Hk;
    s.b = b;
    s.T = sh.T;
    s.t0 = t0_;
    s.t1 = t1_;
    s.h = im_ / sh.M;
    s.row_base = (im_ - s.h * sh.M) * 2 * ROWS;
    s.rows = rows_of(a, b, s.r0);
    s.live = min(s.rows * G - s.row_base, 2 * ROWS);
    s.pair = s.live > ROWS;
    s.start = start_of(a, b);
    s.len = max(0, min(a.kv_len[b], a.cap - s.start));
    s.first = a.kv_len[b] - s.rows;
    s.kb = a.kv_batch == 1 ? 0 : b;
  }
  __device__ __forceinline__ bool next(const dspark_tree_attn_args& a, Segment& s) {
    if (t1 > 0) {
      fill(a, s, shape_of(a, b), im, t0, t1);
      t1 = 0;
      return true;
    }
    while (x < end) {
      const Shape sh = shape_of(a, b);
      const int head = cost_of(sh);
      if (x >= base + head * a.Hk) {
        base += head * a.Hk;
        ++b;
        continue;
      }
      const int local = x - base, h = local / head, rem = local - h * head;
      const int full = SEG + PAIR * sh.T, m = min(rem / full, sh.M - 1);
      start = base + h * head + m * full;
      w = m + 1 < sh.M ? PAIR : sh.wl;
      const int stop = start + SEG + w * sh.T;
      const int u0 = tile_at(x, start, w, sh.T), u1 = end >= stop ? sh.T : tile_at(end, start, w, sh.T);
      x = stop;
      if (u0 < u1) {
        fill(a, s, sh, h * sh.M + m, u0, u1);
        return true;
      }
    }
    return false;
  }
};

// A segment as the preparing warps hand it to the softmax threads.
struct Handed {
  Segment s;
  int more;
};
static_assert(sizeof(Handed) <= 64, "Lay::SEGS");

// Ring use (within the segment) of the V tile of local tile t: the order of loads is K0 V0 K1 V1 ..
// (pair) or K0 K1 V0 K2 V1 .. (tiles alternate between the slots).
__device__ __forceinline__ int v_use(bool pair, int t, int n) {
  return pair ? 2 * t + 1 : t == n - 1 ? 2 * n - 1 : 2 * t + 2;
}

// Whether a row (its ancestor words, or its place in a chain) sees tree place j.
__device__ __forceinline__ bool sees(const uint32_t* anc, int words, int place, int j) {
  return anc ? j < 32 * words && ((anc[j >> 5] >> (j & 31)) & 1u) : j <= place;
}

// The place within its request of a slot's row (0 where there is none).
__device__ __forceinline__ int place_of(const dspark_tree_attn_args& a, const Segment& s, int slot, int row) {
  const int G = a.Hq / a.Hk, my = s.row_base + (s.pair ? slot * ROWS : 0) + row;
  return my < s.rows * G ? my / G : 0;
}

// The visibility bits of a tile's keys for one row; key k0 + c is bit c.
__device__ __forceinline__ void tile_bits(const dspark_tree_attn_args& a, const Segment& s, int r, int i,
                                          int k0, uint32_t* w) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int j = k0 + 32 * x - s.first;  // tree place of the word's first key
    uint32_t bits;
    if (j > -32) {
      uint32_t lo = 0, hi = 0;  // tree places [jw, jw + 64) that the row sees
      const int jw = j >= 0 ? j >> 5 : -1;
      if (a.anc) {
        const uint32_t* row = a.anc + int64_t(r) * a.anc_words;
        lo = jw >= 0 && jw < a.anc_words ? row[jw] : jw < 0 ? 0xffffffffu : 0u;
        hi = jw + 1 < a.anc_words ? row[jw + 1] : 0u;
      } else {
        const int n0 = i + 1 - 32 * jw, n1 = n0 - 32;
        lo = jw < 0 || n0 >= 32 ? 0xffffffffu : n0 > 0 ? (1u << n0) - 1u : 0u;
        hi = n1 >= 32 ? 0xffffffffu : n1 > 0 ? (1u << n1) - 1u : 0u;
      }
      bits = __funnelshift_r(lo, hi, uint32_t(j - 32 * jw));
    } else {
      bits = 0xffffffffu;
    }
    const int n = s.len - (k0 + 32 * x);  // keys that exist
    w[x] = n >= 32 ? bits : n > 0 ? bits & ((1u << n) - 1u) : 0u;
  }
}

// A tile whose V rows are not all plain values of visible or cached keys: rows past the request's
// keys are zeroed; non-finite values among the tree's keys are zeroed and reported (add_hidden
// gives them to the rows that see them). Thread x of the warpgroup has key x of the tile. A 16-bit
// value is not finite iff its exponent is all ones: adding one to the exponent field then carries
// into the sign's place, for both values of a word at once.
template <typename T, int D>
__device__ __noinline__ void fix_values(uint8_t* tile, int key, int len, int first, int* flag,
                                        int seg) {
  const int x = threadIdx.x & 127;
  const bool past = key + x >= len;
  if (!past && key + x < first) return;
  constexpr uint32_t em = Elem<T>::kExpMask, one = em & (0u - em);
  constexpr uint32_t MASK = em | (em << 16), ADD = one | (one << 16), TOP = 0x80008000u;
  auto at = [&](int c) {
    return reinterpret_cast<uint4*>(tile + (c >> 3) * Lay<D>::HALF + x * 128 + (((c & 7) ^ (x & 7)) << 4));
  };
  if (past) {
#pragma unroll
    for (int c = 0; c < D / 8; ++c) *at(c) = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  uint32_t bad = 0;
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    const uint4 v = *at(c);
    bad |= ((v.x & MASK) + ADD) | ((v.y & MASK) + ADD) | ((v.z & MASK) + ADD) | ((v.w & MASK) + ADD);
  }
  if (!(bad & TOP)) return;
  for (int c = 0; c < D / 8; ++c) {
    uint4 v = *at(c);
    uint32_t* w = &v.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t b = ((w[e] & MASK) + ADD) & TOP;
      if (b & 0x8000u) w[e] &= 0xffff0000u;
      if (b & 0x80000000u) w[e] &= 0x0000ffffu;
    }
    *at(c) = v;
  }
  *flag = seg;
}

// The non-finite values that fix_values took out of the segment's tiles, added to what a row that
// sees them has stored (`out`: the output, or `part`: the fp32 part, 256 values a step).
template <typename T>
struct Hidden {
  const T* v;             // the request's first value row of this kv head
  int64_t stride;
  const uint32_t* anc;    // the row's words, or null
  int words, place, k0, k1, first, d0, d1;
};

template <typename T>
__device__ __noinline__ void add_hidden(const Hidden<T> x, T* out, float* part) {
  for (int k = x.k0; k < x.k1; ++k) {
    if (!sees(x.anc, x.words, x.place, k - x.first)) continue;
    for (int d = x.d0; d < x.d1; ++d) {
      const float v = Elem<T>::to_f(x.v[int64_t(k) * x.stride + d]);
      if (isfinite(v)) continue;
      if (part) part[d * 2 * ROWS] += v;
      else out[d] = Elem<T>::from_f(Elem<T>::to_f(out[d]) + v);
    }
  }
}

// ------------------------------------------------------------------ workspace

// A cut item as one of its CTAs sees it: the CTA of its first part, how many there are (one CTA after
// the other), and its rows.
struct Cut {
  int first, parts, r0, live, row_base, h, pad[2];
};
constexpr int MAX_CTA = 160;

// The workspace: a count a CTA (of the item whose first part it has), two flags a CTA (of its parts),
// the number of failures, then part `which` of CTA c: D values (divided by the part's sum) and the logarithm of the sum, m + log2 l, of 256 rows (row
// innermost, as a warp of 32 rows writes them). An item's first part is its CTA's part 1, the others
// are part 0.
// words before the parts, which begin on a 128-byte line (off one, 61 nodes over 16k: 36.6 us for 35.0)
constexpr int HEAD = 3 * MAX_CTA + 16;
template <int D>
__device__ __forceinline__ float* part(void* ws, int c, int which) {
  return reinterpret_cast<float*>(static_cast<uint64_t*>(ws) + HEAD) +
         int64_t(2 * c + which) * (2 * ROWS) * (D + 1);
}

// Flags and counts live in memory that nobody clears beforehand: a flag is up when it is this run's
// tag, a count without the tag is zero. The tag is the launch's own, changed by the number of failures in the
// workspace: a replayed launch has the same, and after a wait that ran out flags may be left up and counts
// short. Whoever sees such a wait adds one to that number (any start value will do), so that the next
// run takes no flag of this one for its own. A flag costs its writer no answer from L2; a count of the parts
// took three (1.3 us). The last of an item's CTAs to say that it has seen all flags puts zeros back,
// so that a replayed launch (same tag) starts anew.
__device__ __forceinline__ uint64_t* flag_of(void* ws, int c, int which) {
  return static_cast<uint64_t*>(ws) + MAX_CTA + 2 * c + which;
}
__device__ __forceinline__ unsigned long long* failures_of(void* ws) {
  return static_cast<unsigned long long*>(ws) + 3 * MAX_CTA;
}
__device__ __forceinline__ uint64_t run_tag(uint64_t tag, uint64_t failures) {
  return (tag ^ (failures << 16)) | 1ull << 63;  // the low 16 bits stay zero: a count's
}
__device__ __forceinline__ void seen_all(void* ws, int first, int parts, uint64_t tag) {
  unsigned long long* p = static_cast<unsigned long long*>(ws) + first;
  __threadfence();
  const unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(p);
  int n = 0;
  if ((seen & ~0xffffull) != tag && atomicCAS(p, seen, tag | 1ull) == seen) n = 1;
  if (n == 0) n = int(atomicAdd(p, 1ull) & 0xffffu) + 1;
  if (n != parts) return;
  *reinterpret_cast<volatile unsigned long long*>(p) = 0;
  for (int x = 0; x < parts; ++x) *reinterpret_cast<volatile uint64_t*>(flag_of(ws, first + x, x == 0)) = 0;
}
__device__ __forceinline__ bool wait_flag(const uint64_t* word, uint64_t tag, int* status) {
  const uint64_t t0 = globaltimer_ns(), limit = wait_limit_ns(status);
  while (true) {
    uint64_t v;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(word) : "memory");
    if (v == tag) return true;
    if (globaltimer_ns() - t0 > limit) {
      report_error(status, kErrWaitPeer);
      return false;
    }
  }
}

// One warp beside the softmax threads' join: it shows the CTA's parts and waits for the other CTAs',
// so that nobody else waits for what it tells them afterwards.
__device__ __noinline__ void show_and_wait(void* workspace, const Cut* cuts, int n_cuts, int cta, uint64_t tag,
                                           int* status) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    __threadfence();
    for (int k = 0; k < n_cuts; ++k)
      asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(flag_of(workspace, cta, cuts[k].first == cta)),
                   "l"(tag)
                   : "memory");
  }
  __syncwarp();
  for (int k = 0; k < n_cuts; ++k) {
    const int first = cuts[k].first, parts = cuts[k].parts;
    for (int x = lane; x < parts; x += 32)
      if (!wait_flag(flag_of(workspace, first + x, x == 0), tag, status)) atomicAdd(failures_of(workspace), 1ull);
    named_sync(4, 288);
    if (lane == 0) seen_all(workspace, first, parts, tag);
    __syncwarp();
  }
}

// The 256 softmax threads, after the CTA's last segment: its share of the join of each item that it has
// a part of. The weights of all parts' rows go into shared memory, whose tiles are no longer needed; the
// sums are dealt out over the item's CTAs in blocks of 32 rows (lanes) x 4 values (a warp). The values of
// the first HELD parts are under way together, the first block's beside the weights.
template <typename T, int D>
__device__ __noinline__ void join_parts(void* workspace, T* o_base, int64_t o_row, int64_t o_head, int G,
                                        const Cut* cuts, int n_cuts, int cta, uint8_t* smem) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int64_t STRIDE = int64_t(2) * (2 * ROWS) * (D + 1);  // floats between the CTAs' parts
  // A part held costs its instructions whether it is there or not (code that runs once is paid by its length);
  // of more parts the rest comes a latency later. Mean of 40 mixes (one request of 1 to 61 rows over 1.5k
  // to 24k keys with 1, 2, 4 and 8 kv heads, which is 6 to 148 parts, and two and four requests) by parts
  // held: 8 22.5 us, 12 21.3, 16 21.4, 18 21.1, 20 21.0, 24 21.6.
  constexpr int HELD = 20;
  static_assert(MAX_CTA * 2 * ROWS * 4 <= Lay<D>::ML, "the weights' room");
  float* w = reinterpret_cast<float*>(smem);  // [parts][256]
  for (int k = 0; k < n_cuts; ++k) {
    const Cut c = cuts[k];
    named_sync(4, 288);  // show_and_wait has seen the item's flags
    const float* first = part<D>(workspace, c.first, 1);
    const float* rest = part<D>(workspace, c.first, 0);
    auto at = [&](int x) { return x == 0 ? first : rest + x * STRIDE; };
    const int live = c.live, rounds = (live + 31) / 32, blocks = rounds * (D / 4);
    float v[HELD], m = -INFINITY;
    if (tid < live) {
#pragma unroll
      for (int x = 0; x < HELD; ++x) v[x] = x < c.parts ? __ldcg(at(x) + 2 * ROWS * D + tid) : -INFINITY;
    }
    bool weighed = false;
    for (int z = (cta - c.first) + c.parts * warp; !weighed || z < blocks; z += c.parts * 8) {
      const int i = (z % rounds) * 32 + lane, d0 = z / rounds * 4;
      const bool mine = z < blocks && i < live;
      float o[HELD][4];
      if (mine) {
#pragma unroll
        for (int x = 0; x < HELD; ++x) {
          const float* p = at(x) + d0 * (2 * ROWS) + i;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[x][e] = x < c.parts ? __ldcg(p + e * (2 * ROWS)) : 0.f;
        }
      }
      if (!weighed) {
        if (tid < live) {
          float sum = 0.f;
#pragma unroll
          for (int x = 0; x < HELD; ++x) m = max3(m, v[x], v[x]);
#pragma unroll 8
          for (int x = HELD; x < c.parts; ++x) {
            const float y = __ldcg(at(x) + 2 * ROWS * D + tid);
            w[x * 2 * ROWS + tid] = y;
            m = max3(m, y, y);
          }
          const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int x = 0; x < HELD; ++x) {
            v[x] = ex2(v[x] - ref);
            sum += v[x];
          }
          for (int x = HELD; x < c.parts; ++x) {
            const float f = ex2(w[x * 2 * ROWS + tid] - ref);
            w[x * 2 * ROWS + tid] = f;
            sum += f;
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
          for (int x = 0; x < HELD; ++x) w[x * 2 * ROWS + tid] = v[x] * inv;  // (zero behind the last part)
          for (int x = HELD; x < c.parts; ++x) w[x * 2 * ROWS + tid] *= inv;
        }
        named_sync(3, 256);
        weighed = true;
      }
      if (mine) {
        float r[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < HELD; ++x) {
          const float f = w[x * 2 * ROWS + i];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] += o[x][e] * f;
        }
#pragma unroll 8
        for (int x = HELD; x < c.parts; ++x) {
          const float* p = at(x) + d0 * (2 * ROWS) + i;
          const float f = w[x * 2 * ROWS + i];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] += __ldcg(p + e * (2 * ROWS)) * f;
        }
        const int x = c.row_base + i, node = x / G, hq = c.h * G + x - node * G;
        T* out = o_base + int64_t(c.r0 + node) * o_row + hq * o_head + d0;
        *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack(r[0], r[1]), Elem<T>::pack(r[2], r[3]));
      }
    }
    named_sync(3, 256);  // the weights have been read: the next item's may land there
  }
}

// ------------------------------------------------------------------ the kernel

template <typename T, int D>
__global__ void __launch_bounds__(NTHR, 1)
    attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                const dspark_tree_attn_args a, const float c_log2, const uint32_t q_neg,
                const uint64_t tag, int* status) {
  typedef Lay<D> L;
  constexpr int NB = L::NB;
  constexpr uint32_t FMT = std::is_same<T, bf16>::value ? 1u : 0u;
  const uint32_t ID_QK = q_neg | (1u << 4) | (FMT << 7) | (FMT << 10) | (uint32_t(BN >> 3) << 17) |
                             (uint32_t(ROWS >> 4) << 24);
  constexpr uint32_t ID_PV = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) |
                             (uint32_t(D >> 3) << 17) | (uint32_t(ROWS >> 4) << 24);
  constexpr uint32_t O_COL = 256;
  // The weights are rounded to the input's type for the product with V (their sum is not). fp16 loses what
  // is below 2^-25, which adds up over a long row far below its largest key: all weights of all parts
  // are 2^7 times as large there (at most 2^15, with a reference 2^8 too low), which cancels in the end.
  constexpr float LIFT = std::is_same<T, bf16>::value ? 0.f : 7.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + L::RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty = full + NB;
  uint64_t* q_full = empty + NB;
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* p_part = p_full + 2;
  uint64_t* o_full = p_part + 2;
  uint64_t* q_empty = o_full + 2;
  uint64_t* seg_full = q_empty + 2;
  uint64_t* seg_empty = seg_full + 2;
  uint64_t* fin = seg_empty + 2;
  float2* ml = reinterpret_cast<float2*>(smem + L::ML);
  Cut* cuts = reinterpret_cast<Cut*>(smem + L::CUTS);
  int* n_cuts = reinterpret_cast<int*>(cuts + 2);
  int* flag = reinterpret_cast<int*>(smem + L::FLAG);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(flag + 2);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles need it; never seen without static arrays
    if (tid == 0) report_error(status, 0x205);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {  // p_*, q_full and seg_empty count warps
      mbar_init(&q_full[i], 2);
      mbar_init(&q_empty[i], 1);
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], 8);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_part[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      flag[i] = 0;
    }
    mbar_init(fin, 1);
    *n_cuts = 0;
    fence_mbar_init();
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  if (warp == WARP_MMA) tcg::tmem_alloc(tmem_slot, 512);
  pdl_launch_dependents();
  pdl_wait();
  const int cta = blockIdx.x;
  const Range range = locate(a, cta, gridDim.x);
  tcg::tc_fence_before();
  __syncthreads();
  tcg::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walker wk(range);
  bool ok = true;

  if (warp < WARP_TMA) {
    // ------------------------------------------- softmax: slot = warpgroup, row = TMEM lane
    // (registers: 256 * 216 + 128 * 72 = 384 * 168, what the block was launched with)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int slot = warp >> 2, row = tid & 127;
    const uint32_t t_s = tmem + (uint32_t((warp & 3) * 32) << 16) + uint32_t(slot * 128);
    const uint32_t t_o = t_s + O_COL;
    uint32_t n_s = 0;              // completed phases of s_full
    uint32_t n_o0 = 0, n_o1 = 0;   // of o_full
    int use0 = 0;                  // ring uses before this segment
    auto arrive = [&](uint64_t* bar) {  // this warp's stores to tensor memory are done
      tcg::tmem_wait_st();
      tcg::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // flag[seg & 1] == seg: a hidden non-finite value in segment `seg`. One slot may be a segment
    // ahead of the other, never two: the products of a segment need both slots' weights.
    for (int seg = 1;; ++seg) {
      const int hand = (seg - 1) & 1;
      const Handed& sh = *reinterpret_cast<const Handed*>(smem + L::SEGS + 64 * hand);
      if (ok) ok = mbar_wait(&seg_full[hand], uint32_t((seg - 1) >> 1) & 1u, status, kErrWaitPeer);
      // after a wait that ran out all leave together: the barriers below count all of them
      ok = named_all(3, 256, ok);
      if (!ok || !sh.more) break;
      const Segment& s = sh.s;
      const int n = s.t1 - s.t0;
      const bool pair = s.pair;
      const int steps = pair ? n : (n - slot + 1) >> 1;
      const int tile0 = pair ? s.t0 : s.t0 + slot, tstep = pair ? 1 : 2;
      const int edge0 = min(s.first, s.len) - BN;  // a tile from a later key on has hidden keys
      const int G = a.Hq / a.Hk;
      const bool warp_alive = s.row_base + (pair ? slot * ROWS : 0) + (warp & 3) * 32 < s.rows * G;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < steps; ++j) {
        const int k0 = (tile0 + j * tstep) * BN;
        const bool edge = k0 > edge0;
        uint32_t bits[4];
        if (edge) {  // while the scores are under way: who sees what
          const int place = place_of(a, s, slot, row);
          tile_bits(a, s, s.r0 + place, place, k0, bits);
        }
        if (ok) ok = mbar_wait(&s_full[slot], n_s & 1, status, kErrWaitMma);
        ++n_s;
        tcg::tc_fence_after();
        if (edge && (slot == 0 || !pair)) {
          // V put right. Not before the scores: they are made of K(t), and the previous use of V(t)'s
          // buffer was loaded before K(t) (at most NB - 2 uses lie between), so the parity waited for
          // here cannot be that of an earlier, still missing load
          const int g = use0 + v_use(pair, k0 / BN - s.t0, n);
          if (ok) ok = mbar_wait(&full[g % NB], uint32_t(g / NB) & 1u, status, kErrWaitKV);
          fix_values<T, D>(ring + (g % NB) * L::TILE, k0, s.len, s.first, flag + (seg & 1), seg);
          fence_proxy_async_smem();
        }
        if (warp_alive) {
          float x[128];
#pragma unroll
          for (int i = 0; i < 4; ++i) ld_x32(t_s + uint32_t(32 * i), x + 32 * i);
          tcg::tmem_wait_ld();
          if (edge) {
#pragma unroll
            for (int i = 0; i < 128; ++i) x[i] = (bits[i >> 5] >> (i & 31)) & 1u ? x[i] : -INFINITY;
          }
          float mx[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) mx[e] = max3(x[2 * e], x[2 * e + 1], x[16 + e]);
#pragma unroll
          for (int i = 24; i < 120; i += 16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) mx[e] = max3(mx[e], x[i + 2 * e], x[i + 2 * e + 1]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[120 + 2 * e], x[120 + 2 * e + 1]);
          const float mt = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), max3(mx[6], mx[7], mx[7]));
          if (!(mt < INFINITY)) m = NAN;  // a visible score of +inf or NaN: the row is NaN
          const bool raise = (mt - m) * c_log2 > 8.f;
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = raise ? mt : m;
            const float f = raise ? ex2((m - mn) * c_log2) : 1.f;
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
          const float mc = m == -INFINITY ? 0.f : m * c_log2;
          const f32x2 c2 = pack2(c_log2, c_log2), nm2 = pack2(LIFT - mc, LIFT - mc);
          f32x2 sum[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[e] = pack2(0.f, 0.f);
          // pair by pair, sums and packing LAG pairs behind the exponentials: the special-function
          // unit (8 cycles a warp instruction) then never waits for them
          constexpr int LAG = 4;
          f32x2 e[64];
          uint32_t p[64];
#pragma unroll
          for (int i = 0; i < 64 + LAG; ++i) {
            if (i < 64) {
              float e0, e1;
              unpack2(fma2(pack2(x[2 * i], x[2 * i + 1]), c2, nm2), e0, e1);
              e[i] = pack2(ex2(e0), ex2(e1));
            }
            const int z = i - LAG;
            if (z >= 0) {
              float e0, e1;
              unpack2(e[z], e0, e1);
              sum[z & 3] = add2(sum[z & 3], e[z]);
              p[z] = Elem<T>::pack(e0, e1);
              if ((z & 15) == 15) st_x16(t_s + uint32_t(z - 15), p + z - 15);
              if (z == 47) arrive(&p_part[slot]);  // three quarters' products may start
            }
          }
          float s0, s1;
          unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
          l += s0 + s1;
        } else {
          arrive(&p_part[slot]);
        }
        arrive(&p_full[slot]);
      }
      use0 += 2 * n;
      // ---- end of the segment: with one row block, both slots' O of half of the values
      if (ok && steps > 0) ok = mbar_wait(&o_full[slot], (slot ? n_o1 : n_o0) & 1, status, kErrWaitMma);
      const bool both = !pair && n > 1;
      if (ok && both) ok = mbar_wait(&o_full[slot ^ 1], (slot ? n_o0 : n_o1) & 1, status, kErrWaitMma);
      if (!pair && slot == 1 && n == 1 && ok) ok = mbar_wait(&o_full[0], n_o0 & 1, status, kErrWaitMma);
      ++n_o0;
      n_o1 += pair || n > 1;
      tcg::tc_fence_after();
      const bool whole = s.t0 == 0 && s.t1 == s.T;
      const int my = s.row_base + (pair ? slot * ROWS : 0) + row;  // (node, head) row of this thread
      const bool alive = my < s.rows * G;
      const int place = alive ? my / G : 0;
      float f0 = 1.f, f1 = 0.f;
      if (!pair) {
        ml[slot * ROWS + row] = make_float2(m, l);
        named_sync(3, 256);
        const float2 a0 = ml[row], a1 = ml[ROWS + row];
        const float mn = fmaxf(a0.x, a1.x), ref = mn == -INFINITY ? 0.f : mn;
        f0 = ex2((a0.x - ref) * c_log2);
        f1 = ex2((a1.x - ref) * c_log2);
        l = a0.y * f0 + a1.y * f1;
        m = mn;
      }
      const bool hidden = *reinterpret_cast<volatile int*>(&flag[seg & 1]) == seg;
      if (warp_alive) {
        const int hq = s.h * G + my - place * G;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float* pp = whole ? nullptr : part<D>(a.workspace, cta, s.t0 == 0 ? 1 : 0);
        const int prow = (pair ? slot * ROWS : 0) + row;
        // 32-value chunks: all of the slot's own, or every second one of both slots'
        const int i0 = pair ? 0 : slot * (D / 64), i1 = pair ? D / 32 : i0 + D / 64;
        const uint32_t t_0 = pair ? t_o : tmem + (uint32_t((warp & 3) * 32) << 16) + O_COL;
        T* out = static_cast<T*>(a.out) + int64_t(s.r0 + place) * a.o_strides[0] + hq * a.o_strides[1];
        if (!whole && (pair || slot == 0)) pp[2 * ROWS * D + prow] = m * c_log2 + lg2(l);
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
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) pp[(32 * i + e) * (2 * ROWS) + prow] = l == 0.f ? 0.f : o[e] * inv;
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
        if (hidden && alive) {
          Hidden<T> hd;
          hd.v = static_cast<const T*>(a.v) + s.kb * a.v_strides[0] + s.h * a.v_strides[1] +
                 int64_t(s.start) * a.v_strides[2];
          hd.stride = a.v_strides[2];
          hd.anc = a.anc ? a.anc + int64_t(s.r0 + place) * a.anc_words : nullptr;
          hd.words = a.anc_words;
          hd.place = place;
          hd.k0 = max(s.t0 * BN, max(s.first, 0));
          hd.k1 = min(s.t1 * BN, s.len);
          hd.first = s.first;
          hd.d0 = 32 * i0;
          hd.d1 = 32 * i1;
          add_hidden<T>(hd, out, whole ? nullptr : pp + prow);
        }
      }
      tcg::tc_fence_before();
      if (!pair) named_sync(3, 256);  // both have read both: the next weights may be given
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[hand]);
    }
    ok = named_all(4, 288, ok);  // this CTA's parts are written
    if (ok && *n_cuts)
      join_parts<T, D>(a.workspace, static_cast<T*>(a.out), a.o_strides[0], a.o_strides[1], a.Hq / a.Hk, cuts,
                       *n_cuts, cta, smem + L::Q);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    Segment s{};
    if (warp >= WARP_PREP) {
      // -------------------------------------------------------------- segments and Q, ahead
      constexpr int CH = D / 8, STEP = 64 / CH;  // 16-byte chunks a row, rows the 64 threads load at a time
      const int t = tid - WARP_PREP * 32, c = t % CH, first_row = t / CH, G = a.Hq / a.Hk;
      uint32_t n_q[2] = {0, 0};
      auto load_q = [&](int slot) {
        if (n_q[slot] > 0 && ok) ok = mbar_wait(&q_empty[slot], (n_q[slot] - 1) & 1u, status, kErrWaitMma);
        ++n_q[slot];
        const int row0 = s.row_base + (s.pair ? slot * ROWS : 0);
        const int live = min(ROWS, s.rows * G - row0);  // rows past it are never looked at
        const T* q = static_cast<const T*>(a.q) + int64_t(s.r0) * a.q_strides[0] + s.h * G * a.q_strides[1] + c * 8;
        const uint32_t dst = smem_u32(smem + L::Q + slot * L::TILE) + uint32_t((c >> 3) * L::HALF);
        const int dn = STEP / G, dg = STEP - dn * G;  // a step in (node, head of the group)
        int node = (row0 + first_row) / G, g = row0 + first_row - node * G;
        for (int r = first_row; r < live; r += STEP) {
          cp_async_16_zfill(dst + uint32_t(r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                            q + node * a.q_strides[0] + g * a.q_strides[1], true);
          node += dn;
          g += dg;
          if (g >= G) {
            g -= G;
            ++node;
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      auto give_q = [&](int slot) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[slot]);
      };
      for (int k = 0;; ++k) {
        const bool more = __all_sync(0xffffffffu, ok) && wk.next(a, s);
        const int hand = k & 1;
        if (warp == WARP_PREP) {
          if (k >= 2 && ok) ok = mbar_wait(&seg_empty[hand], uint32_t((k >> 1) - 1) & 1u, status, kErrWaitPeer);
          if (lane == 0) {
            Handed* h = reinterpret_cast<Handed*>(smem + L::SEGS + 64 * hand);
            if (more) {
              h->s = s;
              if (s.t0 > 0 || s.t1 < s.T) {
                int c0 = range.first, n_parts = range.parts;
                if (n_parts == 0) {
                  const int from = wk.start + SEG;  // cost of the item's first tile
                  int c1 = cta + 1;
                  for (c0 = cta; c0 > 0 && range.dealt(c0) > from; --c0) {}
                  while (c1 < range.n && range.dealt(c1) <= from + wk.w * (s.T - 1)) ++c1;
                  n_parts = c1 - c0;
                }
                cuts[(*n_cuts)++] = Cut{c0, n_parts, s.r0, s.live, s.row_base, s.h, {0, 0}};
              }
            }
            h->more = more;
            mbar_arrive(&seg_full[hand]);
          }
        }
        if (!more) break;
        const bool two = s.pair || s.t1 - s.t0 > 1;
        load_q(0);
        if (two) {
          load_q(1);
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          give_q(0);
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          give_q(1);
        } else {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          give_q(0);
        }
      }
      __syncwarp();
    } else if (warp == WARP_TMA) {
      // -------------------------------------------------------------- producer
      const uint64_t failures = *reinterpret_cast<volatile unsigned long long*>(failures_of(a.workspace));
      if (lane == 0) {
        int g = 0;
        auto load = [&](const CUtensorMap* map, int tile) {
          const int x = g % NB;
          if (g >= NB && ok)
            ok = mbar_wait(&empty[x], uint32_t(g / NB - 1) & 1u, status, kErrWaitKVEmpty);
          if (!ok) return;
          mbar_arrive_expect_tx(&full[x], L::TILE);
#pragma unroll
          for (int d = 0; d < D / 64; ++d)
            tma_load_4d(ring + x * L::TILE + d * L::HALF, map, &full[x], d * 64,
                        s.start + (s.t0 + tile) * BN, s.h, s.kb);
          ++g;
        };
        while (ok && wk.next(a, s)) {
          const int n = s.t1 - s.t0;
          load(&kmap, 0);
          if (!s.pair && n > 1) load(&kmap, 1);
          const int ahead = s.pair ? 1 : 2;
          for (int t = 0; t < n && ok; ++t) {
            load(&vmap, t);
            if (t + ahead < n) load(&kmap, t + ahead);
          }
        }
        // no copy may still be in flight when the CTA exits (under the default limit, whatever is set)
        for (int i = max(0, g - NB); i < g; ++i) mbar_wait(&full[i % NB], uint32_t(i / NB) & 1u, nullptr, 0);
      }
      __syncwarp();
      if (!named_all(4, 288, true)) {
        if (lane == 0) atomicAdd(failures_of(a.workspace), 1ull);
      } else if (*n_cuts) {
        show_and_wait(a.workspace, cuts, *n_cuts, cta, run_tag(tag, failures), status);
      }
    } else if (warp == WARP_MMA) {
      // -------------------------------------------------------------- products
      // The whole warp walks and waits; one lane issues. What an instruction needs is then the same in
      // every lane and can sit in uniform registers.
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
      auto scores = [&](int slot, int x, bool last) {
        if (!ok) return;
        const uint32_t qd = q_lo + uint32_t(slot) * (L::TILE >> 4);
        const uint32_t kd = desc_lo(ring_a + uint32_t(x) * L::TILE, 16);
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = uint32_t((k >> 2) * (L::HALF >> 4) + (k & 3) * 2);
            umma_ss(tmem + uint32_t(slot * 128), desc_sw128(qd + off), desc_sw128(kd + off), ID_QK,
                    k ? 1u : 0u);
          }
          tcg::umma_commit(&s_full[slot]);
          if (last) tcg::umma_commit(&q_empty[slot]);  // the segment's last use of this Q
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
            tcg::umma_ts(d, p + uint32_t(8 * k), desc_sw128(vd + uint32_t(k * (2048 >> 4))), ID_PV,
                    first && k == 0 ? 0u : 1u);
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
      while (__all_sync(0xffffffffu, ok) && wk.next(a, s)) {
        const int n = __shfl_sync(0xffffffffu, s.t1 - s.t0, 0);
        const bool pair = __shfl_sync(0xffffffffu, int(s.pair), 0);
        if (pair) {
          int x = take();
          q_ready(0);
          scores(0, x, n == 1);
          q_ready(1);
          scores(1, x, n == 1);
          release(x);
          for (int t = 0; t < n; ++t) {
            const int v = take();
            const bool more = t + 1 < n;
            values(0, v, t == 0);
            if (more) {
              x = take();
              scores(0, x, t + 2 == n);
            } else if (ok) {
              commit(&o_full[0]);
            }
            values(1, v, t == 0);
            release(v);
            if (more) {
              scores(1, x, t + 2 == n);
              release(x);
            } else if (ok) {
              commit(&o_full[1]);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
          }
        } else {
          for (int z = 0; z < min(n, 2); ++z) {
            const int x = take();
            q_ready(z);
            scores(z, x, z + 2 >= n);
            release(x);
          }
          for (int t = 0; t < n; ++t) {
            const int v = take(), z = t & 1;
            values(z, v, t < 2);
            release(v);
            if (t + 2 < n) {
              const int x = take();
              scores(z, x, t + 4 >= n);
              release(x);
            } else if (ok) {
              commit(&o_full[z]);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
          }
        }
      }
      if (issued) {  // nothing may write tensor memory after the CTA releases it
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

static int grid_of(int device) { return std::min(sm_count(device), MAX_CTA); }

template <typename T, int D>
static int launch(const dspark_tree_attn_args& a, cudaStream_t s) {
  const int dev = current_device();
  int* st = status_word(dev);
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    const int64_t* str = i ? a.v_strides : a.k_strides;
    // a dimension of one entry is never stepped: any valid stride does
    const uint64_t e = 2;
    const uint64_t ss = a.cap > 1 ? str[2] * e : D * e;
    const uint64_t sh = a.Hk > 1 ? str[1] * e : D * e;
    const uint64_t sb = a.kv_batch > 1 ? str[0] * e : D * e;
    const uint64_t dims[4] = {uint64_t(D), uint64_t(a.cap), uint64_t(a.Hk), uint64_t(a.kv_batch)};
    const uint64_t strides[3] = {ss, sh, sb};
    const uint32_t box[4] = {64, BN, 1, 1};
    if (!encode_tmap_nd(&maps[i], std::is_same<T, bf16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        4, i ? a.v : a.k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return fail(DSPARK_ERR_UNSUPPORTED, "tree_attn: cache strides {%lld, %lld, %lld}",
                  (long long)str[0], (long long)str[1], (long long)str[2]);
  }
  const int n_cta = grid_of(dev);
  // costs are summed in 32 bits, and tiles times CTAs too
  const int64_t G = a.Hq / a.Hk;
  if ((int64_t(a.R) * G / (2 * ROWS) + a.B) * a.Hk * (PAIR * ((int64_t(a.cap) + BN - 1) / BN + 1) + SEG) > 0x7fffffff ||
      a.cap / BN >= 1 << 24)
    return fail(DSPARK_ERR_UNSUPPORTED, "tree_attn: %d rows over %d positions in one call", a.R, a.cap);
  const size_t smem = Lay<D>::TOTAL;
  DSPARK_CUDA_TRY(configure_once((const void*)attn_kernel<T, D>, int(smem),
                                 [&] {
                                   return cudaFuncSetAttribute(attn_kernel<T, D>,
                                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                               int(smem));
                                 }),
                  "tree_attn: shared memory");
  // the running maximum needs a positive factor: a negative scale goes into the product (A negated),
  // and zero becomes one that leaves all weights equal
  const float c = a.scale == 0.f ? 1e-30f : fabsf(a.scale) * 1.4426950408889634f;
  const uint32_t neg = a.scale < 0.f ? 1u << 13 : 0u;
  static std::atomic<uint64_t> launches{uint64_t(std::chrono::steady_clock::now().time_since_epoch().count())};
  const uint64_t tag = (launches.fetch_add(1, std::memory_order_relaxed) * 0x9E3779B97F4A7C15ull | 1ull << 63) &
                       ~0xffffull;
  DSPARK_CUDA_TRY(launch_all_at_once(attn_kernel<T, D>, dim3(n_cta), dim3(NTHR), smem, s, maps[0], maps[1],
                                     a, c, neg, tag, st),
                  "tree_attn");
  return DSPARK_OK;
}

}  // namespace tattn
}  // namespace dspark

using namespace dspark;

extern "C" {

size_t dspark_tree_attn_workspace(int B, int Hq, int Hk, int D, int max_rows) {
  if (B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || D <= 0 || max_rows <= 0) return 0;
  return tattn::HEAD * sizeof(uint64_t) +
         size_t(tattn::grid_of(current_device())) * 2 * (2 * tattn::ROWS) * (D + 1) * sizeof(float);
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
  if (a.cap == 0 || a.max_rows == 0) return fail(DSPARK_ERR_ARG, "tree_attn: empty cache or max_rows 0");
  if (!a.q || !a.k || !a.v || !a.out || !a.cu_rows || !a.kv_len)
    return fail(DSPARK_ERR_ARG, "tree_attn: null pointer");
  if (a.anc && a.anc_words <= 0) return fail(DSPARK_ERR_ARG, "tree_attn: %d words a row", a.anc_words);
  bool aligned = true;
  for (const void* x : {a.q, a.k, a.v, (const void*)a.out}) aligned &= reinterpret_cast<uintptr_t>(x) % 16 == 0;
  for (int i = 0; i < 2; ++i) aligned &= a.q_strides[i] % 8 == 0 && a.o_strides[i] % 8 == 0;
  for (int i = 0; i < 3; ++i) aligned &= a.k_strides[i] % 8 == 0 && a.v_strides[i] % 8 == 0;
  if (!aligned) return fail(DSPARK_ERR_UNSUPPORTED, "tree_attn: rows must be 16-byte aligned");
  if (!a.workspace || a.ws_bytes < dspark_tree_attn_workspace(a.B, a.Hq, a.Hk, a.D, a.max_rows))
    return fail(DSPARK_ERR_ARG, "tree_attn: workspace of %zu bytes", a.ws_bytes);
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return fail(DSPARK_ERR_ARG, "tree_attn: the workspace must be 16-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a.dtype == DSPARK_DTYPE_BF16) return a.D == 128 ? tattn::launch<bf16, 128>(a, s) : tattn::launch<bf16, 64>(a, s);
  return a.D == 128 ? tattn::launch<__half, 128>(a, s) : tattn::launch<__half, 64>(a, s);
}

}  // extern "C"
