// What the attention kernels over pages share: how the work of a call is cut into equal shares, one a block, from the
// lengths on the device, and how the parts of an item that was cut are joined.
#pragma once

#include "../../include/dspark.h"
#include "paged.cuh"

namespace dspark {
namespace paged {

constexpr int BN = 128;      // keys a tile
constexpr int MAX_CTA = 320;

// paged_wide.cu: blocks of many rows.
size_t wide_workspace(int D);
int launch_wide(const dspark_paged_attn_args& a, cudaStream_t s);
constexpr int NO_MAP = -1;  // launch_wide: pages of strides that no tensor map has

// ------------------------------------------------------------------ shares and segments

struct Shape {
  int rows, r0;       // packed rows, the first of them
  int len, before;    // keys that there are, those before the rows' own
  int M, T;           // row blocks, tiles that a row block has (on average)
  int C;              // what they cost: a tile of up to 128 rows 1, of more 2
};

// RB: rows of an item.
template <int RB>
struct Plan {
  const dspark_paged_attn_args& a;
  int seg;  // cost of a segment

  // Tiles of row block m: up to the last key that one of its rows sees, and one at least.
  __device__ __forceinline__ int tiles(const Shape& s, int m) const {
    const int G = a.Hq / a.Hk, last = min(s.rows - 1, ((m + 1) * RB - 1) / G);
    const int n = a.causal ? min(s.len, s.before + last + 1) : s.len;
    return max(1, (n + BN - 1) / BN);
  }
  __device__ __forceinline__ Shape shape(int b) const {
    Shape s;
    s.r0 = first_row(a.cu_rows, b, a.R);
    s.rows = max(first_row(a.cu_rows, b + 1, a.R) - s.r0, 0);
    const int len = max(a.kv_len[b], 0);
    s.len = min(len, a.max_pages * a.page);
    s.before = len - s.rows;
    const int G = a.Hq / a.Hk;
    s.M = (s.rows * G + RB - 1) / RB;
    s.T = s.M ? (tiles(s, 0) + tiles(s, s.M - 1) + 1) >> 1 : 0;
    s.C = s.rows * G > 128 && RB > 128 ? 2 * s.T : s.T;
    return s;
  }
};

// The line of costs (32 bits: refused above) cut into n shares.
struct Deal {
  uint32_t q, rem, total;
  int n;
  __device__ __forceinline__ Deal(uint32_t t, int most) : total(t), n(int(min(uint32_t(most), t))) {
    q = n ? t / n : 0;
    rem = n ? t - q * n : 0;
  }
  __device__ __forceinline__ uint32_t from(int c) const { return c < n ? c * q + min(uint32_t(c), rem) : total; }
  __device__ __forceinline__ int owner(uint32_t x) const {
    const uint32_t wide = rem * (q + 1);
    return x < wide ? int(x / (q + 1)) : int(rem + (x - wide) / q);
  }
};

// A run of tiles [t0, t1) of one item.
struct Segment {
  int b, h, r0, rows, len, before;
  int row_base, live;  // the item's first (node, head) row, how many
  int t0, t1;
  int first, parts;    // block of the item's first part, parts (1: whole)
};

template <int RB>
struct Walker {
  uint32_t x, end, base;  // next cost, end of the share, first cost of request b
  int b;
  Shape s;
  bool have;
  __device__ __forceinline__ bool next(const Plan<RB>& p, const Deal& deal, Segment& g) {
    const dspark_paged_attn_args& a = p.a;
    while (x < end) {
      if (!have) s = p.shape(b);
      have = true;
      const uint32_t item = p.seg + s.C, all = s.M * a.Hk * item;
      if (x >= base + all) {
        base += all;
        ++b;
        have = false;
        continue;
      }
      const uint32_t i = (x - base) / item, start = base + i * item, stop = start + item;
      // neighbours in the line are a short and a long row block: shares of equal cost are of equal work
      const int h = i / uint32_t(s.M), k = i - h * s.M, m = k & 1 ? s.M - 1 - (k >> 1) : k >> 1;
      const int T = p.tiles(s, m);
      auto tile_at = [&](uint32_t y) {
        const int d = int(y - start) - p.seg;
        return d <= 0 ? 0 : d >= s.C ? T : T == s.C ? d : int(int64_t(d) * T / s.C);
      };
      g.b = b;
      g.h = h;
      g.r0 = s.r0;
      g.rows = s.rows;
      g.len = s.len;
      g.before = s.before;
      g.row_base = m * RB;
      g.live = min(s.rows * (a.Hq / a.Hk) - g.row_base, RB);
      g.t0 = tile_at(x);
      g.t1 = end >= stop ? T : tile_at(end);
      g.first = deal.owner(start);
      g.parts = deal.owner(stop - 1) - g.first + 1;
      x = min(stop, end);
      return true;
    }
    return false;
  }
};

// The block's share of the line: the walker at its first request. All THREADS threads together; s_cost: THREADS / 32.
template <int RB, int THREADS>
__device__ __forceinline__ Deal find_share(Plan<RB>& plan, int seg, Walker<RB>& wk, uint2* s_cost, uint2* s_req) {
  const dspark_paged_attn_args& a = plan.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t items = 0, tiles = 0;  // of the thread's request; of the first THREADS requests they are kept
  auto weigh = [&](int b) {
    items = tiles = 0;
    if (b >= a.B) return;
    const Shape s = plan.shape(b);
    items = s.M * a.Hk;
    tiles = items * s.C;
  };
  uint32_t all_items = 0, all_tiles = 0;
  for (int b0 = (a.B - 1) / THREADS * THREADS; b0 >= 0; b0 -= THREADS) {
    weigh(b0 + tid);
    const uint32_t i = __reduce_add_sync(0xffffffffu, items), t = __reduce_add_sync(0xffffffffu, tiles);
    __syncthreads();
    if (lane == 0) s_cost[warp] = make_uint2(i, t);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      all_items += s_cost[w].x;
      all_tiles += s_cost[w].y;
    }
  }
  // a tile a block: nothing is gained by fuller shares
  plan.seg = all_tiles <= gridDim.x ? 0 : seg;
  const Deal deal(all_tiles + plan.seg * all_items, int(gridDim.x));
  wk.x = deal.from(blockIdx.x);
  wk.end = deal.from(blockIdx.x + 1);
  wk.have = false;
  if (tid == 0) *s_req = make_uint2(a.B, 0);
  uint32_t at = 0;
  for (int b0 = 0; b0 < a.B && wk.x < wk.end; b0 += THREADS) {
    if (b0 > 0) weigh(b0 + tid);
    const uint32_t v = tiles + plan.seg * items;
    uint32_t sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    __syncthreads();
    if (lane == 31) s_cost[warp].x = sum;
    __syncthreads();
    uint32_t before = at + sum - v;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += s_cost[w].x;
      at += s_cost[w].x;
    }
    if (v > 0 && wk.x >= before && wk.x < before + v) *s_req = make_uint2(b0 + tid, before);
  }
  __syncthreads();
  wk.b = s_req->x;
  wk.base = s_req->y;
  if (wk.b >= a.B) wk.end = wk.x;  // (no share, and never a request that is not there)
  return deal;
}

// ------------------------------------------------------------------ workspace

// What a block tells the join of the cut item whose first part it has (parts 0: none).
struct Cut {
  int parts, r0, live, row_base, h, pad[3];
};

template <int D, int RB>
__host__ __device__ constexpr size_t part_floats() {
  return size_t(RB) * (D + 1);
}
template <int D, int RB>
__device__ __forceinline__ float* part_of(void* ws, int cta, int which) {
  return reinterpret_cast<float*>(static_cast<Cut*>(ws) + MAX_CTA) + (size_t(cta) * 2 + which) * part_floats<D, RB>();
}

// One warp a row of a cut item: its parts in order.
template <typename T, int D, int RB>
__global__ void __launch_bounds__(128) join_kernel(const dspark_paged_attn_args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, r = blockIdx.y * 4 + (threadIdx.x >> 5);
  const Cut* cuts = static_cast<const Cut*>(a.workspace);
  const int cta = blockIdx.x;
  const Cut c = cuts[cta];
  if (r >= c.live || c.parts == 0) return;
  constexpr int V = D / 32;
  auto at = [&](int x) { return part_of<D, RB>(a.workspace, cta + x, x == 0); };
  float m = -INFINITY, sum = 0.f, v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  constexpr int HELD = 8;  // parts under way together
  for (int x0 = 0; x0 < c.parts; x0 += HELD) {
    float y[HELD], u[HELD][V];
#pragma unroll
    for (int x = 0; x < HELD; ++x) {
      const float* p = at(min(x0 + x, c.parts - 1));
      y[x] = __ldcg(p + RB * D + r);
      if (V == 4) {
        const float4 t = __ldcg(reinterpret_cast<const float4*>(p + r * D) + lane);
        u[x][0] = t.x; u[x][1] = t.y; u[x][V - 2] = t.z; u[x][V - 1] = t.w;
      } else {
        const float2 t = __ldcg(reinterpret_cast<const float2*>(p + r * D) + lane);
        u[x][0] = t.x; u[x][1] = t.y;
      }
    }
    float top = m;
#pragma unroll
    for (int x = 0; x < HELD; ++x) {
      if (x0 + x >= c.parts) y[x] = -INFINITY;
      top = fmaxf(top, y[x]);
    }
    const float ref = top == -INFINITY ? 0.f : top, old = ex2(m - ref);
    m = top;
    sum *= old;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= old;
#pragma unroll
    for (int x = 0; x < HELD; ++x) {
      if (y[x] == -INFINITY) continue;  // a part that saw nothing, or none
      const float f = ex2(y[x] - ref);
      sum += f;
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = fmaf(u[x][i], f, v[i]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int G = a.Hq / a.Hk, node = (c.row_base + r) / G, hq = c.h * G + c.row_base + r - node * G;
  T* out = static_cast<T*>(a.out) + int64_t(c.r0 + node) * a.o_strides[0] + hq * a.o_strides[1] + lane * V;
  if (V == 4)
    *reinterpret_cast<uint2*>(out) = make_uint2(Elem<T>::pack(v[0] * inv, v[1] * inv),
                                                Elem<T>::pack(v[V - 2] * inv, v[V - 1] * inv));
  else
    *reinterpret_cast<uint32_t*>(out) = Elem<T>::pack(v[0] * inv, v[1] * inv);
}

}  // namespace paged
}  // namespace dspark
