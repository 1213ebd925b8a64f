// Packing of drafted trees (dspark_tree_pack) and the cache's side of an accepted path
// (dspark_kv_keep_path). Integer and byte paths around the tree attention: latency-bound.
#include "common.cuh"
#include "host_common.h"

namespace dspark {
namespace tree {

// One block a request, one thread a row: the row walks up its ancestors (places descend, so the
// words of its bit row are finished from the top down).
__global__ void __launch_bounds__(256) pack_kernel(const int32_t* cu, const int32_t* parent,
                                                   const int32_t* kv_len, const int32_t* kv_start,
                                                   const int32_t* kv_cap, int B, int R, int32_t* row_pos,
                                                   int32_t* row_slot, int32_t* row_req,
                                                   uint32_t* anc, int words, int32_t* kv_len_new,
                                                   int32_t* room) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const int r0 = min(max(cu[b], 0), R), r1 = min(max(cu[b + 1], r0), R);
  const int L0 = kv_len[b];
  const int fit = kv_cap ? min(max(kv_cap[b] - L0, 0), r1 - r0) : r1 - r0;  // rows that have a place
  if (threadIdx.x == 0 && kv_len_new) kv_len_new[b] = L0 + (r1 - r0);
  if (threadIdx.x == 0 && room) room[b] = fit;
  for (int i = threadIdx.x; i < r1 - r0; i += blockDim.x) {
    const int r = r0 + i;
    int depth = 0;
    if (parent == nullptr) {
      depth = i;
      if (anc) {
        for (int w = 0; w < words; ++w) {
          const int n = i + 1 - 32 * w;  // places of this word up to the row's own
          anc[int64_t(r) * words + w] = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u;
        }
      }
    } else {
      uint32_t bits = 0;
      int w = words - 1;
      for (int at = i; at >= 0;) {
        if (anc && at < 32 * words) {
          for (; w > (at >> 5); --w) {
            anc[int64_t(r) * words + w] = bits;
            bits = 0;
          }
          bits |= 1u << (at & 31);
        }
        const int up = parent[r0 + at];
        if (up < 0 || up >= at) break;
        at = up;
        ++depth;
      }
      if (anc) {
        for (; w >= 0; --w) {
          anc[int64_t(r) * words + w] = bits;
          bits = 0;
        }
      }
    }
    if (row_pos) row_pos[r] = L0 + depth;
    if (row_slot) row_slot[r] = i < fit ? L0 + i + (kv_start ? kv_start[b] : 0) : -1;
    if (row_req) row_req[r] = kv_start ? 0 : b;
  }
  // rows behind the last request's: nobody's, so that nothing indexes with what the arrays held before
  if (b == B - 1) {
    for (int r = r1 + threadIdx.x; r < R; r += blockDim.x) {
      if (row_pos) row_pos[r] = 0;
      if (row_slot) row_slot[r] = -1;
      if (row_req) row_req[r] = -1;
      if (anc)
        for (int w = 0; w < words; ++w) anc[int64_t(r) * words + w] = 0u;
    }
  }
}

// A lane owns a 16-byte column of one head's rows in one cache and moves the path's rows in ascending
// order, KEEP_U at a time. A row's source never lies before its destination and sources ascend, so a
// destination is read by no later row, and no column depends on another. Grid: x columns of all
// heads, y requests, z caches (K and V of every layer). Bound: latency, or HBM with a large batch; only
// rows that move are touched. Measured in a graph: 36 layers of 8 heads of 128, one request 2.0 us, 64
// requests 10.2 us (7.2 TB/s of moved bytes: part of them still in L2).
constexpr int KEEP_U = 8;
__global__ void __launch_bounds__(128) keep_kernel(
    void* const* k_layers, void* const* v_layers, int64_t k_b, int64_t k_h, int64_t k_t, int64_t v_b,
    int64_t v_h, int64_t v_t, const int32_t* path, const int32_t* cu, const int32_t* n_accept,
    const int32_t* lens, const int32_t* kv_start, int chunks, int H, int cap, int kv_batch, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int col = blockIdx.x * 128 + threadIdx.x, b = blockIdx.y, layer = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const int r0 = cu[b], rows = cu[b + 1] - r0, na = n_accept[b];
  const int start = kv_start ? kv_start[b] : 0, base = lens[b] - na - 1 + start;
  const int n = min(na, rows - 1);
  uint8_t* p = static_cast<uint8_t*>(is_v ? v_layers[layer] : k_layers[layer]);
  if (col >= H * chunks) return;
  const int h = col / chunks, c = col - h * chunks;
  const int64_t ts = is_v ? v_t : k_t;
  p += (kv_batch == 1 ? 0 : b) * (is_v ? v_b : k_b) + h * (is_v ? v_h : k_h) + int64_t(base) * ts + c * 16;
  for (int i0 = 0; i0 <= n; i0 += KEEP_U) {
    int src[KEEP_U];
    bool stop = false;
#pragma unroll
    for (int u = 0; u < KEEP_U; ++u) src[u] = i0 + u <= n ? path[r0 + i0 + u] : i0 + u;
    uint4 v[KEEP_U];
#pragma unroll
    for (int u = 0; u < KEEP_U; ++u) {
      if (src[u] != i0 + u) {
        stop |= src[u] < i0 + u || src[u] >= rows || base < 0 || base + src[u] >= cap;
        if (!stop) v[u] = *reinterpret_cast<const uint4*>(p + int64_t(src[u]) * ts);
        else src[u] = i0 + u;  // outside the cache or out of order: nothing from here on
      }
    }
#pragma unroll
    for (int u = 0; u < KEEP_U; ++u)
      if (src[u] != i0 + u) *reinterpret_cast<uint4*>(p + int64_t(i0 + u) * ts) = v[u];
    if (stop) {
      report_error(status, 0x204);
      return;
    }
  }
}

}  // namespace tree
}  // namespace dspark

using namespace dspark;

extern "C" {

int dspark_tree_pack(const int32_t* cu_rows, const int32_t* parent, const int32_t* kv_len,
                     const int32_t* kv_start, int B, int R, int32_t* row_pos, int32_t* row_slot, int32_t* row_req, uint32_t* anc,
                     int anc_words, int32_t* kv_len_new, void* stream) {
  return dspark_tree_pack_capped(cu_rows, parent, kv_len, kv_start, nullptr, B, R, row_pos, row_slot, row_req,
                                 anc, anc_words, kv_len_new, nullptr, stream);
}

int dspark_tree_pack_capped(const int32_t* cu_rows, const int32_t* parent, const int32_t* kv_len,
                            const int32_t* kv_start, const int32_t* kv_cap, int B, int R, int32_t* row_pos,
                            int32_t* row_slot, int32_t* row_req, uint32_t* anc, int anc_words,
                            int32_t* kv_len_new, int32_t* room, void* stream) {
  if (B < 0 || R < 0) return fail(DSPARK_ERR_ARG, "tree_pack: bad shape (%d requests, %d rows)", B, R);
  if (B == 0) return DSPARK_OK;
  if (!cu_rows || !kv_len) return fail(DSPARK_ERR_ARG, "tree_pack: null pointer");
  if (anc && anc_words <= 0) return fail(DSPARK_ERR_ARG, "tree_pack: %d words a row", anc_words);
  DSPARK_CUDA_TRY(launch_ex(tree::pack_kernel, dim3(B), dim3(256), 0,
                            reinterpret_cast<cudaStream_t>(stream), 1, true, cu_rows, parent, kv_len,
                            kv_start, kv_cap, B, R, row_pos, row_slot, row_req, anc, anc_words, kv_len_new,
                            room),
                  "tree_pack");
  return DSPARK_OK;
}

int dspark_kv_keep_path(void* const* k_layers, void* const* v_layers, int n_layers,
                        const int64_t k_strides[3], const int64_t v_strides[3],
                        const int32_t* path, const int32_t* cu_rows, const int32_t* n_accept,
                        const int32_t* lens, const int32_t* kv_start, int B, int H, int D,
                        int elem_size, int cap, int kv_batch, void* stream) {
  if (n_layers < 0 || B < 0 || H <= 0 || D <= 0 || cap <= 0 || kv_batch <= 0)
    return fail(DSPARK_ERR_ARG, "kv_keep_path: bad shape");
  if (n_layers == 0 || B == 0) return DSPARK_OK;
  if (!k_layers || !v_layers || !k_strides || !v_strides || !path || !cu_rows || !n_accept || !lens)
    return fail(DSPARK_ERR_ARG, "kv_keep_path: null pointer");
  if (kv_batch != 1 && kv_batch < B)
    return fail(DSPARK_ERR_ARG, "kv_keep_path: %d requests, %d cache entries", B, kv_batch);
  const int64_t row_bytes = int64_t(D) * elem_size;
  if (elem_size <= 0 || row_bytes % 16 || row_bytes > 16384)
    return fail(DSPARK_ERR_UNSUPPORTED, "kv_keep_path: rows of %lld bytes (a multiple of 16)",
                (long long)row_bytes);
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] * elem_size % 16 || v_strides[i] * elem_size % 16)
      return fail(DSPARK_ERR_UNSUPPORTED, "kv_keep_path: cache rows must be 16-byte aligned");
  if (B > 65535 || n_layers > 32767)
    return fail(DSPARK_ERR_UNSUPPORTED, "kv_keep_path: %d requests, %d layers", B, n_layers);
  const int64_t e = elem_size;
  const int chunks = int(row_bytes / 16);
  DSPARK_CUDA_TRY(launch_ex(tree::keep_kernel, dim3((H * chunks + 127) / 128, B, 2 * n_layers), dim3(128), 0,
                            reinterpret_cast<cudaStream_t>(stream), 1, true, k_layers, v_layers,
                            k_strides[0] * e, k_strides[1] * e, k_strides[2] * e, v_strides[0] * e,
                            v_strides[1] * e, v_strides[2] * e, path, cu_rows, n_accept, lens,
                            kv_start, chunks, H, cap, kv_batch, status_word(current_device())),
                  "kv_keep_path");
  return DSPARK_OK;
}

}  // extern "C"
