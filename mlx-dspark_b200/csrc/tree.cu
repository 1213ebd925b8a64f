// Packing of drafted trees (dspark_tree_pack) and the cache's side of an accepted path
// (dspark_kv_keep_path). Integer and byte paths around the tree attention: latency-bound.
#include "common.cuh"
#include "host_common.h"

namespace dspark {
namespace tree {

// One block a request, one thread a row: the row walks up its ancestors (places descend, so the
// words of its bit row are finished from the top down).
__global__ void __launch_bounds__(256) pack_kernel(const int32_t* cu, const int32_t* parent,
                                                   const int32_t* kv_len, int R, int32_t* row_pos,
                                                   int32_t* row_slot, int32_t* row_req,
                                                   uint32_t* anc, int words, int32_t* kv_len_new) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const int r0 = min(max(cu[b], 0), R), r1 = min(max(cu[b + 1], r0), R);
  const int L0 = kv_len[b];
  if (threadIdx.x == 0 && kv_len_new) kv_len_new[b] = L0 + (r1 - r0);
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
    if (row_slot) row_slot[r] = L0 + i;
    if (row_req) row_req[r] = b;
  }
}

// Simple form: one warp a (layer, K or V, request, head); each lane owns 16-byte columns and moves
// the path's rows in ascending order. A row's source never lies before its destination and sources
// ascend, so a destination is read by no later row and no row needs to wait for another column.
__global__ void __launch_bounds__(32) keep_simple_kernel(
    void* const* k_layers, void* const* v_layers, int64_t k_b, int64_t k_h, int64_t k_t, int64_t v_b,
    int64_t v_h, int64_t v_t, const int32_t* path, const int32_t* cu, const int32_t* n_accept,
    const int32_t* lens, const int32_t* kv_start, int row_bytes, int cap, int kv_batch, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  const int rows = cu[b + 1] - cu[b];
  const int n = min(n_accept[b], rows - 1);
  const int base = lens[b] - n_accept[b] - 1 + (kv_start ? kv_start[b] : 0);
  const int64_t bs = is_v ? v_b : k_b, hs = is_v ? v_h : k_h, ts = is_v ? v_t : k_t;
  uint8_t* p = static_cast<uint8_t*>(is_v ? v_layers[layer] : k_layers[layer]) +
               (kv_batch == 1 ? 0 : b) * bs + h * hs;
  for (int i = 0; i <= n; ++i) {
    const int src = path[cu[b] + i];
    if (src == i) continue;
    if (src < i || src >= rows || base < 0 || base + src >= cap) {
      if (threadIdx.x == 0) report_error(status, 0x204);
      return;
    }
    for (int d = threadIdx.x * 16; d < row_bytes; d += 512)
      *reinterpret_cast<uint4*>(p + int64_t(base + i) * ts + d) =
          *reinterpret_cast<const uint4*>(p + int64_t(base + src) * ts + d);
  }
}

}  // namespace tree
}  // namespace dspark

using namespace dspark;

extern "C" {

int dspark_tree_pack(const int32_t* cu_rows, const int32_t* parent, const int32_t* kv_len, int B,
                     int R, int32_t* row_pos, int32_t* row_slot, int32_t* row_req, uint32_t* anc,
                     int anc_words, int32_t* kv_len_new, void* stream) {
  if (B < 0 || R < 0) return fail(DSPARK_ERR_ARG, "tree_pack: bad shape (%d requests, %d rows)", B, R);
  if (B == 0) return DSPARK_OK;
  if (!cu_rows || !kv_len) return fail(DSPARK_ERR_ARG, "tree_pack: null pointer");
  if (anc && anc_words <= 0) return fail(DSPARK_ERR_ARG, "tree_pack: %d words a row", anc_words);
  DSPARK_CUDA_TRY(launch_ex(tree::pack_kernel, dim3(B), dim3(256), 0,
                            reinterpret_cast<cudaStream_t>(stream), 1, true, cu_rows, parent, kv_len,
                            R, row_pos, row_slot, row_req, anc, anc_words, kv_len_new),
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
  DSPARK_CUDA_TRY(launch_ex(tree::keep_simple_kernel, dim3(H, B, 2 * n_layers), dim3(32), 0,
                            reinterpret_cast<cudaStream_t>(stream), 1, true, k_layers, v_layers,
                            k_strides[0] * e, k_strides[1] * e, k_strides[2] * e, v_strides[0] * e,
                            v_strides[1] * e, v_strides[2] * e, path, cu_rows, n_accept, lens,
                            kv_start, int(row_bytes), cap, kv_batch, status_word(current_device())),
                  "kv_keep_path");
  return DSPARK_OK;
}

}  // extern "C"
