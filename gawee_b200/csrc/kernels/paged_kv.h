// Launch interfaces of the paged key/value cache kernels (paged_kv.cu).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "paged_index.h"

namespace gawee {
namespace kern {

// Attention: the query heads of a key/value head that a block computes together
// at most (a larger group takes several runs over the same keys) and the blocks
// that an SM holds at most.  They size the workspace.
constexpr int kKvHeadsMost = 16, kKvMaxBlocksPerSm = 4;

// The attention's workspace.  A part is the state of `heads` heads, in units of
// 16 bytes: maxima and sums, then the weighted sums of values.
GAWEE_HD int kv_part_head(int heads) { return (2 * heads + 3) / 4; }
GAWEE_HD int kv_part_vecs(int heads, int head_dim) { return kv_part_head(heads) + heads * head_dim / 4; }
// Floats of the parts on `sms` SMs, and segments (sequence, key/value head, chunk of heads).
inline int64_t kv_parts_floats(int sms, int group, int head_dim) {
  return (int64_t)2 * sms * kKvMaxBlocksPerSm * 4 * kv_part_vecs(group > 8 ? kKvHeadsMost : 8, head_dim);
}
inline int64_t kv_blocks(int sms) { return (int64_t)sms * kKvMaxBlocksPerSm; }
inline int64_t kv_segments(int64_t batch, int kv_heads, int group) { return batch * kv_heads * ((group + 3) / 4); }
// Attention by fp32 lanes: the lanes that hold a row, and the keys of a warp's
// tile (paged_attend.cuh, which is instantiated by these).
constexpr int kKvWarps = 4;
constexpr int kv_row_lanes(int head_dim) { return head_dim <= 32 ? 4 : head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32; }
constexpr int kv_warp_keys(int row_lanes) { return 128 / row_lanes; }
// Launches of an attention over f32 pages without weights: a second one joins
// the parts where a sequence may be longer than a block's tile.
inline int kv_attend_launches_f32(int head_dim, int64_t max_len) {
  return max_len > kKvWarps * kv_warp_keys(kv_row_lanes(head_dim)) ? 2 : 1;
}
// SMs that a graph's workspace is planned for; a GPU with more uses this many.
constexpr int kKvPlanSms = 160;

// Rows of new tokens into the pages: token t's key k[t * k_stride + h * D ..]
// goes to row positions[t] of sequence sequences[t] (nullptr: sequence t).  A
// token with a negative position or sequence is left out.
struct KvAppendParams {
  PageGeom geom;
  void *k_pages, *v_pages;
  int page_dt;
  const void *k, *v;
  int dt;
  int64_t k_stride, v_stride;
  int64_t tokens;
  const int32_t *sequences, *positions;
  const int32_t* table;
  int64_t table_stride, table_cols;
  int batch;
  int* status;
};
cudaError_t launch_kv_append(const KvAppendParams& p, cudaStream_t s);

// Attention of one new token per sequence over its cached rows.
struct KvAttendParams {
  PageGeom geom;
  void *k_pages, *v_pages;
  int page_dt;
  const void* q;
  void* out;
  int dt;  // of q, out, k and v
  int64_t q_stride, out_stride;
  int batch, heads;
  float scale;
  const int32_t* table;
  int64_t table_stride, table_cols;
  const int32_t* lengths;
  int64_t max_len;  // a longer length is an error
  const void *k, *v;  // the new token's row, stored first (nullptr: none)
  int64_t k_stride, v_stride;
  bool k_as_stored;      // k and v have the pages' type and 16-byte aligned rows (set by launch_kv_attend)
  const float* mask;
  int64_t mask_stride;
  const float* weights;  // accumulators before (nullptr with weights_out set: zeros) ..
  float* weights_out;    // .. and after this step (nullptr: not wanted)
  int64_t w_stride, w_batch, wo_stride, wo_batch;
  float* scores;         // [batch][kv_heads][max_len][heads / kv_heads], with weights_out
  float* stats;          // [batch][heads][2]: maximum and sum, with weights_out
  float* parts;          // states of parts of segments: two a block
  int2* info;            // of each segment: its first block, and the number of its blocks
  int2* splits;          // of each block: the segment that begins in its run and goes on behind it, and
                         // the number of its blocks (0: none)
  int device, sms;
  int page_shift;        // log2 of the page size, -1 where it is no power of two
  int* status;
};
cudaError_t launch_kv_attend(const KvAttendParams& p, cudaStream_t s);
// The same for pages of one type (paged_attend_*.cu), without the join.
struct KvAttendShape {
  int blocks;  // of the grid
  int heads;   // of a part: the heads that a block computes together
  bool split;  // a segment may have several tiles, and so several blocks
};
cudaError_t launch_kv_attend_f32(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s);
cudaError_t launch_kv_attend_f16(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s);
cudaError_t launch_kv_attend_bf16(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s);

// Eviction by accumulated weight.
struct KvEvictParams {
  PageGeom geom;
  void *k_pages, *v_pages;
  int page_dt;
  const float* weights;
  float* weights_out;
  int64_t w_stride, w_batch, wo_stride, wo_batch;
  const int32_t *table, *to_table;  // to_table nullptr: in place
  int64_t table_stride, to_stride, table_cols, to_cols;
  const int32_t* lengths;
  int32_t* lengths_out;
  int64_t max_len;
  int batch, budget, recent;
  int32_t* kept;     // [batch][kv_heads][budget]
  int32_t* plan;     // [batch][2] scratch: rows before, and the length to pass on
  int sms;
  int* status;
};
cudaError_t launch_kv_evict(const KvEvictParams& p, cudaStream_t s);

}  // namespace kern
}  // namespace gawee
