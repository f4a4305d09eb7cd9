// Kernels of the paged key/value cache: append, the weights' pass of
// attend (the attention itself is in paged_attend.cuh) and eviction by
// accumulated attention weight.
#include <algorithm>
#include <cstdint>

#include "paged_common.cuh"

namespace gawee {
namespace kern {

using namespace paged;

namespace {

// --- append -------------------------------------------------------------------
// One thread per element of a token's row over the heads.
template <class T>
__global__ void kv_append_kernel(KvAppendParams p) {
  const int row = p.geom.kv_heads * p.geom.head_dim;
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const int64_t seq = p.sequences ? (int64_t)p.sequences[t] : t;
    const int64_t pos = p.positions[t];
    if (seq < 0 || pos < 0) continue;
    const int64_t page = seq < p.batch ? page_of(p.table + seq * p.table_stride, p.table_cols, pos, p.geom) : -1;
    if (page < 0) {
      if (threadIdx.x == 0) set_status(p.status, seq < p.batch ? ST_KV_PAGE : ST_KV_SEQUENCE);
      continue;
    }
    const int slot = (int)(pos % p.geom.page_size);
    for (int i = threadIdx.x; i < row; i += blockDim.x) {
      const int h = i / p.geom.head_dim, d = i % p.geom.head_dim;
      const int64_t o = row_offset(page, h, slot, p.geom) + d;
      static_cast<T*>(p.k_pages)[o] = from_f<T>(load_act(p.k, p.dt, t * p.k_stride + i));
      static_cast<T*>(p.v_pages)[o] = from_f<T>(load_act(p.v, p.dt, t * p.v_stride + i));
    }
  }
}

// weights_out = weights + the attention weights of this step, summed over the
// query heads of the key/value head in their order.
__global__ void kv_weights_kernel(KvAttendParams p) {
  const int kvh = blockIdx.x % p.geom.kv_heads, b = blockIdx.x / p.geom.kv_heads;
  const int group = p.heads / p.geom.kv_heads;
  const int64_t len = p.lengths[b];
  if (len > p.max_len) return;
  const float* stats = p.stats + ((int64_t)b * p.heads + kvh * group) * 2;
  for (int64_t i = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; i < len; i += (int64_t)gridDim.y * blockDim.x) {
    const float* s = p.scores + ((int64_t)blockIdx.x * p.max_len + i) * group;
    float w = 0.f;
    for (int g = 0; g < group; ++g) {
      const float m = stats[2 * g], l = stats[2 * g + 1];
      w += s[g] == -INFINITY ? 0.f : exp2f((s[g] - m) * kLog2e) / l;
    }
    const float before = p.weights ? p.weights[b * p.w_batch + kvh * p.w_stride + i] : 0.f;
    p.weights_out[b * p.wo_batch + kvh * p.wo_stride + i] = before + w;
  }
}

// --- evict ---------------------------------------------------------------------
constexpr int kSelectThreads = 1024;

// Weights in ascending order of their values as unsigned integers; both zeros
// are equal and NaN is below every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Inclusive sums over the block of two flags; every thread calls it.
__device__ __forceinline__ int2 block_scan(int a, int b, int2* warp_sums, int2& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int packed = a | (b << 16);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, packed, o);
    if (lane >= o) packed += up;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = make_int2(packed & 0xffff, packed >> 16);
  __syncthreads();
  int2 before = make_int2(0, 0);
  total = make_int2(0, 0);
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    if (w == warp) before = total;
    total.x += warp_sums[w].x;
    total.y += warp_sums[w].y;
  }
  return make_int2(before.x + (packed & 0xffff), before.y + (packed >> 16));
}

// One block per (sequence, key/value head): the smallest weight that stays, by
// radix selection over the bits of weight_key, then the kept positions in
// order, with their weights moved to the front.
__global__ void __launch_bounds__(kSelectThreads) kv_select_kernel(KvEvictParams p) {
  __shared__ int hist[256];
  __shared__ int2 warp_sums[kSelectThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int kvh = blockIdx.x % p.geom.kv_heads, b = blockIdx.x / p.geom.kv_heads;
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
  int64_t len = p.lengths[b];
  if (len > p.max_len) {
    if (threadIdx.x == 0) set_status(p.status, ST_KV_LENGTH);
    len = -1;
  }
  const bool first = kvh == 0 && threadIdx.x == 0;
  if (first) p.new_len[b] = len > p.budget ? p.budget : p.lengths[b];
  const float* w = p.weights + b * p.w_batch + kvh * p.w_stride;
  float* wo = p.weights_out + b * p.wo_batch + kvh * p.wo_stride;
  if (len <= p.budget) {
    for (int j = threadIdx.x; j < p.budget; j += kSelectThreads) kept[j] = j < len ? j : -1;
    for (int j = threadIdx.x; j < len; j += kSelectThreads) wo[j] = w[j];
    return;
  }
  const int cand = (int)len - p.recent;
  uint32_t prefix = 0;
  int need = p.budget - p.recent;  // still to choose among the keys with this prefix
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int i = threadIdx.x; i < cand; i += kSelectThreads) {
      const uint32_t k = weight_key(w[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int bin = 255, n = need;
      while (hist[bin] < n) n -= hist[bin--];
      s_prefix = prefix | ((uint32_t)bin << shift);
      s_need = n;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // keys above `prefix` stay, and the first `need` of those equal to it
  const bool none = p.budget == p.recent;
  int out = 0, equal = 0;
  for (int base = 0; base < len; base += kSelectThreads) {
    const int i = base + threadIdx.x;
    const float x = i < len ? w[i] : 0.f;
    const uint32_t k = weight_key(x);
    const bool old = i < cand && !none;
    const bool eq = old && k == prefix;
    int2 total;
    const int2 e = block_scan(eq, 0, warp_sums, total);
    const bool keep = i < len && (i >= cand || (old && (k > prefix || (eq && equal + e.x <= need))));
    equal += total.x;
    const int2 r = block_scan(keep, 0, warp_sums, total);
    if (keep) {
      kept[out + r.x - 1] = i;
      wo[out + r.x - 1] = x;
    }
    out += total.x;
  }
  for (int i = p.budget + threadIdx.x; i < len; i += kSelectThreads) wo[i] = 0.f;
}

// Moves the kept rows to their places.  A block takes one (sequence, head) and
// one slice of the row's 16-byte vectors, in ascending order of the rows: row
// j goes to a place at or before its own, so that in place a block overwrites
// only what it has read.
constexpr int kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(KvEvictParams p, int vecs_slice, int elem_bytes) {
  const int kvh = blockIdx.x % p.geom.kv_heads, b = blockIdx.x / p.geom.kv_heads;
  const int row_vecs = p.geom.head_dim * elem_bytes / 16, slices = row_vecs / vecs_slice;
  char* pages = static_cast<char*>((int)blockIdx.y < slices ? p.k_pages : p.v_pages);
  const int v0 = (int)blockIdx.y % slices * vecs_slice;
  const int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
  const int32_t* from = p.table + b * p.table_stride;
  const int32_t* to = p.to_table ? p.to_table + b * p.to_stride : from;
  const int64_t to_cols = p.to_table ? p.to_cols : p.table_cols;
  const int rows = kMoveThreads / vecs_slice;
  if (kvh == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.lengths_out[b] = p.new_len[b];
  for (int j0 = 0; j0 < p.budget; j0 += rows) {
    const int j = j0 + threadIdx.x / vecs_slice;
    int src = -1;
    if (j < p.budget && (int)threadIdx.x < rows * vecs_slice) src = kept[j];
    uint4 x = make_uint4(0, 0, 0, 0);
    char* dst = nullptr;
    if (src >= 0 && (p.to_table || src != j)) {
      const int64_t fp = page_of(from, p.table_cols, src, p.geom), tp = page_of(to, to_cols, j, p.geom);
      if (fp < 0 || tp < 0) {
        set_status(p.status, ST_KV_PAGE);
      } else {
        const int64_t v = (int64_t)(v0 + threadIdx.x % vecs_slice) * 16;
        x = *reinterpret_cast<const uint4*>(
            pages + row_offset(fp, kvh, src % p.geom.page_size, p.geom) * elem_bytes + v);
        dst = pages + row_offset(tp, kvh, j % p.geom.page_size, p.geom) * elem_bytes + v;
      }
    }
    __syncthreads();  // every row of this step is read
    if (dst) *reinterpret_cast<uint4*>(dst) = x;
  }
}

template <class F>
cudaError_t by_type(int dt, F f) {
  if (dt == DT_F32) f(float());
  else if (dt == DT_F16) f(__half());
  else f(__nv_bfloat16());
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, cudaStream_t s) {
  if (p.tokens == 0) return cudaSuccess;
  const unsigned grid = (unsigned)std::min<int64_t>(p.tokens, 148 * 16);
  return by_type(p.page_dt, [&](auto t) { kv_append_kernel<decltype(t)><<<grid, 256, 0, s>>>(p); });
}

cudaError_t launch_kv_attend(const KvAttendParams& p, cudaStream_t s) {
  if (p.batch == 0) return cudaSuccess;
  cudaError_t e = p.page_dt == DT_F32   ? launch_kv_attend_f32(p, s)
                  : p.page_dt == DT_F16 ? launch_kv_attend_f16(p, s)
                                        : launch_kv_attend_bf16(p, s);
  if (e == cudaSuccess && p.weights_out) {
    kv_weights_kernel<<<dim3((unsigned)(p.batch * p.geom.kv_heads), 16), 256, 0, s>>>(p);
    e = cudaGetLastError();
  }
  return e;
}

cudaError_t launch_kv_evict(const KvEvictParams& p, cudaStream_t s) {
  if (p.batch == 0) return cudaSuccess;
  const unsigned pairs = (unsigned)(p.batch * p.geom.kv_heads);
  kv_select_kernel<<<pairs, kSelectThreads, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int es = p.page_dt == DT_F32 ? 4 : 2, row_vecs = p.geom.head_dim * es / 16;
  const int slice = row_vecs % 2 == 0 ? 2 : 1;
  kv_move_kernel<<<dim3(pairs, 2 * row_vecs / slice), kMoveThreads, 0, s>>>(p, slice, es);
  return cudaGetLastError();
}

}  // namespace kern
}  // namespace gawee
