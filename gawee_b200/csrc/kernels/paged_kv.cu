// Kernels of the paged key/value cache: append, attention of one new token
// over the pages, and eviction by accumulated attention weight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>

#include "paged_kv.h"

namespace gawee {
namespace kern {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void set_status(int* st, int code) {
  if (st) atomicCAS(st, 0, code);
}

// --- element types ----------------------------------------------------------
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Element i of an activation array whose type is only known at run time: the
// few values a block reads once or writes once.
__device__ __forceinline__ float load_act(const void* p, int dt, int64_t i) {
  if (dt == DT_F32) return static_cast<const float*>(p)[i];
  if (dt == DT_F16) return to_f(static_cast<const __half*>(p)[i]);
  return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_act(void* p, int dt, int64_t i, float x) {
  if (dt == DT_F32) static_cast<float*>(p)[i] = x;
  else if (dt == DT_F16) static_cast<__half*>(p)[i] = from_f<__half>(x);
  else static_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(x);
}

// Eight consecutive values of a 16-byte aligned row.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f(h[i]);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// --- append -------------------------------------------------------------------
// One thread per element of a token's row over the heads.
template <class T>
__global__ void kv_append_kernel(KvAppendParams p) {
  const int row = p.geom.kv_heads * p.geom.head_dim;
  for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const int64_t seq = p.sequences ? (int64_t)p.sequences[t] : t;
    int64_t pos = p.positions[t];
    if (p.last) pos = pos > p.last ? -1 : pos - 1;
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

// --- attend --------------------------------------------------------------------
// One block per (sequence, key/value head, chunk of query heads).  A warp takes
// every fourth key; lane l holds elements 8l .. 8l+7 of the row.
constexpr int kAttendThreads = 128;

template <class T>
__global__ void __launch_bounds__(kAttendThreads) kv_attend_kernel(KvAttendParams p) {
  constexpr int kWarps = kAttendThreads / 32;
  const int D = p.geom.head_dim, group = p.heads / p.geom.kv_heads;
  const int chunks = (group + kKvHeadChunk - 1) / kKvHeadChunk;
  const int chunk = blockIdx.x % chunks, kvh = blockIdx.x / chunks % p.geom.kv_heads;
  const int b = blockIdx.x / chunks / p.geom.kv_heads;
  const int h0 = kvh * group + chunk * kKvHeadChunk, nh = min(kKvHeadChunk, group - chunk * kKvHeadChunk);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool active = lane * 8 < D;
  int64_t len = p.lengths[b];
  if (len < 0) return;
  if (len > p.max_len) {
    if (threadIdx.x == 0) set_status(p.status, ST_KV_LENGTH);
    len = 0;
  }
  float q[kKvHeadChunk][8], acc[kKvHeadChunk][8], m[kKvHeadChunk], l[kKvHeadChunk];
#pragma unroll
  for (int g = 0; g < kKvHeadChunk; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[g][i] = 0.f;
      q[g][i] = active && g < nh ? load_act(p.q, p.dt, b * p.q_stride + (int64_t)(h0 + g) * D + lane * 8 + i) * p.scale
                                 : 0.f;
    }
  }
  const int32_t* table = p.table + b * p.table_stride;
  for (int64_t i = warp; i < len; i += kWarps) {
    const int64_t page = page_of(table, p.table_cols, i, p.geom);
    const float add = p.mask ? p.mask[b * p.mask_stride + i] : 0.f;
    if (page < 0 && lane == 0) set_status(p.status, ST_KV_PAGE);
    const bool out = page < 0 || add == -INFINITY;  // takes no part, whatever its rows hold
    float x[8] = {};
    const int64_t o = out ? 0 : row_offset(page, kvh, (int)(i % p.geom.page_size), p.geom) + lane * 8;
    if (active && !out) load8(static_cast<const T*>(p.k_pages) + o, x);
    float s[kKvHeadChunk];
#pragma unroll
    for (int g = 0; g < kKvHeadChunk; ++g) {
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) d = fmaf(q[g][j], x[j], d);
      s[g] = out ? -INFINITY : warp_sum(d) + add;
    }
    if (p.weights_out && lane == 0)
      for (int g = 0; g < nh; ++g) p.scores[((int64_t)b * p.heads + h0 + g) * p.max_len + i] = s[g];
    if (out) continue;
    if (active) load8(static_cast<const T*>(p.v_pages) + o, x);
#pragma unroll
    for (int g = 0; g < kKvHeadChunk; ++g) {
      const float mn = fmaxf(m[g], s[g]);
      const float c = mn == -INFINITY ? 1.f : exp2f((m[g] - mn) * kLog2e);
      const float e = mn == -INFINITY ? 0.f : exp2f((s[g] - mn) * kLog2e);
      m[g] = mn;
      l[g] = l[g] * c + e;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[g][j] = fmaf(e, x[j], acc[g][j] * c);
    }
  }
  // join the warps
  __shared__ float sm[kWarps][kKvHeadChunk], sl[kWarps][kKvHeadChunk], so[kWarps][256];
#pragma unroll
  for (int g = 0; g < kKvHeadChunk; ++g)
    if (lane == 0) {
      sm[warp][g] = m[g];
      sl[warp][g] = l[g];
    }
  __syncthreads();
  for (int g = 0; g < nh; ++g) {
    float mt = -INFINITY, lt = 0.f;
    for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sm[w][g]);
    for (int w = 0; w < kWarps; ++w) lt += sm[w][g] == -INFINITY ? 0.f : sl[w][g] * exp2f((sm[w][g] - mt) * kLog2e);
#pragma unroll
    for (int gg = 0; gg < kKvHeadChunk; ++gg)
      if (gg == g && active)
#pragma unroll
        for (int j = 0; j < 8; ++j) so[warp][lane * 8 + j] = acc[gg][j];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kAttendThreads) {
      float o = 0.f;
      for (int w = 0; w < kWarps; ++w) o += sm[w][g] == -INFINITY ? 0.f : so[w][d] * exp2f((sm[w][g] - mt) * kLog2e);
      store_act(p.out, p.dt, b * p.out_stride + (int64_t)(h0 + g) * D + d, lt != 0.f ? o / lt : 0.f);
    }
    if (p.weights_out && threadIdx.x == 0) {
      p.stats[((int64_t)b * p.heads + h0 + g) * 2] = mt;
      p.stats[((int64_t)b * p.heads + h0 + g) * 2 + 1] = lt;
    }
    __syncthreads();
  }
}

// weights_out = weights + the attention weights of this step, summed over the
// query heads of the key/value head in their order.
__global__ void kv_weights_kernel(KvAttendParams p) {
  const int kvh = blockIdx.x % p.geom.kv_heads, b = blockIdx.x / p.geom.kv_heads;
  const int group = p.heads / p.geom.kv_heads;
  const int64_t len = p.lengths[b];
  if (len > p.max_len) return;
  for (int64_t i = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; i < len; i += (int64_t)gridDim.y * blockDim.x) {
    float w = 0.f;
    for (int g = 0; g < group; ++g) {
      const int64_t row = (int64_t)b * p.heads + kvh * group + g;
      const float s = p.scores[row * p.max_len + i], m = p.stats[row * 2], l = p.stats[row * 2 + 1];
      w += s == -INFINITY ? 0.f : exp2f((s - m) * kLog2e) / l;
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
  if (p.k) {
    // the new token of sequence b is its last row
    KvAppendParams a{};
    a.geom = p.geom;
    a.k_pages = p.k_pages;
    a.v_pages = p.v_pages;
    a.page_dt = p.page_dt;
    a.k = p.k;
    a.v = p.v;
    a.dt = p.dt;
    a.k_stride = p.k_stride;
    a.v_stride = p.v_stride;
    a.tokens = p.batch;
    a.positions = p.lengths;
    a.table = p.table;
    a.table_stride = p.table_stride;
    a.table_cols = p.table_cols;
    a.batch = p.batch;
    a.last = p.max_len;
    a.status = p.status;
    if (cudaError_t e = launch_kv_append(a, s)) return e;
  }
  const int group = p.heads / p.geom.kv_heads, chunks = (group + kKvHeadChunk - 1) / kKvHeadChunk;
  const unsigned grid = (unsigned)(p.batch * p.geom.kv_heads * chunks);
  cudaError_t e = by_type(p.page_dt, [&](auto t) { kv_attend_kernel<decltype(t)><<<grid, kAttendThreads, 0, s>>>(p); });
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
