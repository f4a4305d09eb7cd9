// Kernels of the paged key/value cache: append, the join and the
// weights of attend (the attention itself is in paged_attend.cuh) and eviction by
// accumulated attention weight.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdint>

#include "paged_common.cuh"

namespace gawee {
namespace kern {

using namespace paged;

namespace {

// --- append -------------------------------------------------------------------
// A thread takes 16-byte vectors of a token's row over the heads, of K and of V.
// The floor is HBM bandwidth; many tokens are on the way at once, but a block's work
// is short and begins with the chain sequence and position -> page -> row.
// 13,786 tokens of 8 x 128, fp32 to bf16 pages of 16 rows: 35 us, 4.8 TB/s, 0.73 of
// the copy rate (an element a thread: 68 us); 63 tokens: 2.2 us.
constexpr int kAppendThreads = 256;

// `n` consecutive values as fp32; 16-byte loads where the caller knows the alignment.
template <class A, int N, bool ALIGNED>
__device__ __forceinline__ void load_n(const A* p, float (&x)[N]) {
  if constexpr (ALIGNED) {
    constexpr int kPer = 16 / sizeof(A), kV = N >= kPer ? N / kPer : 1;
    if constexpr (N >= kPer) {
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const uint4 a = *reinterpret_cast<const uint4*>(p + v * kPer);
        const A* e = reinterpret_cast<const A*>(&a);
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[v * kPer + i] = to_f(e[i]);
      }
    } else {  // four 16-bit values: 8 bytes
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      const A* e = reinterpret_cast<const A*>(&a);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = to_f(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f(p[i]);
  }
}

template <class T, class A, bool ALIGNED>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(KvAppendParams p, int lanes) {
  constexpr int kPer = 16 / sizeof(T);
  const int64_t t = (int64_t)blockIdx.x * (kAppendThreads / lanes) + threadIdx.x / lanes;
  if (t >= p.tokens) return;
  const int64_t seq = p.sequences ? (int64_t)p.sequences[t] : t;
  const int64_t pos = p.positions[t];
  const int lane = threadIdx.x % lanes, head_vecs = p.geom.head_dim / kPer, vecs = p.geom.kv_heads * head_vecs;
  const A *k = static_cast<const A*>(p.k) + t * p.k_stride, *v = static_cast<const A*>(p.v) + t * p.v_stride;
  // the first vectors are on the way while the page is looked up
  float x[kPer], y[kPer];
  if (lane < vecs) {
    load_n<A, kPer, ALIGNED>(k + lane * kPer, x);
    load_n<A, kPer, ALIGNED>(v + lane * kPer, y);
  }
  if (seq < 0 || pos < 0) return;
  const int64_t page = seq < p.batch ? page_of(p.table + seq * p.table_stride, p.table_cols, pos, p.geom) : -1;
  if (page < 0) {
    if (lane == 0) set_status(p.status, seq < p.batch ? ST_KV_PAGE : ST_KV_SEQUENCE);
    return;
  }
  const int slot = (int)(pos % p.geom.page_size);
  for (int i = lane; i < vecs; i += lanes) {
    const int64_t o = row_offset(page, i / head_vecs, slot, p.geom) + i % head_vecs * kPer;
    if (i != lane) {
      load_n<A, kPer, ALIGNED>(k + i * kPer, x);
      load_n<A, kPer, ALIGNED>(v + i * kPer, y);
    }
    uint4 a, b;
    T *ka = reinterpret_cast<T*>(&a), *va = reinterpret_cast<T*>(&b);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      ka[e] = from_f<T>(x[e]);
      va[e] = from_f<T>(y[e]);
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(p.k_pages) + o) = a;
    *reinterpret_cast<uint4*>(static_cast<T*>(p.v_pages) + o) = b;
  }
}

// --- the join of attend ------------------------------------------------------------
//
// A segment that several blocks of the attention shared is joined here, a block per query
// head: the parts' maxima and sums give each part's factor, and groups of
// threads add the scaled parts, in a fixed order.  A block of the attention leaves at most one
// segment unfinished behind it, so the grid is over the blocks of the attention
// or over the segments, whichever are fewer (bf16, 32/8 heads x 128: 64 of up to 512
// rows, 512 segments on 296 blocks, 29.0 us in all, over the segments 31.8; one
// of 16,385 rows, 8 segments, 21.3, over the blocks 22.3).  Further blocks add the
// weights of this step to their accumulators, over the query heads of a
// key/value head in their order.  Both are short of work and bound by latency
// (a block of the attention itself that joined 148 parts took 7 us more), so the
// grid is launched while the attention runs and waits for its end.
constexpr int kJoinThreads = 256;

// A head's maximum and sum over its n parts, from the whole warp; `first` the segment's first block.
__device__ __forceinline__ float2 join_stats(const KvAttendParams& p, int heads, int first, int n, int h) {
  const int lane = threadIdx.x % 32, part = kv_part_vecs(heads, p.geom.head_dim);
  const float4* parts = reinterpret_cast<const float4*>(p.parts);
  float mt = -INFINITY, lt = 0.f;
  for (int i0 = 0; i0 < n; i0 += 128) {
    float2 x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + r * 32 + lane;
      x[r] = i < n ? reinterpret_cast<const float2*>(parts + (i == 0 ? 2 * first + 1 : 2 * (first + i)) * part)[h]
                   : make_float2(-INFINITY, 0.f);
    }
    float m = mt;
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, x[r].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    lt *= exp_from(mt, m);
#pragma unroll
    for (int r = 0; r < 4; ++r) lt += x[r].y * exp_from(x[r].x, m);
    mt = m;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) lt += __shfl_xor_sync(0xffffffffu, lt, o);
  return make_float2(mt, lt);
}

__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const __grid_constant__ KvAttendParams p, int heads,
                                                               int joins, bool by_segment, int stretches) {
  extern __shared__ float4 s_join[];
  const int kv = p.geom.kv_heads, D = p.geom.head_dim, group = p.heads / kv, chunks = (group + heads - 1) / heads;
  const int tid = threadIdx.x, warp = tid / 32;
  const bool none = (int)blockIdx.x < joins && by_segment &&  // lengths were there before the attention began
                    p.lengths[blockIdx.x / min(heads, group) / chunks / kv] < 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the attention has ended and its results are visible
  if (none) return;
  if ((int)blockIdx.x < joins) {
    const int most = min(heads, group), index = blockIdx.x / most, h = blockIdx.x % most;
    int segment = index;
    int2 info;  // the segment's first block and the number of its blocks
    if (by_segment) {
      info = p.info[segment];
    } else {
      const int2 split = p.splits[index];
      segment = split.x;
      info = make_int2(index, split.y);
    }
    const int chunk = segment % chunks, kvh = segment / chunks % kv, b = segment / chunks / kv;
    const int head = chunk * heads + h;
    // a sequence outside the batch: the scratch of another call, which overlaps against the rule
    if (info.y <= 1 || head >= group || b >= p.batch) return;
    const int dv = D / 4, part = kv_part_vecs(heads, D);
    int lanes = 2;  // threads of a group: one for each 16 bytes of the row
    while (lanes < dv) lanes *= 2;
    const int groups = kJoinThreads / lanes, g = tid / lanes, x = tid % lanes;
    float4 sum = make_float4(0, 0, 0, 0);
    const float4* parts = reinterpret_cast<const float4*>(p.parts);
    constexpr int kAtOnce = 8;
    float4 o[kAtOnce];
    float f[kAtOnce];
    auto load = [&](int i0) {
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) {
        const int i = i0 + r * groups;
        const float4* q = parts + (i == 0 ? 2 * info.x + 1 : 2 * (info.x + i)) * part;
        const bool in = i < info.y && x < dv;
        f[r] = in ? reinterpret_cast<const float2*>(q)[h].x : -INFINITY;
        o[r] = in ? q[kv_part_head(heads) + h * dv + x] : make_float4(0, 0, 0, 0);
      }
    };
    load(g);  // on the way while the statistics are formed
    const float2 top = join_stats(p, heads, info.x, info.y, h);  // every warp for itself
    for (int i0 = g;;) {
#pragma unroll
      for (int r = 0; r < kAtOnce; ++r) add_scaled(sum, o[r], exp_from(f[r], top.x));
      i0 += kAtOnce * groups;
      if (i0 >= info.y) break;
      load(i0);
    }
    s_join[tid] = sum;
    __syncthreads();
    if (g == 0 && x < dv) {
      for (int r = 1; r < groups; ++r) {
        const float4 o = s_join[r * lanes + x];
        add_scaled(sum, o, 1.f);
      }
      store_result(p, b, kvh * group + head, x * 4, top.x, top.y, sum);
    }
    return;
  }
  // the weights: several blocks a sequence and key/value head
  const int pair = (blockIdx.x - joins) / stretches, stretch = (blockIdx.x - joins) % stretches;
  const int kvh = pair % kv, b = pair / kv;
  int len = p.lengths[b];
  if (len > p.max_len) len = 0;
  if ((int64_t)stretch * kJoinThreads >= len) return;
  float2* s_head = reinterpret_cast<float2*>(s_join);  // maximum and 1 / sum of each query head of the group
  for (int g = warp; g < group; g += kJoinThreads / 32) {
    const int2 info = p.info[pair * chunks + g / heads];
    const float2 top = info.y > 1 ? join_stats(p, heads, info.x, info.y, g % heads)
                                  : reinterpret_cast<const float2*>(p.stats)[(int64_t)b * p.heads + kvh * group + g];
    if (tid % 32 == 0) s_head[g] = make_float2(top.x, 1.f / top.y);
  }
  __syncthreads();
  for (int i = stretch * kJoinThreads + tid; i < len; i += stretches * kJoinThreads) {
    const float* s = p.scores + ((int64_t)pair * p.max_len + i) * group;
    const float before = p.weights ? p.weights[b * p.w_batch + kvh * p.w_stride + i] : 0.f;
    float w = 0.f;
    for (int g = 0; g < group; ++g) {
      const float2 t = s_head[g];
      w += s[g] == -INFINITY ? 0.f : exp_from(s[g], t.x) * t.y;
    }
    p.weights_out[b * p.wo_batch + kvh * p.wo_stride + i] = before + w;
  }
}

// --- evict ---------------------------------------------------------------------
//
// Selection: a cluster of blocks per (sequence, key/value head), each a
// contiguous range of the positions.  The smallest weight that stays is found
// by radix selection over the bits of weight_key, 11 + 11 + 10 of them, with
// the blocks' histograms summed through distributed shared memory; equal
// weights stay from the lowest position on, so a kept row's new place is
//   (kept for certain before it) + min(equal before it, equal ones that stay).
// The weights are read five times, the first time from HBM, and the bound is the
// latency of the passes: 256 pairs of up to 8192 rows 21 us, 48 of 2048 about 8.
// A block that works alone ranks the last candidates directly as soon as no more
// of them are left than it has threads: mostly after the first 11 bits.
constexpr int kBins = 2048, kMostBlocks = 8;  // of a cluster

// Weights in ascending order of their values as unsigned integers; both zeros
// are equal and NaN is below every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sums of x over the block's threads before this one, and over all; every thread calls it.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int scan = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  const int mine = lane < THREADS / 32 ? warp_sums[lane] : 0;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  total = __shfl_sync(0xffffffffu, upto, 31);
  const int before = __shfl_sync(0xffffffffu, upto - mine, warp);
  return before + scan - x;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv_select_kernel(KvEvictParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = cluster.num_blocks(), rank = cluster.block_rank();
  __shared__ __align__(16) int hist[2][kBins];
  __shared__ int warp_sums[32];
  __shared__ int s_bin, s_need, s_left;
  __shared__ uint32_t s_key[THREADS];
  __shared__ int s_at[THREADS];
  __shared__ int2 s_counts;
  const int pair = blockIdx.x / blocks;
  const int kvh = pair % p.geom.kv_heads, b = pair / p.geom.kv_heads;
  const int tid = threadIdx.x;
  int32_t* kept = p.kept + (int64_t)pair * p.budget;
  int len = p.lengths[b];
  if (len > p.max_len) {
    if (tid == 0) set_status(p.status, ST_KV_LENGTH);
    len = -1;
  }
  if (kvh == 0 && rank == 0 && tid == 0) {
    p.plan[2 * b] = len;
    p.plan[2 * b + 1] = len > p.budget ? p.budget : p.lengths[b];
  }
  if (len <= p.budget) {  // the whole cluster
    for (int j = rank * THREADS + tid; j < p.budget; j += blocks * THREADS) kept[j] = j < len ? j : -1;
    return;
  }
  const float* w = p.weights + b * p.w_batch + kvh * p.w_stride;
  const int cand = len - p.recent;  // positions below it are chosen by weight
  const int range = (len + blocks - 1) / blocks, begin = min(rank * range, len), end = min(begin + range, len);
  const int old_end = min(end, cand);
  uint32_t prefix = 0;
  int need = p.budget - p.recent;  // still to choose among the keys with this prefix
  const bool choose = need > 0;
  for (int pass = 0; pass < 3 && choose; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t above = pass == 0 ? 0u : 0xffffffffu << (shift + bits);
    int* mine = hist[pass & 1];
    for (int i = tid; i < kBins; i += THREADS) mine[i] = 0;
    __syncthreads();
    for (int base = begin; base < old_end; base += 8 * THREADS) {
      float x[8];  // eight loads on the way
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int i = base + r * THREADS + tid;
        x[r] = i < old_end ? w[i] : 0.f;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const uint32_t k = weight_key(x[r]);
        if (base + r * THREADS + tid < old_end && (k & above) == prefix)
          atomicAdd(&mine[(k >> shift) & ((1u << bits) - 1)], 1);
      }
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    // this thread's bins, from the highest down
    constexpr int kEach = kBins / THREADS;
    const int lo = kBins - kEach * (tid + 1);
    int h[kEach] = {}, sum = 0;
    if (blocks == 1) {
#pragma unroll
      for (int x = 0; x < kEach; ++x) h[x] = mine[lo + x];
    } else {
#pragma unroll
      for (int r = 0; r < kMostBlocks; ++r)
        if (r < blocks) {
          const int2* theirs = reinterpret_cast<const int2*>(cluster.map_shared_rank(mine, r) + lo);
#pragma unroll
          for (int x = 0; x < kEach; x += 2) {
            const int2 y = theirs[x / 2];
            h[x] += y.x;
            h[x + 1] += y.y;
          }
        }
    }
#pragma unroll
    for (int x = 0; x < kEach; ++x) sum += h[x];
    int total;
    int before = block_scan<THREADS>(sum, warp_sums, total);
#pragma unroll
    for (int x = kEach - 1; x >= 0; --x) {
      if (before < need && before + h[x] >= need) {
        s_bin = lo + x;
        s_need = need - before;
        s_left = h[x];
      }
      before += h[x];
    }
    __syncthreads();
    prefix |= (uint32_t)s_bin << shift;
    need = s_need;
    // a block clears this histogram again only two passes on, behind the next cluster.sync
    if (blocks == 1 && shift && s_left <= THREADS) {
      const int left = s_left;
      __syncthreads();
      if (tid == 0) s_left = 0;
      __syncthreads();
      const uint32_t upto = 0xffffffffu << shift;
      for (int base = begin; base < old_end; base += 8 * THREADS) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int i = base + r * THREADS + tid;
          x[r] = i < old_end ? w[i] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int i = base + r * THREADS + tid;
          const uint32_t k = weight_key(x[r]);
          if (i < old_end && (k & upto) == prefix) {
            const int at = atomicAdd(&s_left, 1);
            if (at < THREADS) {  // more of them only if the weights change meanwhile
              s_key[at] = k;
              s_at[at] = i;
            }
          }
        }
      }
      __syncthreads();
      if (tid < left) {
        const uint32_t k = s_key[tid];
        const int i = s_at[tid];
        int greater = 0, first = 0;
        for (int x = 0; x < left; ++x) {
          greater += s_key[x] > k;
          first += s_key[x] == k && s_at[x] < i;
        }
        if (greater + first == need - 1) {  // the last one that stays
          s_bin = (int)k;
          s_need = need - greater;
        }
      }
      __syncthreads();
      prefix = (uint32_t)s_bin;
      need = s_need;
      break;
    }
  }
  // keys above `prefix` and the recent rows stay for certain, and the first `need` of those equal to it
  auto classify = [&](int i, float x, int& sure, int& equal) {
    const uint32_t k = weight_key(x);
    const bool old = choose && i < old_end;
    sure = i < end && (i >= cand || (old && k > prefix));
    equal = old && k == prefix;
  };
  int sure_before = 0, equal_before = 0;
  if (blocks > 1) {  // how many of each lie in the blocks before
    int sure = 0, equal = 0;
    for (int base = begin; base < end; base += 8 * THREADS) {
      float x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int i = base + r * THREADS + tid;
        x[r] = i < old_end ? w[i] : 0.f;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        int a, e;
        classify(base + r * THREADS + tid, x[r], a, e);
        sure += a;
        equal += e;
      }
    }
    int all_sure, all_equal;
    block_scan<THREADS>(sure, warp_sums, all_sure);
    block_scan<THREADS>(equal, warp_sums, all_equal);
    if (tid == 0) s_counts = make_int2(all_sure, all_equal);
    cluster.sync();
#pragma unroll
    for (int r = 0; r < kMostBlocks; ++r)
      if (r < rank) {
        const int2 x = *cluster.map_shared_rank(&s_counts, r);
        sure_before += x.x;
        equal_before += x.y;
      }
    cluster.sync();  // no block leaves while its shared memory is read
  }
  constexpr int kEach = 4;  // consecutive positions of a thread
  for (int base = begin; base < end; base += THREADS * kEach) {
    int a[kEach], e[kEach], packed = 0;
    float y[kEach];
#pragma unroll
    for (int x = 0; x < kEach; ++x) y[x] = base + tid * kEach + x < old_end ? w[base + tid * kEach + x] : 0.f;
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      classify(base + tid * kEach + x, y[x], a[x], e[x]);
      packed += a[x] | e[x] << 16;
    }
    int total;
    const int before = block_scan<THREADS>(packed, warp_sums, total);
    int s = sure_before + (before & 0xffff), q = equal_before + (before >> 16);
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
      const int place = s + min(q, need);
      if ((a[x] || (e[x] && q < need)) && place < p.budget) kept[place] = base + tid * kEach + x;
      s += a[x];
      q += e[x];
    }
    sure_before += total & 0xffff;
    equal_before += total >> 16;
  }
}

// Moves the kept rows to their places and their weights with them.
//
// To other pages, every row is free to move: a block takes a range of rows.
// In place, row j goes to a place at or before its own, and a place may be
// written only when what lies there has been read: a block takes a slice of
// the rows' 16-byte vectors, all rows of it in ascending order, and writes
// each step's rows after the whole step is read; slices are as narrow as it
// takes to occupy the GPU.  The last block of a pair moves its weights.  Bound by
// HBM: 256 pairs, up to 2048 rows of 256 bytes each, to other pages: 95 us, 5.2 TB/s.
//
// Calls that overlap against the rule exchange their `plan`, and weights that
// change during a call its selection: every position is checked before it is
// used, so that they spoil no more than the results.
constexpr int kMoveThreads = 256, kMoveRows = 4;  // rows of a thread in a step

template <bool IN_PLACE>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(KvEvictParams p, int vecs, int elem_bytes, int row_blocks) {
  const int kvh = blockIdx.x % p.geom.kv_heads, b = blockIdx.x / p.geom.kv_heads;
  const int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
  const int tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the selection has ended
  const int len = (int)min((int64_t)p.plan[2 * b], p.max_len), left = max(min(len, p.budget), 0);
  float* wo = p.weights_out + b * p.wo_batch + kvh * p.wo_stride;
  // zeros from the new length to the old one: by all blocks, or, where the
  // weights themselves are overwritten, by the block that has read them
  const bool alone = p.weights == p.weights_out;
  const int fill_blocks = alone ? 1 : row_blocks + 1, fill_block = alone ? 0 : (int)blockIdx.y;
  auto fill = [&] {
    for (int j = left + fill_block * kMoveThreads + tid; j < len; j += fill_blocks * kMoveThreads) wo[j] = 0.f;
  };
  if ((int)blockIdx.y == row_blocks) {  // the weights
    if (kvh == 0 && tid == 0) p.lengths_out[b] = p.plan[2 * b + 1];
    const float* w = p.weights + b * p.w_batch + kvh * p.w_stride;
    constexpr int kEach = 8;
    for (int j0 = 0; j0 < left; j0 += kMoveThreads * kEach) {
      float x[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int j = j0 + e * kMoveThreads + tid;
        const int src = j < left ? kept[j] : -1;
        x[e] = src >= 0 && src < len ? w[src] : 0.f;
      }
      __syncthreads();  // read before they are written over
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int j = j0 + e * kMoveThreads + tid;
        if (j < left) wo[j] = x[e];
      }
    }
    __syncthreads();
    fill();
    return;
  }
  if (!alone) fill();
  const int32_t* from = p.table + b * p.table_stride;
  const int32_t* to = IN_PLACE ? from : p.to_table + b * p.to_stride;
  const int64_t to_cols = IN_PLACE ? p.table_cols : p.to_cols;
  const int row_vecs = p.geom.head_dim * elem_bytes / 16;
  // in place: the block's slice of K or of V; else all of K's rows and all of V's
  const int slices = row_vecs / vecs, slice = IN_PLACE ? blockIdx.y % slices : 0;
  char* pages = static_cast<char*>(IN_PLACE && (int)blockIdx.y >= slices ? p.v_pages : p.k_pages);
  const long long to_v = static_cast<char*>(p.v_pages) - static_cast<char*>(p.k_pages);
  const int rows = kMoveThreads / vecs, row = tid / vecs, at = (slice * vecs + tid % vecs) * 16;
  const int step = rows * kMoveRows;
  const int first = IN_PLACE ? 0 : (int)blockIdx.y * step, stride = IN_PLACE ? step : row_blocks * step;
  for (int j0 = first; j0 < p.budget; j0 += stride) {
    uint4 x[kMoveRows], y[kMoveRows];
    char* dst[kMoveRows];
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r) {
      const int j = j0 + r * rows + row;
      dst[r] = nullptr;
      if (row >= rows || j >= p.budget) continue;
      const int src = kept[j];
      if (src < 0 || (IN_PLACE && src == j)) continue;
      const int64_t fp = page_of(from, p.table_cols, src, p.geom), tp = page_of(to, to_cols, j, p.geom);
      if (fp < 0 || tp < 0) {
        set_status(p.status, ST_KV_PAGE);
        continue;
      }
      const char* a = pages + row_offset(fp, kvh, src % p.geom.page_size, p.geom) * elem_bytes + at;
      x[r] = *reinterpret_cast<const uint4*>(a);
      if (!IN_PLACE) y[r] = *reinterpret_cast<const uint4*>(a + to_v);
      dst[r] = pages + row_offset(tp, kvh, j % p.geom.page_size, p.geom) * elem_bytes + at;
    }
    if (IN_PLACE) __syncthreads();  // every row of this step is read
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r)
      if (dst[r]) {
        *reinterpret_cast<uint4*>(dst[r]) = x[r];
        if (!IN_PLACE) *reinterpret_cast<uint4*>(dst[r] + to_v) = y[r];
      }
  }
}

template <class F>
cudaError_t by_type(int dt, F f) {
  if (dt == DT_F32) f(float());
  else if (dt == DT_F16) f(__half());
  else f(__nv_bfloat16());
  return cudaGetLastError();
}

int elem_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, cudaStream_t s) {
  if (p.tokens == 0) return cudaSuccess;
  const int vecs = p.geom.kv_heads * p.geom.head_dim * elem_bytes(p.page_dt) / 16;
  int lanes = 1;  // threads of a token
  while (lanes < vecs && lanes < kAppendThreads) lanes *= 2;
  const int per_block = kAppendThreads / lanes;
  const unsigned grid = (unsigned)((p.tokens + per_block - 1) / per_block);
  const int es = elem_bytes(p.dt);
  const bool aligned = reinterpret_cast<uintptr_t>(p.k) % 16 == 0 && reinterpret_cast<uintptr_t>(p.v) % 16 == 0 &&
                       (p.tokens == 1 || (p.k_stride * es % 16 == 0 && p.v_stride * es % 16 == 0));
  return by_type(p.page_dt, [&](auto t) {
    by_type(p.dt, [&](auto a) {
      if (aligned) kv_append_kernel<decltype(t), decltype(a), true><<<grid, kAppendThreads, 0, s>>>(p, lanes);
      else kv_append_kernel<decltype(t), decltype(a), false><<<grid, kAppendThreads, 0, s>>>(p, lanes);
    });
  });
}

cudaError_t launch_kv_attend(const KvAttendParams& given, cudaStream_t s) {
  if (given.batch == 0) return cudaSuccess;
  KvAttendParams p = given;
  auto rows_aligned = [&](const void* at, int64_t stride) {
    return reinterpret_cast<uintptr_t>(at) % 16 == 0 && (p.batch == 1 || stride * elem_bytes(p.dt) % 16 == 0);
  };
  p.k_as_stored = p.k && p.dt == p.page_dt && rows_aligned(p.k, p.k_stride) && rows_aligned(p.v, p.v_stride);
  KvAttendShape shape{};
  cudaError_t e = p.page_dt == DT_F32   ? launch_kv_attend_f32(p, &shape, s)
                  : p.page_dt == DT_F16 ? launch_kv_attend_f16(p, &shape, s)
                                        : launch_kv_attend_bf16(p, &shape, s);
  if (e != cudaSuccess || !(shape.split || p.weights_out)) return e;
  const int group = p.heads / p.geom.kv_heads, pairs = p.batch * p.geom.kv_heads;
  const int64_t segments = (int64_t)pairs * ((group + shape.heads - 1) / shape.heads);
  const bool by_segment = segments <= shape.blocks;
  const int joins = shape.split ? (int)std::min<int64_t>(segments, shape.blocks) * std::min(shape.heads, group) : 0;
  int stretches = 0;
  size_t smem = sizeof(float4) * kJoinThreads;
  if (p.weights_out) {
    // about eight blocks an SM over all pairs; a block beyond a sequence's end leaves at once
    const int64_t most = (p.max_len + kJoinThreads - 1) / kJoinThreads;
    const int64_t want = std::max<int64_t>(1, (8ll * p.sms + pairs - 1) / pairs);
    stretches = (int)std::min(most, want);
    smem = std::max(smem, sizeof(float2) * group);
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cfg.gridDim = dim3((unsigned)joins + (unsigned)pairs * stretches);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_join_kernel, p, shape.heads, joins, by_segment, stretches);
}

cudaError_t launch_kv_evict(const KvEvictParams& p, cudaStream_t s) {
  if (p.batch == 0) return cudaSuccess;
  const int pairs = p.batch * p.geom.kv_heads;
  // Threads of a block: 1024, or 256 where a thread then has 16 positions at
  // most; eight such blocks on an SM hide each other's waits (75 x 6 pairs of up to 400
  // rows of 32, cut to 23: 11.7 us; with 1024 threads 21.8).  Blocks of a pair's cluster: doubled
  // while each keeps 2048 positions and the clusters of 1024 threads find room at once, at 96 blocks
  // (1 x 8 pairs of 65,537 rows of 128, cut to 4097: 73 us alone, 42 with 4, 37 with 8; 5 x 4
  // pairs of 25,551 rows of 64, cut to 1024: 50 us alone, 27 with 4, but 39 with 8, in two waves).
  const bool small = p.max_len <= 4096;
  int cluster = 1;
  while (!small && cluster < kMostBlocks && pairs * cluster * 2 <= 96 && p.max_len / (cluster * 2) >= 2048) cluster *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cfg.gridDim = dim3((unsigned)(pairs * cluster));
  cfg.blockDim = dim3(small ? 256 : 1024);
  cfg.stream = s;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, small ? kv_select_kernel<256> : kv_select_kernel<1024>, p)) return e;

  // the move takes its place while the selection runs, and waits for its end
  cfg.blockDim = dim3(kMoveThreads);
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;

  const int es = elem_bytes(p.page_dt), row_vecs = p.geom.head_dim * es / 16;
  if (p.to_table) {
    const int step = kMoveThreads / row_vecs * kMoveRows;
    const int64_t want = std::max<int64_t>(1, (16ll * p.sms + pairs - 1) / pairs);
    const int blocks = (int)std::min<int64_t>((p.budget + step - 1) / step, std::min<int64_t>(want, 65534));
    cfg.gridDim = dim3((unsigned)pairs, (unsigned)blocks + 1);
    return cudaLaunchKernelEx(&cfg, kv_move_kernel<false>, p, row_vecs, es, blocks);
  } else {
    int vecs = row_vecs;  // of a slice: halved while the slices leave SMs idle
    while (vecs % 2 == 0 && (int64_t)pairs * 2 * (row_vecs / vecs) < 8ll * p.sms) vecs /= 2;
    const int slices = row_vecs / vecs;
    cfg.gridDim = dim3((unsigned)pairs, (unsigned)(2 * slices + 1));
    return cudaLaunchKernelEx(&cfg, kv_move_kernel<true>, p, vecs, es, 2 * slices);
  }
}

}  // namespace kern
}  // namespace gawee
