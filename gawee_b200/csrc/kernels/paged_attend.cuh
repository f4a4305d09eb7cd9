// Attention of one new token per sequence over a paged key/value cache.
//
//   s_i = scale * (q . K_i) + mask_i,  p = softmax(s),  out = sum_i p_i V_i
//
// Every cached byte is read once and takes part in a few operations, so the
// bound is HBM bandwidth (with few query heads to a key/value head) and the
// kernel is built to keep loads in flight:
//
//   * The keys of a (sequence, key/value head, chunk of query heads) segment
//     are cut into tiles, and all tiles of the batch, in order, are divided
//     evenly over a fixed grid of resident blocks: a block takes a contiguous
//     run of tiles, whatever the lengths are, and goes through several short
//     segments or through a part of a long one.  A segment's begin and end cost
//     as much as a tile or two, and count like them.  The lengths are read on the
//     device, so the balance needs nothing from the host.
//   * A warp takes its own rows of each tile, through a ring of shared-memory
//     stages of its own that cp.async fills: warps wait for no other until
//     the segment ends, and loads run ahead over segment borders.  Page
//     numbers and mask values are fetched one tile ahead of the loads.
//   * Each warp keeps a running maximum, sum and weighted value sum (online
//     softmax, fp32).  At the end of a segment the warps' states are joined in
//     shared memory; a block that has only a part of the segment leaves its
//     state in the workspace, and kv_join_kernel (paged_kv.cu) joins the parts in their order.
//
// Measured, with the join, in a captured graph: 32 sequences of up to 8192 rows,
// 32/8 heads x 128, bf16: 103 us, 5.8 TB/s, 0.88 of the copy rate; one of 131,071
// rows: 87 us, 6.2 TB/s; 64 of up to 2048 rows, 9/3 heads x 64, fp32: 30 us,
// 3.7 TB/s, bound by latency: three warps a scheduler that wait for loads and for each
// other use 39 % of the issue slots and 57 % of DRAM; one of 257 rows, 6 heads x 48: 8 us, a
// chain of lookups.
//
// Rows that the mask takes out, rows behind the length and rows of bad pages
// are not loaded: their stage rows are filled with zeros and their score is
// -inf, so that whatever memory holds there, or the query, cannot reach the result.
#pragma once

#include <algorithm>
#include <atomic>

#include "paged_common.cuh"

namespace gawee {
namespace kern {
namespace paged {

constexpr int kWarps = kKvWarps;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxBlocksPerSm = kKvMaxBlocksPerSm;
constexpr int kMaxSmem = 220 * 1024;  // of a block, beside the kernel's static variables
constexpr int kMaxDevices = 64;

// --- small pieces -------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes from global to shared memory; zeros where !valid (src is then not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Two fp32 multiply-adds in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// A key's score with its mask value added: -inf where that is -inf, also for a
// query that is not finite, whose product with the zeros of the row is NaN.
__device__ __forceinline__ float masked(float s, float add) { return add == -INFINITY ? -INFINITY : s; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// --- the two ways to compute a tile ---------------------------------------------
//
// Lanes: any types, all products in fp32, two to an instruction.  A warp's tile
// has TK = 128 / L keys of D <= 8 L elements: 8 KB of K and V in fp32, 4 KB in 16 bits.
//   scores: W lanes share a key (or two) and take every W-th 16-byte chunk of its
//     row; the query heads come from shared memory, the same address for all
//     keys, so that a score takes its multiplications, a few additions over W lanes and no more.
//   values: L lanes hold the row's elements, eight each, for 32 / L keys at a
//     time, and the weights come from shared memory.
// Chunks are swizzled (rows padded, where a row's chunks are no multiple of
// eight) so that the keys of either pattern lie in different banks.  With FULL,
// D is 8 L: known to the compiler, no lane idle.
template <class T_, int L, int NH_, bool FULL>
struct LaneTile {
  using T = T_;
  static constexpr int NH = NH_;
  static constexpr int TK = kv_warp_keys(L);  // keys of a warp's tile
  static constexpr int kKeysAtOnce = 32 / L, kSteps = TK / kKeysAtOnce;
  // Lanes that share a key, and the keys that they take at once: two for long
  // fp32 rows and several heads, where the reads of the queries would fill shared
  // memory's time (one of 65,536 rows, 32/4 heads x 128: 69 us, with one key 77; 8 of up to
  // 8192, 32/8 heads: 44.0, 44.6).  Over 16-bit rows one key is the faster (one of 65,536
  // rows, 16/4 heads x 128, bf16 pages: 47.2 us, with two 48.4).
  static constexpr int KL = sizeof(T) == 4 && L >= 16 && NH >= 4 ? 2 : 1;
  static constexpr int W = 32 * KL / TK, kOwn = W / KL;  // kOwn lanes end up with the same key
  // With two stages three blocks find room on an SM, with about 96 KB on the
  // way; twelve warps hide each other's waits better than eight with a third stage (64 of
  // up to 2048 rows, 9/3 x 64 heads, fp32: 29.8 us, with three stages 30.8).
  static constexpr int kStages = (NH <= 6 ? 2 : 3) * (sizeof(T) == 4 ? 1 : 2);
  static constexpr int kMinBlocks = NH <= 6 ? 3 : 2;  // of an SM: what the stages leave room for
  static constexpr int kPer = 16 / sizeof(T);         // elements of a chunk
  static constexpr int NP = NH == 1 ? 1 : (NH + 1) / 2 * 2;
  // Floats a warp: each weight twice, as the operand of a multiplication of pairs.
  static constexpr int kScratch = 2 * TK * NP;
  static constexpr int kD = FULL ? 8 * L : 0;
  using Query = float;                        // in shared memory: scaled
  static constexpr int kMaxD = 8 * L, kQueryPad = 0;
  static_assert(2 * TK * sizeof(T) >= NH * 4, "a warp's state fits into a stage");

  uint64_t acc[NH][4];
  float m[NH], l[NH];
  int D, lane, l_id, group, vecs;
  int own_key;                   // of the scores that this lane ends up with
  int qk_row, qk_xor, pv0, pv1;  // byte offsets into a tile's rows
  bool in0, in1;

  __host__ __device__ static __forceinline__ int row_bytes(int D) {
    const int n = D * (int)sizeof(T);
    if (n % 128 == 0 || W >= 8) return n;  // eight lanes read consecutive chunks of one row, or of swizzled ones
    // a distance of 16 W or -16 W modulo 128 bytes puts the keys of eight lanes into different banks
    const int up = (16 * W % 128 - n % 128 + 128) % 128, down = (128 - 16 * W % 128 - n % 128 + 256) % 128;
    return n + (up < down ? up : down);
  }
  __device__ static __forceinline__ int swizzle(int row, int D) {
    return D * (int)sizeof(T) % 128 == 0 ? row * W & 7 : 0;
  }
  __device__ static __forceinline__ int chunk_at(int row, int chunk, int D) { return chunk ^ swizzle(row, D); }

  __device__ __forceinline__ int elem(int i) const {  // element of slot i (0 .. 7) of this lane
    return sizeof(T) == 4 ? (i < 4 ? l_id * 4 + i : (l_id + L) * 4 + i - 4) : l_id * 8 + i;
  }

  __device__ static __forceinline__ float query(const void* q, int dt, int64_t i, float scale) {
    return load_act(q, dt, i) * scale;
  }
  __device__ __forceinline__ void begin(const KvAttendParams& p, const float*, int) {
    D = FULL ? 8 * L : p.geom.head_dim;
    vecs = D / kPer;
    lane = threadIdx.x % 32;
    l_id = lane % L;
    group = lane / L;
    in0 = FULL || l_id < vecs;
    in1 = FULL || l_id + L < vecs;
    const int rb = row_bytes(D), key = lane / W;
    qk_row = key * rb;
    qk_xor = swizzle(key, D) * 16;
    own_key = key + (KL == 2 && (lane & W / 2) ? TK / 2 : 0);
    // the swizzle of row st * kKeysAtOnce + group does not depend on st: kKeysAtOnce * W is a multiple of 8
    pv0 = group * rb + chunk_at(group, l_id, D) * 16;
    pv1 = group * rb + chunk_at(group, l_id + L, D) * 16;
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[g][i] = 0;
    }
  }

  // A chunk of a row as pairs of fp32 values.
  __device__ static __forceinline__ void load_chunk(const char* at, uint64_t (&x)[kPer / 2]) {
    if constexpr (sizeof(T) == 4) {
      const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(at);
      x[0] = a.x;
      x[1] = a.y;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(at);
      const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = pack2(to_f(h[2 * i]), to_f(h[2 * i + 1]));
    }
  }

  // One tile: K and V rows of TK keys, `add` their mask values, q the scaled
  // queries [NH][D] in shared memory; `live` keys from the first are within
  // the sequence.  Scores go to `scores` (nullptr: not wanted), [key][group size].
  __device__ __forceinline__ void tile(const char* ks, const char* vs, const float* add, float* scratch, const float* q,
                                       float* scores, int live, int group_size, int nh) {
    const int rb = row_bytes(D), key = own_key;
    uint64_t dot[KL][NH] = {};
    const char* krow = ks + qk_row;  // and, with two keys, TK / 2 rows on (the same swizzle: W is then 8 or more)
    const float* qw = q + lane % W * kPer;
    auto chunk = [&](int c0) {  // chunk c0 + lane % W
      uint64_t x[KL][kPer / 2];
#pragma unroll
      for (int u = 0; u < KL; ++u) load_chunk(krow + u * (TK / 2) * rb + ((c0 + lane % W) * 16 ^ qk_xor), x[u]);
#pragma unroll
      for (int g = 0; g < NH; ++g)
#pragma unroll
        for (int i = 0; i < kPer / 2; i += 2) {
          const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(qw + g * D + c0 * kPer + 2 * i);
#pragma unroll
          for (int u = 0; u < KL; ++u) {
            dot[u][g] = fma2(y.x, x[u][i], dot[u][g]);
            dot[u][g] = fma2(y.y, x[u][i + 1], dot[u][g]);
          }
        }
    };
    if constexpr (FULL) {
#pragma unroll
      for (int c0 = 0; c0 < 8 * L / kPer; c0 += W) chunk(c0);
    } else {
      for (int c0 = 0; c0 < vecs; c0 += W)
        if (c0 + lane % W < vecs) chunk(c0);
    }
    float s[NH];
    const float a = add[key];
    bool changed = false;
    float mx[NH];
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      const float2 f = unpack2(dot[0][g]);
      s[g] = f.x + f.y;
      if constexpr (KL == 2) {  // the upper half of the lanes keeps the second key
        const float2 f1 = unpack2(dot[1][g]);
        const float s1 = f1.x + f1.y;
        const bool upper = lane & W / 2;
        s[g] = (upper ? s1 : s[g]) + __shfl_xor_sync(0xffffffffu, upper ? s[g] : s1, W / 2);
      }
#pragma unroll
      for (int o = kOwn / 2; o; o >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
      s[g] = masked(s[g] + a, a);
      mx[g] = fmaxf(m[g], warp_max(s[g]));
      changed |= mx[g] != m[g];
    }
    if (scores && lane % kOwn == 0 && key < live) {
#pragma unroll
      for (int g = 0; g < NH; ++g)
        if (g < nh) scores[key * group_size + g] = s[g];
    }
    if (changed) {  // the same for all lanes
#pragma unroll
      for (int g = 0; g < NH; ++g) {
        const float c = exp_from(m[g], mx[g]);
        m[g] = mx[g];
        l[g] *= c;
        const uint64_t f = pack2(c, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] = mul2(acc[g][i], f);
      }
    }
    uint64_t* pairs = reinterpret_cast<uint64_t*>(scratch);
    uint64_t w[NP];
#pragma unroll
    for (int g = 0; g < NP; ++g) w[g] = 0;
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      const float x = exp_from(s[g], m[g]);
      l[g] += x;
      w[g] = pack2(x, x);
    }
    if (lane % kOwn == 0) {
      if constexpr (NH == 1) {
        pairs[key] = w[0];
      } else {
#pragma unroll
        for (int g = 0; g < NP; g += 2)
          *reinterpret_cast<ulonglong2*>(pairs + key * NP + g) = make_ulonglong2(w[g], w[g + 1]);
      }
    }
    __syncwarp();
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int at = st * kKeysAtOnce * rb;
      uint64_t x[4];
      if constexpr (sizeof(T) == 4) {
        uint64_t h[2];
        load_chunk(vs + at + (in0 ? pv0 : 0), h);
        x[0] = in0 ? h[0] : 0;
        x[1] = in0 ? h[1] : 0;
        load_chunk(vs + at + (in1 ? pv1 : 0), h);
        x[2] = in1 ? h[0] : 0;
        x[3] = in1 ? h[1] : 0;
      } else {
        load_chunk(vs + at + (in0 ? pv0 : 0), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = in0 ? x[i] : 0;
      }
      const uint64_t* row = pairs + (st * kKeysAtOnce + group) * NP;
      uint64_t f[NP];
      if constexpr (NH == 1) {
        f[0] = row[0];
      } else {
#pragma unroll
        for (int g = 0; g < NP; g += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(row + g);
          f[g] = two.x;
          f[g + 1] = two.y;
        }
      }
#pragma unroll
      for (int g = 0; g < NH; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] = fma2(f[g], x[i], acc[g][i]);
    }
  }

  // The warp's state: ml[2 * head] the maximum, ml[2 * head + 1] the sum, o[head * D + d].
  __device__ __forceinline__ void dump(float* ml, float* o) {
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      float sum = lane % kOwn == 0 ? l[g] : 0.f;  // each key once
#pragma unroll
      for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (lane == 0) {
        ml[2 * g] = m[g];
        ml[2 * g + 1] = sum;
      }
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(acc[g][i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
#pragma unroll
      for (int off = 16; off >= L; off >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], off);
      if (group == 0)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          if (elem(i) < D)
            *reinterpret_cast<float4*>(o + g * D + elem(i)) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
  }
};

// Tensor cores: 16-bit pages and activations of one type.  S = Q K^T and O = P V
// by mma.m16n8k16 with the query heads as rows: the multiplications cost next
// to nothing beside the loads, where the lanes' fp32 would bound a larger
// group.  q and K are exact operands.  P is not rounded to the 16-bit type: it
// is split into two terms, p = hi + lo.  In bf16 their relative error is 2^-16
// over fp32's whole range.  fp16 ends at 2^-24, so 2^15 p is split (at most
// 32768 of 65504) and the sums of values are scaled back at the end: relative error
// 2^-21, and 2^-40 of the largest weight where that is more.  (Split as it is, p
// would be lost below 2^-25: of 32 keys 17.4 below one score nothing would be
// left.)  The sum of the weights takes p itself.
// With up to eight heads hi takes rows 0-7 and lo rows 8-15 of the
// same product.  D is padded to DT in shared memory; rows are swizzled by 16-byte
// chunks so that ldmatrix reads eight rows without bank conflicts.
// With FULL, D is DT: no padding.
template <class T_, int DT, int NH_, bool FULL>
struct MmaTile {
  using T = T_;
  static constexpr int NH = NH_;
  static_assert(NH == 8 || NH == 16, "");
  static constexpr int TK = DT == 64 ? 32 : 16;
  static constexpr int kStages = 3;
  static constexpr int kScratch = 0;
  using Query = T;  // in shared memory, rows 16 bytes further apart: eight heads lie in different banks
  static constexpr int kMaxD = DT, kQueryPad = 8;
  static constexpr int kD = FULL ? DT : 0;
  static constexpr int R = NH / 8;  // head rows of a thread
  static constexpr int kMinBlocks = DT == 256 ? 1 : 2;
  static constexpr float kUp = TypeCode<T>::value == DT_F16 ? 32768.f : 1.f;  // of the weights in the products
  static_assert(2 * TK * DT * 2 >= NH * DT * 4, "a warp's state fits into a stage");

  uint32_t q[DT / 16][2 * R];
  float acc[DT / 8][4];
  float m[R], l[R];
  float scale;
  int D, lane;

  __host__ __device__ static int row_bytes(int) { return DT * 2; }
  __device__ static __forceinline__ int chunk_at(int row, int chunk, int = 0) { return chunk ^ (row & 7); }

  __device__ static __forceinline__ T query(const void* q, int, int64_t i, float) { return static_cast<const T*>(q)[i]; }
  __device__ __forceinline__ void begin(const KvAttendParams& p, const T* queries, int nh) {
    D = FULL ? DT : p.geom.head_dim;
    lane = threadIdx.x % 32;
    scale = p.scale;
#pragma unroll
    for (int k = 0; k < DT / 16; ++k)
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) {
        // registers of A: rows g (and g + 8), columns 2c, 2c + 1 (and + 8)
        const int head = lane / 4 + (R == 2 ? (i & 1) * 8 : 0);
        const int d = k * 16 + lane % 4 * 2 + (R == 2 ? i >> 1 : i) * 8;
        const bool in = head < nh && d < D;  // D is even
        q[k][i] = in ? *reinterpret_cast<const uint32_t*>(queries + head * (D + kQueryPad) + d) : 0u;
      }
#pragma unroll
    for (int j = 0; j < DT / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
  }

  __device__ static __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    if constexpr (TypeCode<T>::value == DT_BF16)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  __device__ static __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
  }
  __device__ static __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
  }
  // Two weights, times kUp, as the 16-bit type, and what the rounding left.
  __device__ static __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (kUp != 1.f) {
      x *= kUp;
      y *= kUp;
    }
    T h[2] = {from_f<T>(x), from_f<T>(y)};
    T r[2] = {from_f<T>(x - to_f(h[0])), from_f<T>(y - to_f(h[1]))};
    hi = *reinterpret_cast<uint32_t*>(h);
    lo = *reinterpret_cast<uint32_t*>(r);
  }

  __device__ __forceinline__ void tile(const char* ks, const char* vs, const float* add, float*, const T*, float* scores,
                                       int live, int group_size, int nh) {
    constexpr int RB = DT * 2;
    const uint32_t kb = smem_u32(ks), vb = smem_u32(vs);
    float s[TK / 8][4];
#pragma unroll
    for (int j = 0; j < TK / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] = 0.f;
#pragma unroll
    for (int k = 0; k < DT / 16; k += 2)
#pragma unroll
      for (int j = 0; j < TK / 8; ++j) {
        uint32_t r[4];
        const int row = j * 8 + lane % 8, chunk = 2 * k + lane / 8;
        ldsm(r, kb + row * RB + chunk_at(row, chunk) * 16);
        if constexpr (R == 1) {
          mma(s[j], q[k][0], 0u, q[k][1], 0u, r[0], r[1]);
          mma(s[j], q[k + 1][0], 0u, q[k + 1][1], 0u, r[2], r[3]);
        } else {
          mma(s[j], q[k][0], q[k][1], q[k][2], q[k][3], r[0], r[1]);
          mma(s[j], q[k + 1][0], q[k + 1][1], q[k + 1][2], q[k + 1][3], r[2], r[3]);
        }
      }
    float mx[R];
#pragma unroll
    for (int r = 0; r < R; ++r) mx[r] = m[r];
#pragma unroll
    for (int j = 0; j < TK / 8; ++j) {
      const int key = j * 8 + lane % 4 * 2;
      const float2 a = *reinterpret_cast<const float2*>(add + key);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[j][2 * r] = masked(fmaf(s[j][2 * r], scale, a.x), a.x);
        s[j][2 * r + 1] = masked(fmaf(s[j][2 * r + 1], scale, a.y), a.y);
        mx[r] = fmaxf(mx[r], fmaxf(s[j][2 * r], s[j][2 * r + 1]));
      }
    }
    if (scores) {
#pragma unroll
      for (int j = 0; j < TK / 8; ++j)
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
          const int key = j * 8 + lane % 4 * 2 + i % 2, head = lane / 4 + i / 2 * 8;
          if (head < nh && key < live) scores[key * group_size + head] = s[j][i];
        }
    }
    bool changed = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      changed |= mx[r] != m[r];
    }
    if (__any_sync(0xffffffffu, changed)) {
      float c[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        c[r] = exp_from(m[r], mx[r]);
        l[r] *= c[r];
        m[r] = mx[r];
      }
#pragma unroll
      for (int j = 0; j < DT / 8; ++j) {
        acc[j][0] *= c[0];
        acc[j][1] *= c[0];
        acc[j][2] *= c[R - 1];
        acc[j][3] *= c[R - 1];
      }
    }
#pragma unroll
    for (int j = 0; j < TK / 8; ++j)
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) {
        s[j][i] = exp_from(s[j][i], m[i / 2]);
        l[i / 2] += s[j][i];
      }
#pragma unroll
    for (int kk = 0; kk < TK / 16; ++kk) {
      uint32_t hi[2][R], lo[2][R];  // [columns 0-7 / 8-15 of the 16 keys][head rows]
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) split(s[2 * kk + c][2 * r], s[2 * kk + c][2 * r + 1], hi[c][r], lo[c][r]);
#pragma unroll
      for (int j = 0; j < DT / 8; j += 2) {
        uint32_t r[4];
        const int row = kk * 16 + lane / 8 % 2 * 8 + lane % 8, chunk = j + lane / 16;
        ldsm_t(r, vb + row * RB + chunk_at(row, chunk) * 16);
        if constexpr (R == 1) {
          mma(acc[j], hi[0][0], lo[0][0], hi[1][0], lo[1][0], r[0], r[1]);
          mma(acc[j + 1], hi[0][0], lo[0][0], hi[1][0], lo[1][0], r[2], r[3]);
        } else {
          mma(acc[j], hi[0][0], hi[0][1], hi[1][0], hi[1][1], r[0], r[1]);
          mma(acc[j], lo[0][0], lo[0][1], lo[1][0], lo[1][1], r[0], r[1]);
          mma(acc[j + 1], hi[0][0], hi[0][1], hi[1][0], hi[1][1], r[2], r[3]);
          mma(acc[j + 1], lo[0][0], lo[0][1], lo[1][0], lo[1][1], r[2], r[3]);
        }
      }
    }
  }

  __device__ __forceinline__ void dump(float* ml, float* o) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int head = lane / 4 + 8 * r;
      ml[2 * head] = m[r];
      ml[2 * head + 1] = l[r];
#pragma unroll
      for (int j = 0; j < DT / 8; ++j) {
        const int d = j * 8 + lane % 4 * 2;
        if (d < D) {
          const float x = R == 1 ? acc[j][0] + acc[j][2] : acc[j][2 * r];
          const float y = R == 1 ? acc[j][1] + acc[j][3] : acc[j][2 * r + 1];
          o[head * D + d] = kUp == 1.f ? x : x * (1.f / kUp);
          o[head * D + d + 1] = kUp == 1.f ? y : y * (1.f / kUp);
        }
      }
    }
  }
};

// --- the kernel -------------------------------------------------------------------

// Where a block is in its run of tiles.
struct Cursor {
  int b = 0, kvh = 0, chunk = 0, tile = 0, tiles = 0;
  int len = 0;
};

// Rows that take part: 0 for a length beyond the limit, -1 for no sequence.
__device__ __forceinline__ int length_of(const KvAttendParams& p, int b) {
  const int n = p.lengths[b];
  return n < 0 ? -1 : n > p.max_len ? 0 : n;
}
template <int TILE>
__device__ __forceinline__ int tiles_of(int len) {  // an empty sequence takes one, for its zeros
  return len < 0 ? 0 : len == 0 ? 1 : (len + TILE - 1) / TILE;
}
// Units of work of a segment: `start` for its begin and end, then one a tile;
// tile i is done by the block that has unit i + start.  With four tiles a block
// and more the begin counts as two (9/3 x 64 heads, 64 sequences of up to 2048
// rows, fp32: 29.6 us against 30.4); with fewer as one, or blocks that hold
// nothing else would stand idle (one of 16,385 rows: 14.3 us against 15.9).
template <int TILE>
__device__ __forceinline__ int units_of(int len, int start) {
  return len < 0 ? 0 : tiles_of<TILE>(len) + start;
}

// Shared memory in bytes: the warps' stages, their mask values and scratch, and the queries.  At
// the end of a segment a warp's state takes the place of the stage that it has just
// used, which the next tile's load fills again: in all types NH * D floats fit
// into the 2 * TK rows of a stage.
template <class P>
__host__ __device__ constexpr int attend_stage_bytes(int row_bytes) { return 2 * P::TK * row_bytes; }
template <class P>
inline int attend_smem(int row_bytes, int D) {
  return kWarps * (P::kStages * (attend_stage_bytes<P>(row_bytes) + P::TK * 4) + P::kScratch * 4) +
         P::NH * (D + P::kQueryPad) * (int)sizeof(typename P::Query);
}

template <class P>
__global__ void __launch_bounds__(kThreads, P::kMinBlocks) kv_attend_kernel(const __grid_constant__ KvAttendParams p) {
  using T = typename P::T;
  constexpr int TK = P::TK, TILE = kWarps * TK, NS = P::kStages, NH = P::NH;
  extern __shared__ __align__(128) char smem[];
  __shared__ long long s_warp[kWarps], s_base;
  __shared__ int s_b0;
  __shared__ float s_ml[kWarps][NH][2];  // the warps' maxima and sums
  __shared__ long long s_new[kWarps][NS];  // of a stage with a sequence's last row: where that is still to be stored, or -1
  asm volatile("griddepcontrol.launch_dependents;");  // the join may take its place early: it waits for this grid's end
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) p.splits[blockIdx.x] = make_int2(0, 0);
  const int D = P::kD ? P::kD : p.geom.head_dim, kv = p.geom.kv_heads, group = p.heads / kv, chunks = (group + NH - 1) / NH;
  const int per_tile = kv * chunks;  // segments of a sequence

  // The block's run of tiles: prefix sums of the sequences' tiles, each thread a slice of the batch.
  long long u0, u1, total, blocks;  // its units
  int start;
  {
    const int slice = (p.batch + kThreads - 1) / kThreads, b0 = min(tid * slice, p.batch), b1 = min(b0 + slice, p.batch);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
      const int len = length_of(p, b);
      if (len >= 0) mine += ((long long)tiles_of<TILE>(len) << 17) + 1;  // tiles, and sequences in the low bits
      if (blockIdx.x == 0 && p.lengths[b] > p.max_len) set_status(p.status, ST_KV_LENGTH);  // length_of takes it as 0
    }
    long long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    long long before = 0, sum = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before = sum;
      sum += s_warp[w];
    }
    start = (sum >> 17) * per_tile >= 4ll * gridDim.x ? 2 : 1;
    auto units = [&](long long x) { return ((x >> 17) + (x & 0x1ffff) * start) * per_tile; };
    total = units(sum);
    blocks = min((long long)gridDim.x, total);  // every one of them has a unit
    if (blockIdx.x >= blocks) return;
    // floor(total * i / blocks), by one long division
    const long long each = total / blocks;
    const unsigned rest = (unsigned)(total - each * blocks), n = (unsigned)blocks, i = blockIdx.x;
    u0 = each * i + rest * i / n;
    u1 = each * (i + 1) + rest * (i + 1) / n;
    before = units(before + scan - mine);
    if (u0 >= before && u0 < before + units(mine)) {  // this thread's slice holds the first unit
      int b = b0;
      for (;; ++b) {
        const long long n = (long long)units_of<TILE>(length_of(p, b), start) * per_tile;
        if (u0 < before + n) break;
        before += n;
      }
      s_b0 = b;
      s_base = before;
    }
    __syncthreads();
  }

  auto enter = [&](Cursor& c) {  // at the first tile of sequence c.b, or of the next one that has tiles
    for (;;) {
      c.len = length_of(p, c.b);
      c.tiles = tiles_of<TILE>(c.len);
      if (c.tiles) return;
      ++c.b;
    }
  };
  auto advance = [&](Cursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.chunk < chunks) return;
    c.chunk = 0;
    if (++c.kvh < kv) return;
    c.kvh = 0;
    ++c.b;
    enter(c);
  };
  Cursor use;
  use.b = s_b0;
  use.len = length_of(p, use.b);
  use.tiles = tiles_of<TILE>(use.len);
  {
    const long long in = u0 - s_base;  // units into the sequence: (kvh, chunk, unit)
    const int units = use.tiles + start;
    const int seg = in >> 32 ? (int)(in / units) : (int)((unsigned)in / (unsigned)units);
    const int unit = (int)(in - (long long)seg * units);
    use.tile = max(unit - start, 0);
    use.chunk = seg % chunks;
    use.kvh = seg / chunks;
  }
  long long seg_begin = 0;  // the segment's first unit
  {
    const int units = use.tiles + start;
    seg_begin = s_base + ((long long)use.kvh * chunks + use.chunk) * units;
  }
  // tiles of the run: a walk over its segments
  int count = 0;
  {
    Cursor c = use;
    long long at = seg_begin;
    for (;;) {
      const long long end = at + start + c.tiles, upto = min(end, u1) - at - start;  // tiles of the segment before u1
      if (upto > c.tile) count += (int)upto - c.tile;
      at = end;
      if (at >= u1) break;
      c.tile = c.tiles - 1;
      advance(c);
    }
  }
  if (count == 0) return;  // a run of no more than the begin of a segment
  Cursor load = use;

  // the warp's part of shared memory
  const int rb = P::row_bytes(D), stage_bytes = attend_stage_bytes<P>(rb);
  char* ring = smem + warp * NS * stage_bytes;
  float* adds = reinterpret_cast<float*>(smem + kWarps * NS * stage_bytes) + warp * NS * TK;
  float* scratch = reinterpret_cast<float*>(smem + kWarps * NS * (stage_bytes + TK * 4)) + warp * P::kScratch;
  // The segment's queries, [NH][D]: fetched into registers while the last
  // segment is joined, then put into shared memory.
  using Query = typename P::Query;
  constexpr int kQueryEach = (NH * P::kMaxD + kThreads - 1) / kThreads;
  Query* queries = reinterpret_cast<Query*>(smem + kWarps * (NS * (stage_bytes + TK * 4) + P::kScratch * 4));
  Query fetched[kQueryEach];
  auto fetch_q = [&](const Cursor& c) {
    const int h = c.kvh * group + c.chunk * NH, n = min(NH, group - c.chunk * NH) * D;
    const int64_t at = c.b * p.q_stride + (int64_t)h * D;
#pragma unroll
    for (int r = 0; r < kQueryEach; ++r) {
      const int x = r * kThreads + tid;
      fetched[r] = x < n ? P::query(p.q, p.dt, at + x, p.scale) : from_f<Query>(0.f);
    }
  };
  auto put_q = [&] {
#pragma unroll
    for (int r = 0; r < kQueryEach; ++r) {
      const int x = r * kThreads + tid;
      if (x < NH * D) queries[P::kQueryPad ? x + x / D * P::kQueryPad : x] = fetched[r];
    }
  };
  // Tensor cores read the padding of K rows up to DT, against zeros of q: it holds zeros, which no load overwrites.
  const bool padded = !P::kD && P::kScratch == 0 && rb != D * (int)sizeof(T);
  auto clear = [&](char* at, int bytes) {
    for (int i = lane; i < bytes / 16; i += 32) reinterpret_cast<uint4*>(at)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  };
  if (padded) clear(ring, NS * stage_bytes);

  // Fetching a tile: lane r holds the page and the mask value of the warp's row r.
  int f_page = -1;
  float f_add = 0.f;
  auto fetch = [&](const Cursor& c) {
    const int i = c.tile * TILE + warp * TK + lane;
    f_page = -1;
    f_add = -INFINITY;
    if (lane < TK && i < c.len) {
      const int col = p.page_shift >= 0 ? i >> p.page_shift : i / p.geom.page_size;
      f_page = col < p.table_cols ? p.table[c.b * p.table_stride + col] : -1;
      f_add = p.mask ? p.mask[c.b * p.mask_stride + i] : 0.f;
    }
  };
  // lane's first vector among a tile's rows, and the step to its next one
  const int vecs = D * (int)sizeof(T) / 16;
  const int row_step = 32 / vecs, col_step = 32 % vecs, row_0 = lane / vecs, col_0 = lane % vecs;
  auto issue = [&](const Cursor& c, int stage) {
    const int first = c.tile * TILE + warp * TK, i = first + lane;
    char* ks = ring + stage * stage_bytes;
    if (first < c.len) {
      char* vs = ks + TK * rb;
      long long off = -1;
      bool fresh = false;
      if (lane < TK && i < c.len) {
        if (f_page < 0 || f_page >= p.geom.num_pages) {
          set_status(p.status, ST_KV_PAGE);
          f_add = -INFINITY;
        } else {
          const int slot = p.page_shift >= 0 ? i & ((1 << p.page_shift) - 1) : i % p.geom.page_size;
          off = row_offset(f_page, c.kvh, slot, p.geom) * (long long)sizeof(T);
          fresh = p.k && i == c.len - 1;
        }
      }
      if (lane < TK) adds[stage * TK + lane] = f_add;
      unsigned fresh_row = 0;
      long long fresh_off = 0;
      if (p.k && first + TK >= c.len) {  // the tile of the last row
        fresh_row = __ballot_sync(0xffffffffu, fresh);
        fresh_off = __shfl_sync(0xffffffffu, off, fresh_row ? __ffs(fresh_row) - 1 : 0);
      }
      if (f_add == -INFINITY || fresh) off = -1;  // nothing to load
      if (__all_sync(0xffffffffu, off >= 0 || lane >= TK)) {  // whole rows: lane l takes vectors l, l + 32, ..
        const char* from = static_cast<const char*>(p.k_pages);
        const long long to_v = static_cast<const char*>(p.v_pages) - from;
        const uint32_t ka = smem_u32(ks), va = smem_u32(vs);
        if constexpr (P::kD != 0) {
          constexpr int V = P::kD * (int)sizeof(T) / 16;
          from += lane % V * 16;
#pragma unroll
          for (int v = 0; v < TK * V; v += 32) {
            const int row = V <= 32 ? v / V + lane / V : v / V, col = V <= 32 ? lane % V : v % V + lane;
            const char* src = from + __shfl_sync(0xffffffffu, off, row) + (V <= 32 ? 0 : v % V * 16);
            const int s = row * rb + P::chunk_at(row, col, D) * 16;
            copy16(ka + s, src);
            copy16(va + s, src + to_v);
          }
        } else {
          int row = row_0, col = col_0;
#pragma unroll 4
          for (int v = 0; v < TK * vecs; v += 32) {
            const char* src = from + __shfl_sync(0xffffffffu, off, row & 31) + col * 16;
            const int s = row * rb + P::chunk_at(row, col, D) * 16;
            if (row < TK) {
              copy16(ka + s, src);
              copy16(va + s, src + to_v);
            }
            row += row_step;
            col += col_step;
            if (col >= vecs) {
              col -= vecs;
              ++row;
            }
          }
        }
        return;
      }
      // The new token's row comes from the call's arguments.  In the pages' type
      // it is copied like the others and stored when its tile is used; another
      // type is rounded and stored below.  A row that the mask takes out stays zeros.
      const int new_row = fresh_row ? __ffs(fresh_row) - 1 : 0;
      const bool live_new = fresh_row && __shfl_sync(0xffffffffu, f_add, new_row) != -INFINITY;
      const bool copy_new = live_new && p.k_as_stored, put_new = live_new && !copy_new;
      const int64_t k_new = c.b * p.k_stride + c.kvh * D, v_new = c.b * p.v_stride + c.kvh * D;
      if (p.k_as_stored && first + TK >= c.len && lane == 0) s_new[warp][stage] = copy_new ? fresh_off : -1;
      int row = row_0, col = col_0;
      for (int v = 0; v < TK * vecs; v += 32) {
        const long long o = __shfl_sync(0xffffffffu, off, row & 31);
        if (row < TK && !(put_new && row == new_row)) {
          const bool ok = o >= 0;
          const long long at = ok ? o + col * 16 : 0;
          const int s = row * rb + P::chunk_at(row, col, D) * 16;
          if (copy_new && row == new_row) {
            copy16(smem_u32(ks + s), reinterpret_cast<const char*>(static_cast<const T*>(p.k) + k_new) + col * 16);
            copy16(smem_u32(vs + s), reinterpret_cast<const char*>(static_cast<const T*>(p.v) + v_new) + col * 16);
          } else {
            copy16(smem_u32(ks + s), static_cast<const char*>(p.k_pages) + at, ok);
            copy16(smem_u32(vs + s), static_cast<const char*>(p.v_pages) + at, ok);
          }
        }
        row += row_step;
        col += col_step;
        if (col >= vecs) {
          col -= vecs;
          ++row;
        }
      }
      if (fresh_row && !copy_new) {
        for (int d = lane; d < D; d += 32) {
          const T k = from_f<T>(load_act(p.k, p.dt, k_new + d));
          const T v = from_f<T>(load_act(p.v, p.dt, v_new + d));
          if (put_new) {
            const int s = new_row * rb + P::chunk_at(new_row, d * (int)sizeof(T) / 16, D) * 16 + d * (int)sizeof(T) % 16;
            *reinterpret_cast<T*>(ks + s) = k;
            *reinterpret_cast<T*>(vs + s) = v;
          }
          if (c.chunk == 0) {  // the block of the first chunk of heads stores it
            reinterpret_cast<T*>(static_cast<char*>(p.k_pages) + fresh_off)[d] = k;
            reinterpret_cast<T*>(static_cast<char*>(p.v_pages) + fresh_off)[d] = v;
          }
        }
      }
    }
  };

  // fill the ring
  int issued = 0;
  fetch(load);
  fetch_q(use);
#pragma unroll 1
  for (; issued < NS - 1; ++issued) {
    if (issued < count) {
      issue(load, issued);
      if (issued + 1 < count) {
        advance(load);
        fetch(load);
      }
    }
    copy_commit();
  }

  put_q();
  __syncthreads();
  int stage = 0, load_stage = NS - 1;  // of the tile in use, and of the next tile to load
  int j = 0;
#pragma unroll 1
  while (j < count) {  // a segment, or the part of it that this block has
    const int h0 = use.kvh * group + use.chunk * NH, nh = min(NH, group - use.chunk * NH);
    const int mine = min(use.tiles - use.tile, count - j);
    const bool own_begin = use.tile == 0, seg_end = use.tile + mine == use.tiles;
    int stage_at = 0;
    {
      P state;
      state.begin(p, queries, nh);
      int first = use.tile * TILE + warp * TK;
      float* scores = nullptr;
      if (p.weights_out)
        scores = p.scores + (((long long)use.b * kv + use.kvh) * p.max_len + first) * group + use.chunk * NH;
#pragma unroll 1
      for (int i = 0; i < mine; ++i) {
        copy_wait<NS - 2>();
        __syncwarp();
        if (issued < count) {
          issue(load, load_stage);
          if (++issued < count) {
            advance(load);
            fetch(load);
          }
        }
        copy_commit();
        load_stage = load_stage + 1 == NS ? 0 : load_stage + 1;
        stage_at = stage * stage_bytes;
        if (p.k_as_stored && use.chunk == 0 && first < use.len && first + TK >= use.len) {  // the tile of the last row
          const int row = use.len - 1 - first;
          const long long to = s_new[warp][stage];
          if (to >= 0)
            for (int v = lane; v < 2 * vecs; v += 32) {
              const int col = v < vecs ? v : v - vecs;
              const char* from = ring + stage_at + (v < vecs ? 0 : TK * rb) + row * rb + P::chunk_at(row, col, D) * 16;
              *reinterpret_cast<uint4*>(static_cast<char*>(v < vecs ? p.k_pages : p.v_pages) + to + col * 16) =
                  *reinterpret_cast<const uint4*>(from);
            }
        }
        if (first < use.len)
          state.tile(ring + stage_at, ring + stage_at + TK * rb, adds + stage * TK, scratch, queries, scores,
                     use.len - first, group, nh);
        stage = stage + 1 == NS ? 0 : stage + 1;
        first += TILE;
        if (p.weights_out) scores += (long long)TILE * group;
      }
      // the warp's state takes the place of the stage it has just used: every lane has read its V rows
      __syncwarp();
      state.dump(&s_ml[warp][0][0], reinterpret_cast<float*>(ring + stage_at));
    }
    j += mine;
    use.tile += mine - 1;  // its last tile here
    {
      // join the warps
      __syncthreads();
      if (j < count) {
        Cursor next = use;
        advance(next);
        fetch_q(next);
      }
      const bool begins = own_begin, whole = begins && seg_end;
      const int dv = D / 4;  // the results are taken four at a time
      // A part in the workspace: [NH][2], padded to 16 bytes, then [nh][D], counted
      // in units of 16 bytes.  A block has two places: 2 i + 1 for the segment that begins
      // in its run and goes on behind it, 2 i for the one that began before.
      float4* part = reinterpret_cast<float4*>(p.parts) +
                     (2 * blockIdx.x + (begins ? 1 : 0)) * kv_part_vecs(NH, D);
      for (int x = tid; x < nh * dv; x += kThreads) {
        const int h = x / dv, d = x % dv * 4;
        float mt = -INFINITY, lt = 0.f;
        float4 ot = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, s_ml[w][h][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float c = exp_from(s_ml[w][h][0], mt);
          lt += s_ml[w][h][1] * c;
          add_scaled(ot, reinterpret_cast<const float4*>(smem + w * NS * stage_bytes + stage_at)[x], c);
        }
        if (whole) store_result(p, use.b, h0 + h, d, mt, lt, ot);
        else part[kv_part_head(NH) + x] = ot;
        if (!whole && d == 0) reinterpret_cast<float2*>(part)[h] = make_float2(mt, lt);
      }
      if (tid == 0 && begins) {
        // for the join: the segment's first block and the number of its blocks; the
        // block that holds unit u is the largest i with floor(total * i / blocks) <= u
        const long long u = (seg_begin + use.tiles + start) * blocks - 1;
        const int last = u >> 32 ? (int)(u / total) : (int)((unsigned)u / (unsigned)total);  // u >= total - 1: both fit
        const int segment = (use.b * kv + use.kvh) * chunks + use.chunk, n = last - (int)blockIdx.x + 1;
        p.info[segment] = make_int2(blockIdx.x, n);
        if (n > 1) p.splits[blockIdx.x] = make_int2(segment, n);
      }
      if (j < count) put_q();
      __syncthreads();  // the stages are free again, and the next queries there
      if (padded) clear(ring + stage_at, stage_bytes);
      seg_begin += use.tiles + start;
    }
    if (j < count) advance(use);
  }
  copy_wait<0>();
}

// Blocks of this kernel that an SM holds, at most kMaxBlocksPerSm; asked once
// per device and shared-memory size.
template <class P>
cudaError_t blocks_per_sm(int device, int smem, int* out) {
  static std::atomic<int64_t> known[kMaxDevices];  // smem << 8 | blocks
  if (device < kMaxDevices) {
    const int64_t k = known[device].load(std::memory_order_relaxed);
    if (k >> 8 == smem && k) {
      *out = (int)(k & 255);
      return cudaSuccess;
    }
  }
  // the limit covers every head dim, so that calls of two threads do not undo each other's
  cudaError_t e = cudaFuncSetAttribute(kv_attend_kernel<P>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  int n = 0;
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv_attend_kernel<P>, kThreads, smem);
  if (e != cudaSuccess) return e;
  *out = std::min(std::max(n, 1), kMaxBlocksPerSm);
  if (device < kMaxDevices) known[device].store((int64_t)smem << 8 | *out, std::memory_order_relaxed);
  return cudaSuccess;
}

template <class P>
cudaError_t attend_launch(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  const int D = p.geom.head_dim, smem = attend_smem<P>(P::row_bytes(D), D);
  int per_sm = 0;
  if (cudaError_t e = blocks_per_sm<P>(p.device, smem, &per_sm)) return e;
  shape->blocks = p.sms * per_sm;
  shape->heads = P::NH;
  shape->split = p.max_len > kWarps * P::TK;
  kv_attend_kernel<P><<<shape->blocks, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

// The kernel for these types, head dim and group: a group of more than eight
// heads (four, where a stage of four 16-bit rows holds the states of no more)
// is divided evenly.
template <class T, int L, bool FULL>
cudaError_t attend_lanes_group(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  constexpr int kMost = L == 32 && sizeof(T) == 2 ? 4 : 8;
  const int group = p.heads / p.geom.kv_heads, chunks = (group + kMost - 1) / kMost, heads = (group + chunks - 1) / chunks;
  if (heads <= 1) return attend_launch<LaneTile<T, L, 1, FULL>>(p, shape, s);
  if (heads <= 2) return attend_launch<LaneTile<T, L, 2, FULL>>(p, shape, s);
  if (heads <= 3) return attend_launch<LaneTile<T, L, 3, FULL>>(p, shape, s);
  if (heads <= 4) return attend_launch<LaneTile<T, L, 4, FULL>>(p, shape, s);
  if constexpr (kMost == 8) {
    if (heads <= 6) return attend_launch<LaneTile<T, L, 6, FULL>>(p, shape, s);
    return attend_launch<LaneTile<T, L, 8, FULL>>(p, shape, s);
  }
  return cudaErrorInvalidValue;
}
template <class T>
cudaError_t attend_lanes(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  const int D = p.geom.head_dim;
  switch (kv_row_lanes(D)) {
    case 4: return attend_lanes_group<T, 4, false>(p, shape, s);
    case 8:
      return D == 64 ? attend_lanes_group<T, 8, true>(p, shape, s) : attend_lanes_group<T, 8, false>(p, shape, s);
    case 16:
      return D == 128 ? attend_lanes_group<T, 16, true>(p, shape, s) : attend_lanes_group<T, 16, false>(p, shape, s);
    default: return attend_lanes_group<T, 32, false>(p, shape, s);
  }
}
template <class T, int NH>
cudaError_t attend_mma(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  const int D = p.geom.head_dim;
  if (D < 64) return attend_launch<MmaTile<T, 64, NH, false>>(p, shape, s);
  if (D == 64) return attend_launch<MmaTile<T, 64, NH, true>>(p, shape, s);
  if (D < 128) return attend_launch<MmaTile<T, 128, NH, false>>(p, shape, s);
  if (D == 128) return attend_launch<MmaTile<T, 128, NH, true>>(p, shape, s);
  return attend_launch<MmaTile<T, 256, NH, false>>(p, shape, s);
}
template <class T>
cudaError_t attend_16bit(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  // Tensor cores need one type, and pay from 16 to 128 elements a row whatever the
  // group.  bf16, 64 sequences of up to 1024 rows, 8/8 heads, lanes -> tensor cores:
  // 16 elements 30.9 -> 24.0 us, 32 33.5 -> 23.2, 64 24.1 -> 24.0, 128 36.5 -> 34.3.
  // Rows of 8 are mostly padding (17.9 -> 23.1) and longer ones leave an SM one block
  // (192: 84.5 -> 107; two heads a key/value head: 104.5 -> 109), which only the arithmetic
  // of three heads and more outweighs (12/4 heads of 256, one of 65,536 rows: 110 -> 73).
  const int D = p.geom.head_dim, group = p.heads / p.geom.kv_heads;
  if (p.dt == TypeCode<T>::value && ((D >= 16 && D <= 128) || group > 2))
    return group <= 8 ? attend_mma<T, 8>(p, shape, s) : attend_mma<T, 16>(p, shape, s);
  return attend_lanes<T>(p, shape, s);
}

}  // namespace paged
}  // namespace kern
}  // namespace gawee
