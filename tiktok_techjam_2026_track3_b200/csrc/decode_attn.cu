// One decode step over a prefix shared by the batch and each sequence's own cache.
//
// The softmax over all of a row's keys splits into ranges, each giving the partial
//   o_i = sum_u 2^(s_u - lse_i) v_u,   lse_i = log2 sum_u 2^s_u   (s = scale log2(e) q.k)
// and joins as  o = sum_i 2^(lse_i - lse) o_i,  lse = log2 sum_i 2^lse_i.
//
// Ranges of the caches: one block per (sequence, key / value head, range), bound by
// the cache's bytes.  A group has few rows (group heads), so the products run on
// 16-row warp tiles: four warps take 16 or 32 keys in turn, each through its own
// ring of asynchronous copies (no block barrier in the loop), its own running
// maximum, sum and output; the block joins its warps at the end.  Rows of the
// cache past the length are never read: their copies are zero-filled.
//
// Ranges of the prefix: with many rows (batch x group) the 128-row tensor-core
// kernel (launch_prefix_parts), which reads the prefix once for up to 256 rows;
// with few, blocks of the cache kernel whose rows belong to several sequences.
//
// Then one kernel joins the ranges and, with key_weights, turns the stored scores
// into probabilities with the rows' final lse and adds them up over the group.
#include <algorithm>
#include <atomic>

#include "attn_math.cuh"
#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace ttj {
namespace {

constexpr int kRows = 16;    // rows of a warp tile
constexpr int kWarps = 4;
constexpr int kJoinThreads = 256;
constexpr int kWeightSpan = 1024;  // cached keys per join block

template <int HD>
struct RangeSmem {
  static constexpr int kKeys = HD == 64 ? 32 : 16;   // per warp step
  static constexpr int kStages = 3;
  static constexpr int kRowBytes = HD * 2;
  static constexpr int kTensorBytes = kKeys * kRowBytes;
  static constexpr int kStageBytes = 2 * kTensorBytes;   // K and V
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kTotal = kRing + 2 * kWarps * kRows * 4;
  static_assert(kWarps * kRows * HD * 4 <= kRing, "the warps' outputs reuse the ring");
};

// How the step is cut into ranges (host).
struct Cuts {
  bool prefix_tiles;        // prefix on the 128-row tensor-core kernel
  int prefix_parts, prefix_keys;
  int cache_parts, cache_keys;
  int parts() const { return prefix_parts + cache_parts; }
};

struct RangeParams {
  const void *q, *pk, *pv, *kc, *vc;
  const int32_t* lengths;
  float *part_o, *part_lse, *scores;   // scores: [B][Hq][score_pitch] of the cached keys, or null
  int64_t q_seq, q_head, pk_row, pk_head, pv_row, pv_head, kc_seq, kc_row, kc_head, vc_seq, vc_row, vc_head;
  int64_t score_pitch;
  int batch, prefix, capacity, num_heads, kv_heads, group, hd;
  int prefix_blocks;        // blocks of the prefix's ranges, before those of the caches
  int prefix_row_tiles, prefix_keys, prefix_parts, cache_row_tiles, cache_keys;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16-byte chunk c of row r within a [rows][HD] tile, swizzled so that eight rows'
// equal chunks fall into different banks.
template <int HD>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)(r * HD * 2 + ((c ^ (r & 7)) << 4));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kWarps * 32)
range_kernel(const RangeParams p) {
  using L = RangeSmem<HD>;
  constexpr int kKeys = L::kKeys, kStages = L::kStages;
  constexpr int kChunks = HD / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, kq = lane & 3;

  // Which rows and keys: row r of the block is query head h0 + (i % group) of
  // sequence i / group for i = row0 + r < rows.
  const T *kbase, *vbase;
  int64_t krow, vrow, row0, rows;
  int kvh, keys_from, keys_to, part;
  bool cached = false;
  int64_t blk = blockIdx.x;
  if (blk < p.prefix_blocks) {
    part = (int)(blk / (p.kv_heads * p.prefix_row_tiles));
    const int rest = (int)(blk - (int64_t)part * p.kv_heads * p.prefix_row_tiles);
    kvh = rest / p.prefix_row_tiles;
    row0 = (int64_t)(rest - kvh * p.prefix_row_tiles) * kRows;
    rows = (int64_t)p.batch * p.group;
    kbase = static_cast<const T*>(p.pk) + kvh * p.pk_head;
    vbase = static_cast<const T*>(p.pv) + kvh * p.pv_head;
    krow = p.pk_row;
    vrow = p.pv_row;
    keys_from = part * p.prefix_keys;
    keys_to = min(keys_from + p.prefix_keys, p.prefix);
  } else {
    blk -= p.prefix_blocks;
    const int64_t per_part = (int64_t)p.batch * p.kv_heads * p.cache_row_tiles;
    part = (int)(blk / per_part);
    int64_t rest = blk - part * per_part;
    const int64_t b = rest / (p.kv_heads * p.cache_row_tiles);
    rest -= b * p.kv_heads * p.cache_row_tiles;
    kvh = (int)(rest / p.cache_row_tiles);
    row0 = b * p.group + (rest - kvh * p.cache_row_tiles) * kRows;
    rows = (b + 1) * p.group;
    kbase = static_cast<const T*>(p.kc) + b * p.kc_seq + kvh * p.kc_head;
    vbase = static_cast<const T*>(p.vc) + b * p.vc_seq + kvh * p.vc_head;
    krow = p.kc_row;
    vrow = p.vc_row;
    keys_from = part * p.cache_keys;
    keys_to = min(keys_from + p.cache_keys, min(max(__ldg(p.lengths + b), 0), p.capacity));
    part += p.prefix_parts;
    cached = true;
  }
  // row index in [B][Hq] of block row r, or -1
  auto out_row = [&](int r) -> int64_t {
    const int64_t i = row0 + r;
    if (i >= rows) return -1;
    const int64_t b = i / p.group;
    return b * p.num_heads + kvh * p.group + (i - b * p.group);
  };
  const int64_t part_row0 = (int64_t)part * p.batch * p.num_heads;
  if (keys_from >= keys_to) {  // nothing in this range: the join skips it
    if (threadIdx.x < kRows) {
      const int64_t at = out_row(threadIdx.x);
      if (at >= 0) p.part_lse[part_row0 + at] = -INFINITY;
    }
    return;
  }

  const int steps_all = (keys_to - keys_from + kKeys - 1) / kKeys;
  const int steps = (steps_all - warp + kWarps - 1) / kWarps;  // this warp's: warp, warp + kWarps, ...
  uint8_t* ring = smem + warp * kStages * L::kStageBytes;
  const uint32_t ring_s = smem_u32(ring);
  const int ld_chunk = lane % kChunks, ld_row = lane / kChunks;
  constexpr int kRowsPerPass = 32 / kChunks;
  const bool ld_col = ld_chunk * 8 < p.hd;
  auto load = [&](int i) {
    if (i < steps) {
      const int key0 = keys_from + (warp + i * kWarps) * kKeys;
      const uint32_t dst = ring_s + (i % kStages) * L::kStageBytes;
#pragma unroll
      for (int r = 0; r < kKeys; r += kRowsPerPass) {
        const int row = r + ld_row;
        const bool ok = ld_col && key0 + row < keys_to;
        const int64_t key = ok ? key0 + row : keys_from;
        const int col = ok ? ld_chunk * 8 : 0;
        cp_async16(dst + tile_at<HD>(row, ld_chunk), kbase + key * krow + col, ok);
        cp_async16(dst + L::kTensorBytes + tile_at<HD>(row, ld_chunk), vbase + key * vrow + col, ok);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i);

  // Q fragments straight from global memory: rows g and g + 8, columns 16 kk + 2 kq (+ 8)
  uint32_t qf[HD / 16][4];
  {
    const int64_t i0 = row0 + g, i1 = row0 + g + 8;
    auto q_row = [&](int64_t i) -> const T* {
      if (i >= rows) return nullptr;
      const int64_t b = i / p.group;
      return static_cast<const T*>(p.q) + b * p.q_seq + (kvh * p.group + (i - b * p.group)) * p.q_head;
    };
    const T *qa = q_row(i0), *qb = q_row(i1);
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const T* src = (e & 1) ? qb : qa;
        const int col = 16 * kk + 2 * kq + (e >> 1) * 8;
        qf[kk][e] = (src != nullptr && col < p.hd) ? __ldg(reinterpret_cast<const uint32_t*>(src + col)) : 0u;
      }
    }
  }
  float o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int64_t at_a = out_row(g), at_b = out_row(g + 8);
  const bool both = rows - row0 > 8;  // rows 8..15 hold heads

  for (int i = 0; i < steps; ++i) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    load(i + kStages - 1);
    const int key0 = keys_from + (warp + i * kWarps) * kKeys;
    const uint32_t sk = ring_s + (i % kStages) * L::kStageBytes, sv = sk + L::kTensorBytes;
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {
        uint32_t b[4];
        ldmatrix_x4(b, sk + tile_at<HD>(16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
        mma_16x8x16<T>(s[2 * n], qf[kk], b[0], b[1]);
        mma_16x8x16<T>(s[2 * n + 1], qf[kk], b[2], b[3]);
      }
    // s[n][e]: row g + 8 (e >> 1), key 8 n + 2 kq + (e & 1)
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool ok = key0 + 8 * n + 2 * kq + (e & 1) < keys_to;
        s[n][e] = ok ? s[n][e] * p.scale_log2 : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
      }
    if (cached && p.scores != nullptr) {
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        const int key = key0 + 8 * n + 2 * kq;
        if (key < keys_to) {  // the pitch is even: the pair's second key stays in the row
          if (at_a >= 0) *reinterpret_cast<float2*>(p.scores + at_a * p.score_pitch + key) = make_float2(s[n][0], s[n][1]);
          if (at_b >= 0) *reinterpret_cast<float2*>(p.scores + at_b * p.score_pitch + key) = make_float2(s[n][2], s[n][3]);
        }
      }
    }
    float alpha[2], ref[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      const float mn = mx[e] > m[e] + 8.f ? mx[e] : m[e];  // the reference moves lazily: P <= 2^8
      ref[e] = mn == -INFINITY ? 0.f : mn;
      alpha[e] = fast_exp2(m[e] - ref[e]);
      m[e] = mn;
      l[e] *= alpha[e];
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= alpha[e >> 1];
    }
    uint32_t pf[kKeys / 16][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) {
      const float e0 = fast_exp2(s[n][0] - ref[0]), e1 = fast_exp2(s[n][1] - ref[0]);
      l[0] += e0 + e1;
      pf[n >> 1][(n & 1) * 2] = Pack<T>::two(e0, e1);
      if (both) {
        const float e2 = fast_exp2(s[n][2] - ref[1]), e3 = fast_exp2(s[n][3] - ref[1]);
        l[1] += e2 + e3;
        pf[n >> 1][(n & 1) * 2 + 1] = Pack<T>::two(e2, e3);
      } else {
        pf[n >> 1][(n & 1) * 2 + 1] = 0u;
      }
    }
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, sv + tile_at<HD>(16 * kk + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * n + (lane >> 4)));
        mma_16x8x16<T>(o[2 * n], pf[kk], b[0], b[1]);
        mma_16x8x16<T>(o[2 * n + 1], pf[kk], b[2], b[3]);
      }
  }

  // join the warps: o and l rescaled to the block's maximum
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  cp_async_wait<0>();
  float* s_m = reinterpret_cast<float*>(smem + L::kRing);
  float* s_l = s_m + kWarps * kRows;
  if (kq == 0) {
    s_m[warp * kRows + g] = m[0];
    s_m[warp * kRows + g + 8] = m[1];
    s_l[warp * kRows + g] = l[0];
    s_l[warp * kRows + g + 8] = l[1];
  }
  __syncthreads();  // every warp has left its ring
  float* s_o = reinterpret_cast<float*>(smem);  // [kWarps][kRows][HD]
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = g + 8 * e;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * kRows + r]);
    const float f = m[e] == -INFINITY ? 0.f : fast_exp2(m[e] - top);
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
      *reinterpret_cast<float2*>(s_o + (warp * kRows + r) * HD + 8 * n + 2 * kq) =
          make_float2(o[n][2 * e] * f, o[n][2 * e + 1] * f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * (HD / 4); i += kWarps * 32) {
    const int r = i / (HD / 4), col = (i - r * (HD / 4)) * 4;
    const int64_t at = out_row(r);
    if (at < 0) break;  // rows ascend with i
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * kRows + r]);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = s_m[w * kRows + r];
      if (mw != -INFINITY) sum += s_l[w * kRows + r] * fast_exp2(mw - top);
      const float4 x = *reinterpret_cast<const float4*>(s_o + (w * kRows + r) * HD + col);
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    const float inv = 1.f / sum;
    if (col < p.hd)
      *reinterpret_cast<float4*>(p.part_o + (part_row0 + at) * p.hd + col) =
          make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    if (col == 0) p.part_lse[part_row0 + at] = top + log2f(sum);
  }
}

struct JoinParams {
  const float *part_o, *part_lse, *scores, *key_weights;
  float* key_weights_out;
  void* out;
  const int32_t* lengths;
  int64_t score_pitch;
  int batch, capacity, num_heads, kv_heads, group, hd, parts;
};

// One block per (sequence, key / value head) and span of cached keys: lse of the
// group's rows from the ranges'; the first span's block writes the output rows.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const JoinParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ float s_lse[kMaxGroup];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.x / p.kv_heads;
  const int kvh = (int)(blockIdx.x - b * p.kv_heads);
  const int64_t row0 = b * p.num_heads + kvh * p.group;
  const int64_t rows = (int64_t)p.batch * p.num_heads;
  for (int r = warp; r < p.group; r += kJoinThreads / 32) {
    float top = -INFINITY;
    for (int i = lane; i < p.parts; i += 32) top = fmaxf(top, p.part_lse[i * rows + row0 + r]);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    float sum = 0.f;
    for (int i = lane; i < p.parts; i += 32) {
      const float v = p.part_lse[i * rows + row0 + r];
      if (v != -INFINITY) sum += fast_exp2(v - top);
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    const float lse = top + log2f(sum);  // -inf without any key
    if (lane == 0) s_lse[r] = lse;
    if (blockIdx.y == 0) {
      for (int col = lane * 4; col < p.hd; col += 128) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < p.parts; ++i) {
          const float li = p.part_lse[i * rows + row0 + r];
          if (li == -INFINITY) continue;  // an empty range's output is not written
          const float f = fast_exp2(li - lse);
          const float4 x = *reinterpret_cast<const float4*>(p.part_o + (i * rows + row0 + r) * p.hd + col);
          v.x = fmaf(f, x.x, v.x);
          v.y = fmaf(f, x.y, v.y);
          v.z = fmaf(f, x.z, v.z);
          v.w = fmaf(f, x.w, v.w);
        }
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (row0 + r) * p.hd + col) =
            make_uint2(Pack<T>::two(v.x, v.y), Pack<T>::two(v.z, v.w));
      }
    }
  }
  if (p.scores == nullptr) return;
  __syncthreads();
  const int n = min(max(__ldg(p.lengths + b), 0), p.capacity);
  const int64_t base = ((int64_t)b * p.kv_heads + kvh) * p.capacity;
  const int to = min((int)(blockIdx.y + 1) * kWeightSpan, p.capacity);
  for (int c = blockIdx.y * kWeightSpan + threadIdx.x; c < to; c += kJoinThreads) {
    float sum = 0.f;
    if (c < n)
      for (int r = 0; r < p.group; ++r) sum += fast_exp2(p.scores[(row0 + r) * p.score_pitch + c] - s_lse[r]);
    p.key_weights_out[base + c] = p.key_weights[base + c] + sum;
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Ranges for `units` blocks-per-range over `keys` keys: enough blocks to fill the
// GPU's resident blocks a few times over, ranges of 64 to 1024 keys.
void cut_ranges(int64_t units, int64_t keys, int& parts, int& part_keys) {
  if (keys == 0) {
    parts = 0;
    part_keys = 64;
    return;
  }
  int64_t n = ceil_div(8 * (int64_t)sm_count(), units);
  n = std::max(n, ceil_div(keys, 1024));
  n = std::max<int64_t>(1, std::min(n, ceil_div(keys, 64)));
  part_keys = (int)(ceil_div(ceil_div(keys, n), 64) * 64);
  parts = (int)ceil_div(keys, part_keys);
}

Cuts cuts_of(int64_t batch, int64_t prefix, int64_t capacity, int64_t num_heads, int64_t kv_heads, int64_t hd) {
  Cuts c{};
  const int64_t group = num_heads / kv_heads, rows = batch * group;
  cut_ranges(batch * kv_heads * ceil_div(group, kRows), capacity, c.cache_parts, c.cache_keys);
  c.prefix_tiles = prefix > 0 && rows > 32;
  if (!c.prefix_tiles) {
    cut_ranges(kv_heads * ceil_div(rows, kRows), prefix, c.prefix_parts, c.prefix_keys);
    return c;
  }
  // Persistent blocks, one per SM: the number of ranges with the least time, in key
  // tiles of 128: waves x (tiles of a range + about 2 for its start and end).
  const int64_t units = kv_heads * ceil_div(batch, plan_positions(group, hd)), tiles = ceil_div(prefix, 128);
  int64_t best = 1, best_time = INT64_MAX;
  for (int64_t n = 1; n <= std::min<int64_t>(tiles, 64); ++n) {
    const int64_t per = ceil_div(tiles, n);
    if (ceil_div(tiles, per) != n) continue;
    const int64_t time = ceil_div(units * n, sm_count()) * (per + 2) * 16 + n;
    if (time < best_time) best_time = time, best = n;
  }
  c.prefix_keys = (int)(ceil_div(tiles, best) * 128);
  c.prefix_parts = (int)best;
  return c;
}

struct Workspace {
  size_t part_o, part_lse, scores, total;  // byte offsets
  int64_t pitch;
};
Workspace workspace_of(const Cuts& c, int64_t batch, int64_t capacity, int64_t num_heads, int64_t hd, bool weights) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  const size_t rows = (size_t)batch * num_heads;
  Workspace w;
  w.pitch = (capacity + 3) / 4 * 4;
  w.part_o = 0;
  w.part_lse = up((size_t)c.parts() * rows * hd * 4);
  w.scores = w.part_lse + up((size_t)c.parts() * rows * 4);
  w.total = w.scores + (weights ? up(rows * (size_t)w.pitch * 4) : 0);
  return w;
}

template <typename T, int HD>
int launch_ranges(const RangeParams& p, int64_t blocks, cudaStream_t stream) {
  using L = RangeSmem<HD>;
  auto kern = range_kernel<T, HD>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  TTJ_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (dev >= 64 || !(done.load(std::memory_order_acquire) & bit)) {
    TTJ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
    done.fetch_or(bit, std::memory_order_release);
  }
  TTJ_CUDA_TRY(launch_pdl(kern, dim3((unsigned)blocks), dim3(kWarps * 32), L::kTotal, stream, p));
  return TTJ_OK;
}

template <typename T>
int launch_decode(const ttj_shared_prefix_attn_args& a, cudaStream_t stream) {
  const Cuts c = cuts_of(a.batch, a.prefix_len, a.capacity, a.num_heads, a.num_kv_heads, a.head_dim);
  const bool weights = a.key_weights != nullptr && a.capacity > 0;
  const Workspace w = workspace_of(c, a.batch, a.capacity, a.num_heads, a.head_dim, a.key_weights != nullptr);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  float* part_o = reinterpret_cast<float*>(ws + w.part_o);
  float* part_lse = reinterpret_cast<float*>(ws + w.part_lse);
  float* scores = weights ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  const int64_t group = a.num_heads / a.num_kv_heads;
  if (c.prefix_tiles)
    if (int rc = launch_prefix_parts(a, part_o, part_lse, c.prefix_parts, c.prefix_keys, stream)) return rc;
  RangeParams p{};
  p.q = a.q;
  p.pk = a.prefix_k;
  p.pv = a.prefix_v;
  p.kc = a.k_cache;
  p.vc = a.v_cache;
  p.lengths = a.lengths;
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.scores = scores;
  p.q_seq = a.q_seq_stride;
  p.q_head = a.q_head_stride;
  p.pk_row = a.prefix_k_row_stride;
  p.pk_head = a.prefix_k_head_stride;
  p.pv_row = a.prefix_v_row_stride;
  p.pv_head = a.prefix_v_head_stride;
  p.kc_seq = a.k_seq_stride;
  p.kc_row = a.k_row_stride;
  p.kc_head = a.k_head_stride;
  p.vc_seq = a.v_seq_stride;
  p.vc_row = a.v_row_stride;
  p.vc_head = a.v_head_stride;
  p.score_pitch = w.pitch;
  p.batch = (int)a.batch;
  p.prefix = (int)a.prefix_len;
  p.capacity = (int)a.capacity;
  p.num_heads = (int)a.num_heads;
  p.kv_heads = (int)a.num_kv_heads;
  p.group = (int)group;
  p.hd = (int)a.head_dim;
  p.prefix_row_tiles = (int)ceil_div(a.batch * group, kRows);
  p.prefix_keys = c.prefix_keys;
  p.prefix_parts = c.prefix_parts;
  p.prefix_blocks = c.prefix_tiles ? 0 : (int)(c.prefix_parts * a.num_kv_heads * p.prefix_row_tiles);
  p.cache_row_tiles = (int)ceil_div(group, kRows);
  p.cache_keys = c.cache_keys;
  p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  const int64_t blocks = p.prefix_blocks + (int64_t)c.cache_parts * a.batch * a.num_kv_heads * p.cache_row_tiles;
  if (blocks >= (int64_t)1 << 31) return fail(TTJ_ERR_UNSUPPORTED, "too many attention work items");
  if (blocks > 0) {
    int rc = a.head_dim <= 64    ? launch_ranges<T, 64>(p, blocks, stream)
             : a.head_dim <= 128 ? launch_ranges<T, 128>(p, blocks, stream)
                                 : launch_ranges<T, 256>(p, blocks, stream);
    if (rc) return rc;
  }
  JoinParams j{};
  j.part_o = part_o;
  j.part_lse = part_lse;
  j.scores = scores;
  j.key_weights = a.key_weights;
  j.key_weights_out = a.key_weights_out;
  j.out = a.out;
  j.lengths = a.lengths;
  j.score_pitch = w.pitch;
  j.batch = p.batch;
  j.capacity = p.capacity;
  j.num_heads = p.num_heads;
  j.kv_heads = p.kv_heads;
  j.group = p.group;
  j.hd = p.hd;
  j.parts = c.parts();
  const dim3 grid((unsigned)(a.batch * a.num_kv_heads), weights ? (unsigned)ceil_div(a.capacity, kWeightSpan) : 1u);
  if (grid.y > 65535u) return fail(TTJ_ERR_UNSUPPORTED, "capacity above what key_weights supports");
  TTJ_CUDA_TRY(launch_pdl(join_kernel<T>, grid, dim3(kJoinThreads), 0, stream, j));
  return TTJ_OK;
}

}  // namespace

size_t shared_prefix_attn_workspace(int64_t batch, int64_t prefix_len, int64_t capacity, int64_t num_heads,
                                    int64_t num_kv_heads, int64_t head_dim, bool with_key_weights) {
  const Cuts c = cuts_of(batch, prefix_len, capacity, num_heads, num_kv_heads, head_dim);
  return workspace_of(c, batch, capacity, num_heads, head_dim, with_key_weights).total;
}

int launch_shared_prefix_attn(const ttj_shared_prefix_attn_args& a, cudaStream_t stream) {
  return a.dtype == TTJ_F16 ? launch_decode<__half>(a, stream) : launch_decode<__nv_bfloat16>(a, stream);
}

}  // namespace ttj
