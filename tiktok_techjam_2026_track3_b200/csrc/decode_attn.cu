// One decode step over a prefix shared by the batch and each sequence's own cache.
//
// The softmax over all of a row's keys splits into ranges, each giving the partial
//   o_i = sum_u 2^(s_u - lse_i) v_u,   lse_i = log2 sum_u 2^s_u   (s = scale log2(e) q.k)
// and joins as  o = sum_i 2^(lse_i - lse) o_i,  lse = log2 sum_i 2^lse_i.  A range whose
// keys all score -inf has lse_i = -inf and o_i = sum_u 0 v_u: zeros, so that its factor 0
// leaves the others' sum as it is (and NaN where such a key's value is infinite or NaN).
//
// Caches: bound by their bytes, so the work is cut by bytes.  The steps (16
// keys of one cache and head) of all caches form one line, in order; each warp of a
// fixed grid takes an equal stretch of it, whatever the lengths, and streams it
// through its own ring of asynchronous copies (no block barrier, the ring runs on
// across cache boundaries).  Where a stretch enters and leaves a cache it leaves a
// partial result.  A group has few rows (group heads), so the products run on warp
// tiles of 8 or 16 rows.  Cache rows past the length are never read: their copies are
// zero-filled.  (One block per cache range of at most 1024 keys, joined through
// shared memory, took 36 us where the line takes 28 for 33 sequences of up to 2100
// keys, 16 heads of 64: a range's start and end cost as much as its keys.  The line
// streams 128 caches of 1000 to 4096 keys, 8 heads of 128, at 6.4 TB/s, a plain copy's
// rate, with a prefix of 2048 keys among its steps.)
//
// Prefix: with many rows (batch x group) the 128-row tensor-core kernel
// (launch_prefix_parts), which reads the prefix once for up to 256 rows.  With few, or
// with caches long enough to hide it, the prefix's steps, a row tile of the batch at a
// time, come first in the same line: they read it from L2 while the caches' steps wait
// for HBM (cuts_of weighs the two).
//
// Then one kernel joins the partial results and, with key_weights, turns the stored
// scores into probabilities with the rows' final lse and adds them up over the group.
#include <algorithm>
#include <atomic>

#include "attn_math.cuh"
#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace ttj {
namespace {

constexpr int kWarps = 4;
// 256 threads: 45.3 us a step of 33 sequences of 16 ungrouped heads of 64 (128: 43.6)
// and 246.9 us for 128 caches of up to 4096 keys (245.2); 64 with half the step 43.5 and 248.1.
constexpr int kJoinThreads = 128;
constexpr int kWeightStep = 1024;  // cached keys per join block and step
constexpr int64_t kL2Bytes = (int64_t)126 << 20;  // caches above it that are read once: evict-first
constexpr int kMinSteps = 2;       // of a stretch
// Beside the prefix kernel: up to kShareWaves times as many blocks as stay resident,
// with stretches of at least kShareSteps (128 sequences behind 16384 keys with up to
// 4096 cached 221 us a step, with 2 or 16 waves 221 and 234; 128 of 16 heads of 64
// behind 8192 with up to 1000 cached 60.1, with stretches of 8 steps 67.7, 48 64.7).
constexpr int kShareWaves = 8, kShareSteps = 24;

// NR: row tiles of 8 (group heads) that a warp carries, 1 or 2.
template <int HD, int NR>
struct LineShape {
  static constexpr int kKeys = 16;                       // per step
  static constexpr int kStages = 3;
  static constexpr int kTensorBytes = kKeys * HD * 2;
  static constexpr int kStageBytes = 2 * kTensorBytes;   // K and V
  static constexpr int kTotal = kWarps * kStages * kStageBytes;
  // by shared memory; at head_dim 128 three blocks of two stages measured 1 to 3%
  // slower, at 64 three blocks of four stages 0 to 2%
  static constexpr int kBlocksPerSm = HD == 256 ? 1 : (HD == 64 ? 4 : 2);
};
constexpr int kStepKeys = 16;
int line_blocks_per_sm(int64_t hd) { return hd > 128 ? 1 : (hd > 64 ? 2 : 4); }

// How the step is cut (host).
struct Cuts {
  bool prefix_tiles;        // prefix on the 128-row tensor-core kernel, in
  int tile_parts, tile_keys;  // tile_parts ranges of tile_keys keys, on
  int tile_blocks;          // at most this many blocks (one per SM)
  int blocks;               // of the line's grid; workers = blocks * kWarps / heads
  int tile_rows;            // rows of a warp's tile, 8 or 16
  int prefix_row_tiles;     // row tiles of the batch x group rows when the line has the prefix, else 0
  int cache_row_tiles;      // of a group
  int heads;                // consecutive key / value heads that a worker's warps take side by side
  int64_t units;            // (heads, row tile) of the prefix, (sequence, heads, row tile) of the caches
  int pitch;                // rows of a partial result
};

// The line: positions [0, prefix_steps * prefix units) of the prefix, then the
// caches' sequence by sequence, `heads` heads at a time.  A worker is as many warps,
// one per head: in the usual [rows][heads][head_dim] layout they read neighbouring
// pieces of the same rows at about the same time, which DRAM pages reward.  A partial
// result's index is its unit plus its worker (along the line one of the two grows
// from each to the next), then its head.
struct LineParams {
  const void *q, *pk, *pv, *kc, *vc;
  const int32_t* lengths;
  float *part_o, *part_lse;            // [units + workers][heads][pitch][hd], [units + workers][heads][pitch]
  int64_t* before;                     // [B + 2] steps per (head, row tile) of the sequences before, of all, and the stretch
  float* scores;                       // [B][Hq][score_pitch] of the cached keys, or null
  int64_t q_seq, q_head, pk_row, pk_head, pv_row, pv_head, kc_seq, kc_row, kc_head, vc_seq, vc_row, vc_head;
  int64_t score_pitch;
  int batch, prefix, capacity, num_heads, head_groups, heads, group, hd;  // kv heads = head_groups * heads
  int prefix_units, prefix_row_tiles, cache_row_tiles, prefix_steps, pitch;
  int after_prefix;         // launched behind the prefix kernel of the same step
  int large_caches;         // they are larger than L2 and read once
  float scale_log2;
};

__host__ __device__ inline int64_t stretch_of(int64_t total_steps, int workers) {
  const int64_t q = (total_steps + workers - 1) / workers;
  return q < kMinSteps ? kMinSteps : q;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0), "l"(policy)
               : "memory");
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

// Transpose of an 8 x 8 matrix of 16-bit elements held one row per four lanes.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Steps of sequence b per (head, row tile).
__device__ __forceinline__ int seq_steps(const LineParams& p, int64_t b) {
  return (min(max(__ldg(p.lengths + b), 0), p.capacity) + kStepKeys - 1) / kStepKeys;
}

// A place in the line: unit, sequence, head group, row tile, the key of the next step
// and the unit's keys.
struct Place {
  int64_t unit, b;
  int hg, rt, key, keys;
  bool cached;
};

// The products are transposed, S^T = K Q^T and O^T = V^T P^T, so that the keys (then
// the dimensions) fill the 16-row side of the matrix instruction and 8 heads its
// narrow side: a group of up to 8 pays for 8 rows, not 16.  S^T's accumulators
// become P^T's operand by two 8 x 8 register transposes per 16 keys.
template <typename T, int HD, int NR>
__global__ void __launch_bounds__(kWarps * 32, LineShape<HD, NR>::kBlocksPerSm)
line_kernel(const LineParams p) {
  using L = LineShape<HD, NR>;
  constexpr int kKeys = L::kKeys, kStages = L::kStages;
  constexpr int kChunks = HD / 8;
  constexpr int kRows = 8 * NR;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t s_before[kWarps * 32 + 1];  // steps before each thread's sequences, and of all
  // Behind the prefix kernel of the same step nothing of that kernel is read, and it
  // has let this one start only once everything before it was complete: only block 0
  // waits, at its end, which keeps this grid's end, and so the join, behind both (a
  // block that waits holds its place on the SM).
  if (!p.after_prefix) grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, kq = lane & 3;

  // Steps before each thread's run of consecutive sequences.
  const int64_t run = ((int64_t)p.batch + kWarps * 32 - 1) / (kWarps * 32);
  const int64_t b0 = min(threadIdx.x * run, (int64_t)p.batch), b1 = min(b0 + run, (int64_t)p.batch);
  {
    int64_t sum = 0;
    for (int64_t b = b0; b < b1; ++b) sum += seq_steps(p, b);
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) s_before[warp] = inc;
    __syncthreads();
    int64_t base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += s_before[w];
      all += s_before[w];
    }
    __syncthreads();
    s_before[threadIdx.x] = base + inc - sum;
    if (threadIdx.x == 0) s_before[kWarps * 32] = all;
    if (blockIdx.x == 0) {  // for the join
      int64_t at = base + inc - sum;
      for (int64_t b = b0; b < b1; ++b) {
        p.before[b] = at;
        at += seq_steps(p, b);
      }
      if (threadIdx.x == 0) {
        p.before[p.batch] = all;
        p.before[p.batch + 1] =
            stretch_of((int64_t)p.prefix_steps * p.prefix_units + all * p.head_groups * p.cache_row_tiles,
                       gridDim.x * kWarps / p.heads);
      }
    }
    __syncthreads();
  }
  const int64_t per_step = (int64_t)p.head_groups * p.cache_row_tiles;  // units of a sequence
  const int64_t prefix_total = (int64_t)p.prefix_steps * p.prefix_units;
  const int64_t total = prefix_total + s_before[kWarps * 32] * per_step;
  const int side = warp % p.heads;       // this warp's head among the worker's
  const int64_t worker = (int64_t)blockIdx.x * (kWarps / p.heads) + warp / p.heads;
  const int64_t stretch = stretch_of(total, gridDim.x * kWarps / p.heads);
  const int64_t from = worker * stretch;
  const int steps = (int)min(stretch, total - from);
  if (steps <= 0) {  // uniform over the warp; no block barrier follows
    if (p.after_prefix && blockIdx.x == 0) grid_dependency_wait();
    return;
  }

  Place at;
  if (from < prefix_total) {
    at.cached = false;
    at.unit = from / p.prefix_steps;
    at.hg = (int)(at.unit / p.prefix_row_tiles);
    at.rt = (int)(at.unit - (int64_t)at.hg * p.prefix_row_tiles);
    at.key = (int)(from - at.unit * p.prefix_steps) * kKeys;
    at.keys = p.prefix;
    at.b = -1;
  } else {
    const int64_t line = from - prefix_total;
    const int64_t want = line / per_step;  // the sequence b with before[b] <= want < before[b + 1]
    int64_t t = -1;                        // last thread's run starting at or before it
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += __popc(__ballot_sync(0xffffffffu, s_before[32 * w + lane] <= want));
    int64_t b = t * run, base = s_before[t];
    for (;;) {  // 32 sequences at a time
      const int64_t mine = b + lane;
      const int64_t n = mine < p.batch ? seq_steps(p, mine) : 0;
      int64_t inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, base + inc > want);
      if (past != 0u) {
        const int l = __ffs(past) - 1;
        b += l;
        base += __shfl_sync(0xffffffffu, inc - n, l);
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
      b += 32;
    }
    const int64_t n = seq_steps(p, b);
    const int64_t in_seq = line - base * per_step;
    const int64_t u = in_seq / n;
    at.cached = true;
    at.b = b;
    at.unit = p.prefix_units + b * per_step + u;
    at.hg = (int)(u / p.cache_row_tiles);
    at.rt = (int)(u - (int64_t)at.hg * p.cache_row_tiles);
    at.key = (int)(in_seq - u * n) * kKeys;
    at.keys = min(max(__ldg(p.lengths + b), 0), p.capacity);
  }
  // The place after a step; only called while steps remain.
  auto advance = [&](Place& x) {
    x.key += kKeys;
    if (x.key < x.keys) return;
    x.key = 0;
    ++x.unit;
    if (x.cached) {
      if (++x.rt < p.cache_row_tiles) return;
      x.rt = 0;
      if (++x.hg < p.head_groups) return;
    } else {
      if (++x.rt < p.prefix_row_tiles) return;
      x.rt = 0;
      if (++x.hg < p.head_groups) return;
      x.cached = true;
    }
    x.hg = 0;
    do {
      ++x.b;
      x.keys = min(max(__ldg(p.lengths + x.b), 0), p.capacity);
    } while (x.keys == 0);
    x.unit = p.prefix_units + x.b * per_step;
  };

  const uint32_t ring_s = smem_u32(smem) + warp * kStages * L::kStageBytes;
  // Copies: lane -> 16-byte chunk ld_chunk of rows ld_row, ld_row + kRowsPerPass, ...;
  // chunk c of row r lies at c ^ (r & 7), so that eight rows' equal chunks fall into
  // different banks.
  const int ld_chunk = lane % kChunks, ld_row = lane / kChunks;
  constexpr int kRowsPerPass = 32 / kChunks;
  const bool ld_col = ld_chunk * 8 < p.hd;
  const uint32_t ld_dst = ring_s + ld_row * (HD * 2) + ((ld_chunk ^ ld_row) << 4);
  Place next = at;  // where the loads are
  const T *kp = nullptr, *vp = nullptr;  // this lane's first element of the next step
  bool moved = true;                     // `next` has entered another unit
  int64_t kstep = 0, vstep = 0;
  uint64_t policy = 0;
  auto load = [&](int i) {
    if (i < steps) {
      if (moved) {
        // Caches larger than L2 leave it first, so that the prefix, the partial results
        // and the scores stay there for their readers.
        if (next.cached && p.large_caches)
          asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        else
          asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
        kstep = next.cached ? p.kc_row : p.pk_row;
        vstep = next.cached ? p.vc_row : p.pv_row;
        kp = next.cached ? static_cast<const T*>(p.kc) + next.b * p.kc_seq + (next.hg * p.heads + side) * p.kc_head
                         : static_cast<const T*>(p.pk) + (next.hg * p.heads + side) * p.pk_head;
        vp = next.cached ? static_cast<const T*>(p.vc) + next.b * p.vc_seq + (next.hg * p.heads + side) * p.vc_head
                         : static_cast<const T*>(p.pv) + (next.hg * p.heads + side) * p.pv_head;
        kp += (next.key + ld_row) * kstep + ld_chunk * 8;
        vp += (next.key + ld_row) * vstep + ld_chunk * 8;
      }
      const int left = next.keys - next.key - ld_row;
      const uint32_t dst = ld_dst + (i % kStages) * L::kStageBytes;
#pragma unroll
      for (int r = 0; r < kKeys; r += kRowsPerPass) {
        // rows past the end are filled with zeros (their address, this lane's
        // first row or row 0 of the unit's keys, is not read)
        const bool ok = ld_col && r < left;
        const uint32_t to = (dst ^ ((r & 7) << 4)) + r * (HD * 2);
        cp_async16(to, ok ? kp + r * kstep : p.q, ok, policy);
        cp_async16(to + L::kTensorBytes, ok ? vp + r * vstep : p.q, ok, policy);
      }
      if (i + 1 < steps) {
        const int64_t unit = next.unit;
        advance(next);
        moved = next.unit != unit;
        kp += kKeys * kstep;
        vp += kKeys * vstep;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i);

  // Fragments of this lane: Q^T (B side) head g, dimensions 16 kk + 2 kq (+ 8);
  // S^T keys g and g + 8, heads 2 kq and 2 kq + 1; O^T dimensions 16 n + g (+ 8),
  // the same heads; per row tile.
  uint32_t qf[NR][HD / 16][2];
  float o[NR][HD / 16][4];
  float m[NR][2], l[NR][2];
  int64_t at_row[NR][2];         // output rows ([B][Hq]) of heads 2 kq and 2 kq + 1, or -1
  bool fresh = true;
  // operand addresses within a stage, before the step's and column's offset
  const int r7 = lane & 7;
  const uint32_t k_at = (r7 + ((lane >> 3) & 1) * 8) * (HD * 2) + (((lane >> 4) ^ r7) << 4);
  const uint32_t v_at = L::kTensorBytes + (r7 + (lane >> 4) * 8) * (HD * 2) + ((((lane >> 3) & 1) ^ r7) << 4);
  for (int i = 0; i < steps; ++i) {
    if (fresh) {
      // The unit's rows: tile row r is row i0 + r of the batch x group rows.
      const int64_t i0 = (at.cached ? at.b * p.group : 0) + at.rt * kRows;
      const int64_t end = at.cached ? (at.b + 1) * p.group : (int64_t)p.batch * p.group;
      auto row_of = [&](int r, int64_t& b, int& head) -> bool {
        const int64_t x = i0 + r;
        b = at.cached ? at.b : x / p.group;
        head = (at.hg * p.heads + side) * p.group + (int)(x - b * p.group);
        return x < end;
      };
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        int64_t b;
        int head;
        const bool ok = row_of(8 * t + g, b, head);
        const T* src = static_cast<const T*>(p.q) + b * p.q_seq + head * p.q_head + 2 * kq;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            qf[t][kk][e] = ok && 16 * kk + 8 * e < p.hd ? __ldg(reinterpret_cast<const uint32_t*>(src + 16 * kk + 8 * e)) : 0u;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          at_row[t][e] = row_of(8 * t + 2 * kq + e, b, head) ? b * p.num_heads + head : -1;
          m[t][e] = -INFINITY;
          l[t][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < HD / 16; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][n][e] = 0.f;
      }
      fresh = false;
    }
    cp_async_wait<kStages - 2>();
    __syncwarp();
    load(i + kStages - 1);
    const int left = at.keys - at.key;
    const uint32_t stage = ring_s + (i % kStages) * L::kStageBytes;
    float s[NR][4];
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      uint32_t a[4];
      ldmatrix_x4(a, (stage + k_at) ^ (kk << 5));
#pragma unroll
      for (int t = 0; t < NR; ++t) mma_16x8x16<T>(s[t], a, qf[t][kk][0], qf[t][kk][1]);
    }
    uint32_t pf[NR][2];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] *= p.scale_log2;   // s[t][e]: key g + 8 (e >> 1), head 2 kq + (e & 1)
      if (left < kKeys) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = g + 8 * (e >> 1) < left ? s[t][e] : -INFINITY;
      }
      if (at.cached && p.scores != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = g + 8 * (e >> 1);
          if (at_row[t][e & 1] >= 0 && col < left) p.scores[at_row[t][e & 1] * p.score_pitch + at.key + col] = s[t][e];
        }
      }
      float alpha[2], ref[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[t][e], s[t][e + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = mx > m[t][e] + 8.f ? mx : m[t][e];  // the reference moves lazily: P <= 2^8
        ref[e] = mn == -INFINITY ? 0.f : mn;
        alpha[e] = fast_exp2(m[t][e] - ref[e]);
        m[t][e] = mn;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) l[t][e] *= alpha[e];
#pragma unroll
        for (int n = 0; n < HD / 16; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][n][e] *= alpha[e & 1];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // keys g, then g + 8
        const float e0 = fast_exp2(s[t][2 * h] - ref[0]), e1 = fast_exp2(s[t][2 * h + 1] - ref[1]);
        l[t][0] += e0;
        l[t][1] += e1;
        pf[t][h] = movmatrix_trans(Pack<T>::two(e0, e1));  // head g, keys 8 h + 2 kq, 8 h + 2 kq + 1
      }
    }
#pragma unroll
    for (int n = 0; n < HD / 16; ++n) {
      uint32_t a[4];
      ldmatrix_x4_trans(a, (stage + v_at) ^ (n << 5));
#pragma unroll
      for (int t = 0; t < NR; ++t) mma_16x8x16<T>(o[t][n], a, pf[t][0], pf[t][1]);
    }
    if (left <= kKeys || i + 1 == steps) {  // the stretch leaves this unit
#pragma unroll
      for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[t][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          if (at_row[t][e] < 0) continue;
          const int64_t row = ((at.unit + worker) * p.heads + side) * p.pitch + 8 * t + 2 * kq + e;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;  // 0: every key scores -inf
          float* out = p.part_o + row * p.hd + g;
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            if (16 * n < p.hd) out[16 * n] = o[t][n][e] * inv;
            if (16 * n + 8 < p.hd) out[16 * n + 8] = o[t][n][e + 2] * inv;
          }
          if (g == 0) p.part_lse[row] = m[t][e] + log2f(sum);
        }
      fresh = true;
    }
    if (i + 1 < steps) advance(at);
  }
  if (p.after_prefix && blockIdx.x == 0) grid_dependency_wait();
}

struct JoinParams {
  const float *tile_o, *tile_lse;      // [tile_parts][B][Hq][hd], [tile_parts][B][Hq]
  const float *part_o, *part_lse;      // the line's
  const int64_t* before;
  const float *scores, *key_weights;
  float* key_weights_out;
  void* out;
  float* lse;                          // [B][Hq] or null
  const int32_t* lengths;
  int64_t score_pitch, rows, out_blocks;
  int spans, span;                     // spans of `span` cached keys
  int row_warps;                       // warps per output row, a power of two up to 8
  int capacity, batch, num_heads, kv_heads, group, hd, tile_parts;
  int prefix_units, prefix_row_tiles, cache_row_tiles, prefix_steps, pitch, tile_rows;
  int heads_shift;                     // log2 of the line's heads
};

// a / b for a, b >= 0: the 32-bit division where it suffices (a 64-bit one is a
// long dependent chain).
__device__ __forceinline__ int64_t div_of(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Where the partial results of one output row are: tile_parts of the prefix's
// tensor-core ranges, then the line's, consecutive per unit.
struct RowParts {
  int64_t row, prefix_first, cache_first;  // first partial row (index * pitch + tile row)
  int prefix_count, cache_count;
};

__device__ __forceinline__ RowParts row_parts(const JoinParams& p, int64_t b, int head) {
  RowParts x;
  x.row = b * p.num_heads + head;
  const int kvh = (uint32_t)head / (uint32_t)p.group, in_group = head - kvh * p.group;
  const int hg = kvh >> p.heads_shift, side = kvh - (hg << p.heads_shift);
  const int64_t per_seq = (int64_t)(p.kv_heads >> p.heads_shift) * p.cache_row_tiles;
  const int64_t prefix_total = (int64_t)p.prefix_steps * p.prefix_units;
  const int64_t before = p.before[b], steps = p.before[b + 1] - before;
  const int64_t stretch = p.before[p.batch + 1];
  auto locate = [&](int64_t unit, int64_t from, int64_t n, int tile_row, int64_t& first, int& count) {
    const int64_t w0 = div_of(from, stretch), w1 = div_of(from + max(n, (int64_t)1) - 1, stretch);
    first = (((unit + w0) << p.heads_shift) + side) * p.pitch + tile_row;
    count = n > 0 ? (int)(w1 - w0 + 1) : 0;
  };
  x.prefix_count = 0;
  x.prefix_first = 0;
  const int rt_shift = p.tile_rows == 16 ? 4 : 3;
  if (p.prefix_units > 0) {
    const int64_t i = b * p.group + in_group;
    const int64_t unit = hg * p.prefix_row_tiles + (i >> rt_shift);
    locate(unit, unit * p.prefix_steps, p.prefix_steps, (int)(i & (p.tile_rows - 1)), x.prefix_first, x.prefix_count);
  }
  const int64_t u = (int64_t)hg * p.cache_row_tiles + (in_group >> rt_shift);
  locate(p.prefix_units + b * per_seq + u, prefix_total + before * per_seq + u * steps, steps,
         in_group & (p.tile_rows - 1), x.cache_first, x.cache_count);
  return x;
}

// i-th partial result: its lse and (float) offset of its output from `tile_o`.
__device__ __forceinline__ float part_at(const JoinParams& p, const RowParts& x, int i, int64_t& offset) {
  if (i < p.tile_parts) {
    const int64_t r = i * p.rows + x.row;
    offset = r * p.hd;
    return p.tile_lse[r];
  }
  i -= p.tile_parts;
  const int64_t next = (int64_t)p.pitch << p.heads_shift;
  const int64_t r = i < x.prefix_count ? x.prefix_first + i * next : x.cache_first + (i - x.prefix_count) * next;
  offset = (p.part_o - p.tile_o) + r * p.hd;
  return p.part_lse[r];
}

// lse of a row over all its partial results (the whole warp; -inf without any key).
__device__ __forceinline__ float row_lse(const JoinParams& p, const RowParts& x, int count) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.f;
  int64_t unused;
  for (int i = lane; i < count; i += 32) {
    const float v = part_at(p, x, i, unused);
    const float t = fmaxf(top, v);
    if (v != -INFINITY) sum = sum * fast_exp2(top - t) + fast_exp2(v - t);
    top = t;
  }
  float all = top;
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, w));
  sum = sum == 0.f ? 0.f : sum * fast_exp2(top - all);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  return all + log2f(sum);
}

// The first out_blocks blocks write the output: `row_warps` warps of a block share a
// row, each with its share of the row's partial results (one warp per row leaves a
// step of few rows waiting for one batch of loads after the other).  The other blocks
// write the weights of a span of cached keys of one (sequence, key / value head).
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const JoinParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x < p.out_blocks) {
    __shared__ float4 s_part[kJoinThreads / 32][64];  // a warp's 256 columns
    const int share = warp & (p.row_warps - 1);       // this warp's among the row's
    const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / 32 / p.row_warps) + warp / p.row_warps;
    if (row < p.rows) {
      const int64_t b = div_of(row, p.num_heads);
      const RowParts x = row_parts(p, b, (int)(row - b * p.num_heads));
      const int count = p.tile_parts + x.prefix_count + x.cache_count;
      const float lse = row_lse(p, x, count);
      if (p.lse != nullptr && share == 0 && lane == 0) p.lse[row] = lse * 0.69314718055994531f;
      for (int col0 = 0; col0 < p.hd; col0 += 128) {
        const int col = col0 + lane * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < count; i0 += 32) {
          int64_t offset = 0;
          float f = -INFINITY;
          if (i0 + lane < count) f = part_at(p, x, i0 + lane, offset);
          f = f == -INFINITY ? 0.f : fast_exp2(f - lse);
          const int n = min(32, count - i0);
          for (int q0 = share; q0 < n; q0 += 8 * p.row_warps) {
            float4 y[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int i = q0 + q * p.row_warps;
              const int64_t oi = __shfl_sync(0xffffffffu, offset, i & 31);
              y[q] = i < n && col < p.hd ? __ldg(reinterpret_cast<const float4*>(p.tile_o + oi + col))
                                         : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int i = q0 + q * p.row_warps;
              const float fi = __shfl_sync(0xffffffffu, f, i & 31);
              if (i < n) {
                v.x = fmaf(fi, y[q].x, v.x);
                v.y = fmaf(fi, y[q].y, v.y);
                v.z = fmaf(fi, y[q].z, v.z);
                v.w = fmaf(fi, y[q].w, v.w);
              }
            }
          }
        }
        s_part[warp][(col0 >> 2) + lane] = v;
      }
    }
    __syncthreads();
    if (row < p.rows && share == 0) {
      for (int col = lane * 4; col < p.hd; col += 128) {
        float4 v = s_part[warp][col >> 2];
        for (int w = 1; w < p.row_warps; ++w) {
          const float4 y = s_part[warp + w][col >> 2];
          v.x += y.x;
          v.y += y.y;
          v.z += y.z;
          v.w += y.w;
        }
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + row * p.hd + col) =
            make_uint2(Pack<T>::two(v.x, v.y), Pack<T>::two(v.z, v.w));
      }
    }
    return;
  }
  __shared__ float s_lse[kMaxGroup];
  const int64_t rest = blockIdx.x - p.out_blocks;
  const int64_t bh = div_of(rest, p.spans);
  const int64_t b = div_of(bh, p.kv_heads);
  const int kvh = (int)(bh - b * p.kv_heads);
  const int n = min(max(__ldg(p.lengths + b), 0), p.capacity);
  const int from = (int)(rest - bh * p.spans) * p.span, to = (int)min((int64_t)from + p.span, (int64_t)p.capacity);
  constexpr int kPer = kWeightStep / kJoinThreads;
  constexpr int kAhead = 4;      // rows whose scores are read together
  const float* scores = p.scores + (b * p.num_heads + kvh * p.group) * p.score_pitch;
  float x[kAhead][kPer];
  auto fetch = [&](int c0, int r0) {
#pragma unroll
    for (int r = 0; r < kAhead; ++r)
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int c = c0 + q * kJoinThreads;
        x[r][q] = r0 + r < p.group && c < min(n, to) ? __ldg(scores + (r0 + r) * p.score_pitch + c) : -INFINITY;
      }
  };
  fetch(from + threadIdx.x, 0);  // before the lse are known
  if (from < n) {                // uniform
    for (int r = warp; r < p.group; r += kJoinThreads / 32) {
      const RowParts y = row_parts(p, b, kvh * p.group + r);
      const float lse = row_lse(p, y, p.tile_parts + y.prefix_count + y.cache_count);
      if (lane == 0) s_lse[r] = lse == -INFINITY ? INFINITY : lse;  // no key counts: no weight
    }
    __syncthreads();
  }
  for (int c0 = from + threadIdx.x; c0 - (int)threadIdx.x < to; c0 += kWeightStep) {
    float w[kPer], sum[kPer];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int c = c0 + q * kJoinThreads;
      w[q] = c < to ? __ldg(p.key_weights + bh * p.capacity + c) : 0.f;
      sum[q] = 0.f;
    }
    if (c0 - (int)threadIdx.x < n) {
      if (c0 != from + (int)threadIdx.x) fetch(c0, 0);
      for (int r0 = 0; r0 < p.group; r0 += kAhead) {
        if (r0 > 0) fetch(c0, r0);
#pragma unroll
        for (int r = 0; r < kAhead; ++r)
          if (r0 + r < p.group) {
            const float lse = s_lse[r0 + r];
#pragma unroll
            for (int q = 0; q < kPer; ++q) sum[q] += fast_exp2(x[r][q] - lse);
          }
      }
    }
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int c = c0 + q * kJoinThreads;
      if (c < to) p.key_weights_out[bh * p.capacity + c] = w[q] + (c < n ? sum[q] : 0.f);
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Cuts cuts_of(int64_t batch, int64_t prefix, int64_t capacity, int64_t num_heads, int64_t kv_heads, int64_t hd) {
  Cuts c{};
  const int64_t group = num_heads / kv_heads, rows = batch * group;
  const int sms = sm_count();
  const int64_t tile = group <= 8 ? 8 : 16;
  c.tile_rows = (int)tile;
  c.cache_row_tiles = (int)ceil_div(group, tile);
  c.heads = kv_heads % 4 == 0 ? 4 : (kv_heads % 2 == 0 ? 2 : 1);
  const int64_t head_groups = kv_heads / c.heads, line_tiles = ceil_div(rows, tile);
  // The prefix on the tensor-core tiles, in us: a key tile of a block's 256 rows takes
  // ~1.9 and a range about two more for its start and end; its fp32 results are written
  // and read at ~5 TB/s.  `best` ranges take the least.
  const int64_t units = kv_heads * ceil_div(batch, plan_positions(group, hd)), tiles = ceil_div(prefix, 128);
  auto ranges = [&](int blocks, int64_t& best) {
    double least = 1e30;
    best = 1;
    for (int64_t n = 1; n <= std::min<int64_t>(tiles, 64); ++n) {
      const int64_t per = ceil_div(tiles, n);
      if (ceil_div(tiles, per) != n) continue;
      const double us = 1.9 * (double)(ceil_div(units * n, blocks) * (per + 2)) +
                        (double)(n * batch * num_heads) * (double)hd * 8e-6 / 5.;
      if (us < least) least = us, best = n;
    }
    return least;
  };
  if (prefix > 0) {
    // Or in the line, whose warps stream steps at ~10 TB/s from L2 (a unit's start and
    // end costing about four) while its caches, taken as 0.4 full, come from HBM at 6.4:
    // as long as those bound it, the prefix's steps are nearly free, and a launch and
    // the tiles' results are saved.  (Line against tiles: 33 sequences of 16 heads of
    // 64 behind 1001 keys 38.4 us against 43.3, 4 of 32 / 8 heads of 128 behind 2048
    // 18.9 against 25.8, 64 behind 2048 with up to 4096 cached 117 against 129; 32
    // behind 4096 with up to 512 43.5 against 28.8.)  Many partial results of a row
    // cost the join ~0.02 us each.
    const double step = 4e-6 * (double)(kv_heads * kStepKeys) * (double)hd;  // MB of K and V
    const double cache_units = (double)(batch * c.cache_row_tiles), cache_steps = 0.4 * (double)capacity / kStepKeys;
    const double hbm = step * (double)batch * cache_steps / 6.4;
    const double line = step * cache_units * (capacity > 0 ? cache_steps + 4. : 0.) / 10.;
    const double steps = (double)(line_tiles * ceil_div(prefix, kStepKeys));
    const double workers = (double)(line_blocks_per_sm(hd) * (int64_t)sms * kWarps / c.heads);
    const double per_worker = std::max((double)kMinSteps, (steps + cache_units * cache_steps) * (double)head_groups / workers);
    const double more = std::max(hbm, line + step * steps / 10.) - std::max(hbm, line) +
                        0.02 * (double)ceil_div(prefix, kStepKeys) / per_worker;
    int64_t unused;
    c.prefix_tiles = more > ranges(sms, unused);
  }
  c.prefix_row_tiles = prefix > 0 && !c.prefix_tiles ? (int)line_tiles : 0;
  c.units = head_groups * c.prefix_row_tiles + batch * head_groups * c.cache_row_tiles;
  c.pitch = c.prefix_row_tiles > 0 ? (int)tile : (int)std::min<int64_t>(group, tile);
  // As many blocks as stay resident, and no more than the longest line has work for.
  const int64_t steps = head_groups * (c.prefix_row_tiles * ceil_div(prefix, kStepKeys) +
                                       batch * c.cache_row_tiles * ceil_div(capacity, kStepKeys));
  c.blocks = (int)std::min<int64_t>(line_blocks_per_sm(hd) * (int64_t)sms, ceil_div(steps * c.heads, kMinSteps * kWarps));
  if (!c.prefix_tiles) return c;
  // The two kernels share the GPU: the prefix's persistent blocks (one per SM) leave
  // the caches' blocks the SMs that their work is worth, by a key tile's ~1.9 us and
  // ~80 GB/s that an SM streams, caches taken as 0.6 full; as blocks of either end,
  // the line's take their place.  (Each kernel on the whole GPU in turn: 64 sequences
  // behind 32768 keys 69.8 us a step, shared 67.8.)  Steps of less than ~20 us in all gain
  // nothing (33 sequences of up to 2100 keys: 47 us, shared 53).
  const double prefix_us = 1.9 * (double)(units * tiles);
  const double line_us = 0.6 * 4.0 * (double)(batch * kv_heads * c.cache_row_tiles) * (double)(capacity * hd) / 80e3;
  const int64_t want = (int64_t)(sms * prefix_us / (prefix_us + line_us) + 0.5);
  c.tile_blocks = prefix_us + line_us < 20. * sms
                      ? sms
                      : (int)std::max<int64_t>(std::min<int64_t>(want, sms), std::min(24, sms));
  if (c.tile_blocks < sms) {
    // the line's blocks start as SMs become free: shorter stretches even out their ends
    const int64_t whole = steps * c.heads;
    c.blocks = (int)std::max<int64_t>(c.blocks, std::min<int64_t>(kShareWaves * line_blocks_per_sm(hd) * (int64_t)sms,
                                                                  whole / (kShareSteps * kWarps)));
  }
  int64_t best;
  ranges(c.tile_blocks, best);
  c.tile_keys = (int)(ceil_div(tiles, best) * 128);
  c.tile_parts = (int)best;
  return c;
}

// The regions start on multiples of kWorkspaceAlign, whatever the caller's base (a
// multiple of 16 bytes): the prefix tiles store their results 32 bytes at a time.
constexpr size_t kWorkspaceAlign = 256;

struct Workspace {
  size_t tile_o, tile_lse, part_o, part_lse, before, scores, total;  // byte offsets
  int64_t pitch;                                                     // of the scores
};
Workspace workspace_of(const Cuts& c, int64_t batch, int64_t capacity, int64_t num_heads, int64_t hd, bool weights) {
  auto up = [](size_t v) { return (v + kWorkspaceAlign - 1) / kWorkspaceAlign * kWorkspaceAlign; };
  const size_t rows = (size_t)batch * num_heads;
  const size_t parts = c.blocks > 0 ? (size_t)c.units * c.heads + (size_t)c.blocks * kWarps : 0;
  Workspace w;
  w.pitch = (capacity + 3) / 4 * 4;
  w.tile_o = 0;
  w.tile_lse = w.tile_o + up((size_t)c.tile_parts * rows * hd * 4);
  w.part_o = w.tile_lse + up((size_t)c.tile_parts * rows * 4);
  w.part_lse = w.part_o + up(parts * c.pitch * hd * 4);
  w.before = w.part_lse + up(parts * c.pitch * 4);
  w.scores = w.before + up((size_t)(batch + 2) * 8);
  w.total = w.scores + (weights ? up(rows * (size_t)w.pitch * 4) : 0) + kWorkspaceAlign;  // to round the base up
  return w;
}

template <typename T, int HD, int NR>
int launch_line(const LineParams& p, int blocks, cudaStream_t stream) {
  using L = LineShape<HD, NR>;
  auto kern = line_kernel<T, HD, NR>;
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

template <typename T, int NR>
int dispatch_line(const LineParams& p, int blocks, cudaStream_t stream) {
  if (p.hd <= 64) return launch_line<T, 64, NR>(p, blocks, stream);
  if (p.hd <= 128) return launch_line<T, 128, NR>(p, blocks, stream);
  return launch_line<T, 256, NR>(p, blocks, stream);
}

template <typename T>
int launch_decode(const ttj_shared_prefix_attn_args& a, cudaStream_t stream) {
  const Cuts c = cuts_of(a.batch, a.prefix_len, a.capacity, a.num_heads, a.num_kv_heads, a.head_dim);
  const bool weights = a.key_weights != nullptr && a.capacity > 0;
  const Workspace w = workspace_of(c, a.batch, a.capacity, a.num_heads, a.head_dim, a.key_weights != nullptr);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  ws += (kWorkspaceAlign - reinterpret_cast<uintptr_t>(ws) % kWorkspaceAlign) % kWorkspaceAlign;
  float* tile_o = reinterpret_cast<float*>(ws + w.tile_o);
  float* tile_lse = reinterpret_cast<float*>(ws + w.tile_lse);
  const int64_t group = a.num_heads / a.num_kv_heads;
  if (c.prefix_tiles)
    if (int rc = launch_prefix_parts(a, tile_o, tile_lse, c.tile_parts, c.tile_keys, c.tile_blocks, stream)) return rc;
  LineParams p{};
  p.q = a.q;
  p.pk = a.prefix_k;
  p.pv = a.prefix_v;
  p.kc = a.k_cache;
  p.vc = a.v_cache;
  p.lengths = a.lengths;
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  p.part_lse = reinterpret_cast<float*>(ws + w.part_lse);
  p.before = reinterpret_cast<int64_t*>(ws + w.before);
  p.scores = weights ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
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
  p.heads = c.heads;
  p.head_groups = (int)a.num_kv_heads / c.heads;
  p.group = (int)group;
  p.hd = (int)a.head_dim;
  p.prefix_row_tiles = c.prefix_row_tiles;
  p.prefix_units = p.head_groups * c.prefix_row_tiles;
  p.prefix_steps = c.prefix_row_tiles > 0 ? (int)ceil_div(a.prefix_len, kStepKeys) : 0;
  p.cache_row_tiles = c.cache_row_tiles;
  p.pitch = c.pitch;
  p.after_prefix = c.prefix_tiles;
  // (33 sequences of 16 heads of 64, up to 2100 keys: 37.1 us a step, 39.9 without; 128
  // of up to 2100: 92.9 and 101.4; 8 caches of 4 MB each, that fit: 18.3 and 16.4.)  Not
  // where a group takes several row tiles: each reads the cache again.  (Evict-first, with
  // key weights: 32 heads over 1 of 128, 128 caches of 8192 rows 199 us against 188, 64 of
  // 4096 58 against 62; 128 over 1, 32 of 8192 230 against 195; 24 over 2 of 64, 64 of 8192
  // 123 against 115; without weights 0 to 5% slower.)
  p.large_caches = c.cache_row_tiles == 1 && 4 * a.batch * a.capacity * a.num_kv_heads * a.head_dim > kL2Bytes;
  p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  // Without any cached or prefix key the line is empty, but the join reads `before`.
  const int blocks = std::max(c.blocks, 1);
  if (int rc = c.tile_rows == 8 ? dispatch_line<T, 1>(p, blocks, stream) : dispatch_line<T, 2>(p, blocks, stream))
    return rc;
  JoinParams j{};
  j.tile_o = tile_o;
  j.tile_lse = tile_lse;
  j.part_o = p.part_o;
  j.part_lse = p.part_lse;
  j.before = p.before;
  j.scores = p.scores;
  j.key_weights = a.key_weights;
  j.key_weights_out = a.key_weights_out;
  j.out = a.out;
  j.lse = a.lse;
  j.lengths = a.lengths;
  j.score_pitch = w.pitch;
  j.rows = a.batch * a.num_heads;
  // as many warps per row as keep about four per SM busy
  j.row_warps = kJoinThreads / 32;
  while (j.row_warps > 1 && j.row_warps * j.rows > 4 * (int64_t)sm_count()) j.row_warps /= 2;
  j.out_blocks = ceil_div(j.rows, kJoinThreads / 32 / j.row_warps);
  // A block's start (its rows' lse) costs about two steps: only as many spans as fill
  // the GPU once or twice (twice as many: 0.7 to 1.9% slower).
  const int64_t steps = ceil_div(a.capacity, kWeightStep);
  const int64_t wanted = ceil_div(4 * (int64_t)sm_count(), a.batch * a.num_kv_heads);
  j.span = (int)(ceil_div(steps, std::max<int64_t>(1, std::min(steps, wanted))) * kWeightStep);
  j.spans = weights ? (int)ceil_div(a.capacity, j.span) : 0;
  j.capacity = p.capacity;
  j.batch = p.batch;
  j.num_heads = p.num_heads;
  j.kv_heads = (int)a.num_kv_heads;
  j.group = p.group;
  j.hd = p.hd;
  j.tile_parts = c.tile_parts;
  j.heads_shift = c.heads == 4 ? 2 : c.heads - 1;
  j.prefix_units = p.prefix_units;
  j.prefix_row_tiles = p.prefix_row_tiles;
  j.cache_row_tiles = p.cache_row_tiles;
  j.prefix_steps = p.prefix_steps;
  j.pitch = p.pitch;
  j.tile_rows = c.tile_rows;
  const int64_t grid = j.out_blocks + a.batch * a.num_kv_heads * j.spans;
  if (grid >= (int64_t)1 << 31) return fail(TTJ_ERR_UNSUPPORTED, "batch x capacity above what one call supports");
  TTJ_CUDA_TRY(launch_pdl(join_kernel<T>, dim3((unsigned)grid), dim3(kJoinThreads), 0, stream, j));
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
