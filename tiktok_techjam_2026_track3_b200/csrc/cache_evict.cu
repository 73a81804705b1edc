// Eviction from per-sequence caches by accumulated attention weight, two kernels.
//
// 1. Choosing (weights read once, 4 bytes a row): one cluster of blocks per
//    (sequence, key / value head).  A weight compares as a 32-bit unsigned key in the
//    order of its value; each block keeps its slice of the keys in shared memory.  The
//    key of the last row to keep (the need-th largest) comes digit by digit, 11 + 11 +
//    10 bits: a histogram of the digit over the keys that agree so far, summed over
//    the cluster, tells the digit's value and how many of the rows are still to find.
//    With `cut` that key and `ties` the rows equal to it that stay, row i's slot is
//        above(i) + min(ties, equal(i)),
//    above / equal counting the earlier rows with a larger / an equal key: both counts
//    come from one scan, and equal rows are kept lowest index first by construction.
// 2. Copying (bound by the kept rows' bytes): a warp takes 32 output rows in the
//    order of the output's memory and copies K and V rows in 16-byte pieces, eight
//    rows in flight.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace cg = cooperative_groups;

namespace ttj {
namespace {

constexpr int kThreads = 512;
constexpr int kWarpsPerBlock = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kSliceKeys = 8192;         // keys per block that a cluster is sized for
constexpr int kMaxCluster = 8;
constexpr int kMaxStagedKeys = 49152;    // 192 KB; longer slices are re-read from memory

struct ChooseParams {
  const float* weights;   // [B][H][C]
  const int32_t* lengths;
  float* weights_out;     // [B][H][N]
  int32_t* lengths_out;
  int32_t* positions;     // [B][H][N]
  int kv_heads, capacity, budget, recent;
  int slice;              // rows per block of the cluster (a multiple of kThreads)
  int staged;             // the slice's keys fit in shared memory
};

// Ascending unsigned order of the weights; NaN as -infinity, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// A thread's keys are consecutive; one word of padding per 32 keeps them off each
// other's banks for the row counts that occur (1 to 16 and odd ones).
__device__ __forceinline__ int padded(int i) { return i + (i >> 5); }

// Exclusive prefix over the block of two counts packed as (hi, lo) 32-bit halves,
// and the block's total.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* warp_sums, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarpsPerBlock; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  total = all;
  return before + inc - v;
}

__global__ void __launch_bounds__(kThreads) choose_kernel(const ChooseParams p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint64_t s_warp[kWarpsPerBlock];
  __shared__ uint64_t s_totals;           // this block's (above, equal), read by the cluster
  __shared__ int s_digit, s_need;
  cg::cluster_group cluster = cg::this_cluster();
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = (int)cluster.block_rank(), nblocks = (int)cluster.num_blocks();
  const int64_t bh = blockIdx.x / nblocks;
  const int64_t b = bh / p.kv_heads;
  const int n = min(max(__ldg(p.lengths + b), 0), p.capacity);
  const int kept = min(n, p.budget);
  const float* w = p.weights + bh * p.capacity;
  float* w_out = p.weights_out + bh * p.budget;
  int32_t* pos = p.positions + bh * p.budget;
  const int first = min(rank * p.slice, n), last = min(first + p.slice, n);  // this block's rows
  if (rank == 0 && tid == 0 && bh - b * p.kv_heads == 0) p.lengths_out[b] = kept;
  // output rows past the kept ones
  for (int i = kept + rank * kThreads + tid; i < p.budget; i += nblocks * kThreads) {
    w_out[i] = 0.f;
    pos[i] = -1;
  }
  if (n <= p.budget) {  // uniform over the cluster
    for (int i = first + tid; i < last; i += kThreads) {
      w_out[i] = w[i];
      pos[i] = i;
    }
    return;
  }
  const int old = n - p.recent;         // rows below `old` compete
  int need = p.budget - p.recent;       // for this many places
  const int mine = min(last, old);      // end of this block's competing rows
  if (p.staged) {
    for (int i = first + tid; i < last; i += kThreads) s_keys[padded(i - first)] = weight_key(w[i]);
    __syncthreads();
  }
  auto key_at = [&](int i) -> uint32_t { return p.staged ? s_keys[padded(i - first)] : weight_key(__ldg(w + i)); };

  uint32_t cut = 0xffffffffu;           // need == 0: nothing competes
  if (need > 0) {
    uint32_t prefix = 0, mask = 0;      // digits found so far
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const int bins = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < kBins; i += kThreads) s_hist[i] = 0u;
      __syncthreads();
      for (int i0 = first; i0 < mine; i0 += kThreads) {
        const int i = i0 + tid;
        const uint32_t key = i < mine ? key_at(i) : 0u;
        const bool in = i < mine && (key & mask) == prefix;
        const uint32_t bin = in ? (key >> shift) & (bins - 1) : kBins;
        // equal weights fall into one bin: a warp of one bin adds once
        int same;
        __match_all_sync(0xffffffffu, bin, &same);
        if (same) {
          if (in && lane == 0) atomicAdd(&s_hist[bin], 32u);
        } else if (in) {
          atomicAdd(&s_hist[bin], 1u);
        }
      }
      cluster.sync();
      // largest digit with at least `need` keys at or above it: thread t sums bins
      // [top - 4t - 3, top - 4t] of the cluster, from the largest down
      uint32_t c[4];
      uint64_t sum = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int bin = bins - 1 - (4 * tid + q);
        c[q] = 0u;
        if (bin >= 0)
          for (int r = 0; r < nblocks; ++r) c[q] += *cluster.map_shared_rank(&s_hist[bin], r);
        sum += c[q];
      }
      uint64_t total;
      uint64_t before = block_scan(sum, s_warp, total);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (before < (uint64_t)need && before + c[q] >= (uint64_t)need) {
          s_digit = bins - 1 - (4 * tid + q);
          s_need = need - (int)before;
        }
        before += c[q];
      }
      cluster.sync();  // the digit is known, every block has read the histograms
      prefix |= (uint32_t)s_digit << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need = s_need;
    }
    cut = prefix;
  }
  const int ties = need;                // of the rows equal to `cut`, the first `ties` stay

  // counts over this thread's consecutive rows, then over the block, then the cluster
  const int per = p.slice / kThreads;
  const int from = min(first + tid * per, last), to = min(from + per, last);
  uint32_t above = 0, equal = 0;
  for (int i = from; i < to; ++i) {
    if (i >= old) {
      ++above;
    } else {
      const uint32_t key = key_at(i);
      above += key > cut;
      equal += key == cut;
    }
  }
  uint64_t total;
  uint64_t before = block_scan((uint64_t)above << 32 | equal, s_warp, total);
  if (tid == 0) s_totals = total;
  cluster.sync();
  for (int r = 0; r < rank; ++r) before += *cluster.map_shared_rank(&s_totals, r);
  uint32_t a = (uint32_t)(before >> 32), e = (uint32_t)before;
  for (int i = from; i < to; ++i) {
    bool keep;
    const uint32_t slot = a + min((uint32_t)ties, e);
    if (i >= old) {
      keep = true;
      ++a;
    } else {
      const uint32_t key = key_at(i);
      keep = key > cut || (key == cut && e < (uint32_t)ties);
      a += key > cut;
      e += key == cut;
    }
    if (keep) {
      pos[slot] = i;
      w_out[slot] = __ldg(w + i);
    }
  }
  cluster.sync();  // no block leaves while another reads its shared memory
}

struct CopyParams {
  const uint16_t *k, *v;
  uint16_t *k_out, *v_out;
  const int32_t* positions;  // [B][H][N]
  int64_t rows;              // B * N * H
  int64_t k_seq, k_row, k_head, v_seq, v_row, v_head;
  int64_t ko_seq, ko_row, ko_head, vo_seq, vo_row, vo_head;
  int kv_heads, budget, hd;
};

__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// CP 16-byte pieces per row (rounded up to a power of two): 8 or 16: a warp step
// copies the K and V rows of 16 / CP output rows; 32: of one row, K then V.
template <int CP>
__global__ void __launch_bounds__(256) copy_rows_kernel(const CopyParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * 32;
  if (row0 >= p.rows) return;
  // this lane's output row: (sequence, slot, head) and the cache row it takes
  const int64_t mine = min(row0 + lane, p.rows - 1);
  const int64_t bs = mine / p.kv_heads;
  const int h = (int)(mine - bs * p.kv_heads);
  const int64_t b = bs / p.budget;
  const int slot = (int)(bs - b * p.budget);
  const int from = __ldg(p.positions + (b * p.kv_heads + h) * p.budget + slot);
  constexpr int kPer = CP >= 16 ? 1 : 16 / CP;   // output rows per step
  constexpr int kTensors = CP == 32 ? 2 : 1;     // loads per step and lane
  const int piece = lane % CP;
  const int sub = CP >= 16 ? 0 : lane / (2 * CP);
  const bool is_v = CP < 32 && ((lane / CP) & 1);
  const bool col_ok = piece * 8 < p.hd;
  const int steps = (int)((min((int64_t)32, p.rows - row0) + kPer - 1) / kPer);
  const bool one_seq = __all_sync(0xffffffffu, b == __shfl_sync(0xffffffffu, b, 0));
  constexpr int kUnroll = 8;
#pragma unroll 1
  for (int s0 = 0; s0 < steps; s0 += kUnroll) {
    uint4 x[kUnroll][kTensors];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = (s0 + u) * kPer + sub;
      const int src = __shfl_sync(0xffffffffu, from, r & 31), hh = __shfl_sync(0xffffffffu, h, r & 31);
      const int64_t bb = one_seq ? b : __shfl_sync(0xffffffffu, b, r & 31);
#pragma unroll
      for (int q = 0; q < kTensors; ++q) {
        x[u][q] = make_uint4(0u, 0u, 0u, 0u);
        const bool v = CP == 32 ? q == 1 : is_v;
        const uint16_t* at = v ? p.v + bb * p.v_seq + src * p.v_row + hh * p.v_head
                               : p.k + bb * p.k_seq + src * p.k_row + hh * p.k_head;
        if (r < 32 && row0 + r < p.rows && src >= 0 && col_ok) x[u][q] = load_once(at + piece * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = (s0 + u) * kPer + sub;
      const int to = __shfl_sync(0xffffffffu, slot, r & 31), hh = __shfl_sync(0xffffffffu, h, r & 31);
      const int64_t bb = one_seq ? b : __shfl_sync(0xffffffffu, b, r & 31);
#pragma unroll
      for (int q = 0; q < kTensors; ++q) {
        const bool v = CP == 32 ? q == 1 : is_v;
        uint16_t* at = v ? p.v_out + bb * p.vo_seq + to * p.vo_row + hh * p.vo_head
                         : p.k_out + bb * p.ko_seq + to * p.ko_row + hh * p.ko_head;
        if (r < 32 && row0 + r < p.rows && col_ok) *reinterpret_cast<uint4*>(at + piece * 8) = x[u][q];
      }
    }
  }
}

int launch_choose(const ChooseParams& p, int64_t caches, int cluster, int smem, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  TTJ_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (dev >= 64 || !(done.load(std::memory_order_acquire) & bit)) {
    TTJ_CUDA_TRY(cudaFuncSetAttribute(choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (kMaxStagedKeys + kMaxStagedKeys / 32) * 4));
    done.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(caches * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TTJ_CUDA_TRY(cudaLaunchKernelEx(&cfg, choose_kernel, p));
  return TTJ_OK;
}

}  // namespace

int launch_cache_evict(const ttj_cache_evict_args& a, cudaStream_t stream) {
  const int64_t caches = a.batch * a.num_kv_heads;
  ChooseParams c{};
  c.weights = a.key_weights;
  c.lengths = a.lengths;
  c.weights_out = a.weights_out;
  c.lengths_out = a.lengths_out;
  c.positions = a.positions_out;
  c.kv_heads = (int)a.num_kv_heads;
  c.capacity = (int)a.capacity;
  c.budget = (int)a.budget;
  c.recent = (int)a.recent;
  int cluster = 1;
  while (cluster < kMaxCluster && (int64_t)cluster * kSliceKeys < a.capacity) cluster *= 2;
  if (caches * cluster >= (int64_t)1 << 31) return fail(TTJ_ERR_UNSUPPORTED, "too many caches");
  const int64_t per_block = (a.capacity + cluster - 1) / cluster;
  c.slice = (int)(std::max<int64_t>(1, (per_block + kThreads - 1) / kThreads) * kThreads);
  c.staged = c.slice <= kMaxStagedKeys;
  const int smem = c.staged ? (c.slice + c.slice / 32) * 4 : 0;
  if (int rc = launch_choose(c, caches, cluster, smem, stream)) return rc;
  CopyParams p{};
  p.k = static_cast<const uint16_t*>(a.k_cache);
  p.v = static_cast<const uint16_t*>(a.v_cache);
  p.k_out = static_cast<uint16_t*>(a.k_out);
  p.v_out = static_cast<uint16_t*>(a.v_out);
  p.positions = a.positions_out;
  p.rows = caches * a.budget;
  p.k_seq = a.k_seq_stride, p.k_row = a.k_row_stride, p.k_head = a.k_head_stride;
  p.v_seq = a.v_seq_stride, p.v_row = a.v_row_stride, p.v_head = a.v_head_stride;
  p.ko_seq = a.k_out_seq_stride, p.ko_row = a.k_out_row_stride, p.ko_head = a.k_out_head_stride;
  p.vo_seq = a.v_out_seq_stride, p.vo_row = a.v_out_row_stride, p.vo_head = a.v_out_head_stride;
  p.kv_heads = c.kv_heads;
  p.budget = c.budget;
  p.hd = (int)a.head_dim;
  const int64_t blocks = (p.rows + 255) / 256;
  if (blocks >= (int64_t)1 << 31) return fail(TTJ_ERR_UNSUPPORTED, "too many cache rows");
  const dim3 grid((unsigned)blocks);
  if (p.hd <= 64) TTJ_CUDA_TRY(launch_pdl(copy_rows_kernel<8>, grid, dim3(256), 0, stream, p));
  else if (p.hd <= 128) TTJ_CUDA_TRY(launch_pdl(copy_rows_kernel<16>, grid, dim3(256), 0, stream, p));
  else TTJ_CUDA_TRY(launch_pdl(copy_rows_kernel<32>, grid, dim3(256), 0, stream, p));
  return TTJ_OK;
}

}  // namespace ttj
