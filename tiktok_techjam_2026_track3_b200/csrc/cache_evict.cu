// Eviction from per-sequence caches by accumulated attention weight, two kernels (one
// when few rows are kept).
//
// 1. Choosing (weights read once, 4 bytes a row): one cluster of blocks per
//    (sequence, key / value head), each warp a stretch of consecutive rows.  A weight
//    compares as a 32-bit unsigned key in the order of its value, held in registers.
//    The key `cut` of the last row to keep (the need-th largest) is looked for in the
//    range of the positive keys (or at zero, or below), cut to a quarter at a time:
//    every warp counts its keys at or above the three candidates and the counts are
//    summed over the cluster (one barrier).  Once at most kList keys remain in the
//    range, those alone are collected (in any order: only their values count) and
//    every block searches on in a copy.  The search ends as soon as a candidate has
//    exactly `need` keys.  With `ties` the rows equal to the cut that stay, row i's
//    slot is
//        above(i) + min(ties, equal(i)),
//    above / equal counting the earlier rows with a larger / an equal key: equal rows
//    are kept lowest index first by construction.
//    Bound by instruction issue and barriers: a counting pass takes ~1300 cycles to
//    count, ~900 in the cluster barrier and ~700 to sum.  Weights written from their
//    keys instead of read again saved 8.6 us of 89 for 32 caches of 65537 rows cut to
//    8192; a start at the positive range (against all 32 bits) and a list and totals
//    without ballots 4.7 of 80 there and 4.6 of 195 for 512 of up to 4096 cut to 2048.
//    (Digit histograms in shared memory took 33 us for those 512 and 81 us for the 32
//    where the first version of this took 25 and 40; blocks of 256 threads with a
//    one-warp or an all-pairs end of the search, and a fourth resident block, measured
//    0 to 5% slower.)
// 2. Copying (bound by the kept rows' bytes): a warp takes 32 output rows in the
//    order of the output's memory and copies K and V rows in 16-byte pieces, eight
//    rows in flight: 173 us for 64 caches cut to 2048 rows of 8 heads of 128, 6.2
//    TB/s of the 6.45 of a plain copy.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace cg = cooperative_groups;

namespace ttj {
namespace {

constexpr int kThreads = 512;
constexpr int kWarpsPerBlock = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxKeysPerThread = 20;    // held in registers; longer slices are re-read
// rows per block that a cluster is sized for: what a block holds in registers (4096: 3%
// slower for caches of 16384 rows, 9% of 10000, 22% of 40000; 2048: 29% for 16384)
constexpr int kBlockKeys = kThreads * kMaxKeysPerThread;
// Kept rows of up to this many bytes per block are copied by the choosing blocks, which
// saves a launch (2 caches of 256 rows cut to 128, 4 heads of 64: 8.2 us against 12.3;
// 64 of 1000 cut to 128, 8 heads of 128, the size where it ends: 28.6 against 32.8,
// cut to 256: 43.0 against 39.0).
constexpr int64_t kCopyBytes = 65536;
constexpr int kList = 2 * kThreads;      // keys that the search ends on
static_assert(32 * kMaxKeysPerThread < 1024, "a warp's three counts share one word");

struct ChooseParams {
  const float* weights;   // [B][H][C]
  const int32_t* lengths;
  float* weights_out;     // [B][H][N]
  int32_t* lengths_out;
  int32_t* positions;     // [B][H][N]
  int kv_heads, capacity, budget, recent;
  int per;                // rows per thread
};

// Ascending unsigned order of the weights; NaN as -infinity, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// The bits of the weight with this key, or false where several have it (NaN and
// -infinity, the two zeros).
__device__ __forceinline__ bool weight_of(uint32_t key, float* w) {
  *w = __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
  return key != 0x007fffffu && key != 0x80000000u;
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// State of the search: `need` keys are to be kept, `at` keys are >= lo, `above` of
// them >= lo + span, above < need <= at.
struct Cut {
  uint32_t lo, span;
  int at, above;
  __device__ __forceinline__ uint32_t step() const { return (span + 3) >> 2; }
  // n1, n2, n3 keys are >= lo + step, lo + 2 step, lo + 3 step
  __device__ __forceinline__ void take(int n1, int n2, int n3, int need) {
    const uint32_t s = step();
    if (n3 >= need) at = n3, lo += 3 * s, span -= 3 * s;
    else if (n2 >= need) at = n2, lo += 2 * s, span = s, above = n3;
    else if (n1 >= need) at = n1, lo += s, span = s, above = n2;
    else span = s, above = n1;
  }
};

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

// KPT: upper bound on rows per thread, held in registers; 0: any number, read from
// memory each time.  COPY: the blocks copy the kept rows of K and V, too.
template <int KPT, bool COPY>
__global__ void __launch_bounds__(kThreads, KPT == 0 || KPT > 8 ? 2 : (KPT <= 2 && !COPY ? 4 : 3)) choose_kernel(const ChooseParams p, const CopyParams rows) {
  // Every warp of the cluster leaves its counts with every block: [parity][block, warp].
  __shared__ uint32_t s_count[2][3][kMaxCluster * kWarpsPerBlock];
  __shared__ uint64_t s_total[kMaxCluster * kWarpsPerBlock];
  __shared__ uint4 s_first[kWarpsPerBlock];
  __shared__ uint32_t s_list[kList];
  __shared__ int s_listed;
  cg::cluster_group cluster = cg::this_cluster();
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), nblocks = (int)cluster.num_blocks();
  const int nwarps = nblocks * kWarpsPerBlock, my_warp = rank * kWarpsPerBlock + warp;
  const int64_t bh = blockIdx.x / nblocks;
  const int64_t b = bh / p.kv_heads;
  const int n = min(max(__ldg(p.lengths + b), 0), p.capacity);
  const int kept = min(n, p.budget);
  const float* w = p.weights + bh * p.capacity;
  float* w_out = p.weights_out + bh * p.budget;
  int32_t* pos = p.positions + bh * p.budget;
  if (rank == 0 && tid == 0 && bh - b * p.kv_heads == 0) p.lengths_out[b] = kept;
  // output rows past the kept ones
  for (int i = kept + rank * kThreads + tid; i < p.budget; i += nblocks * kThreads) {
    w_out[i] = 0.f;
    pos[i] = -1;
  }
  auto sync_all = [&]() {
    if (nblocks > 1) cluster.sync();
    else __syncthreads();
  };
  // The rows themselves, when there are few: a share of the slots per block.
  auto copy_rows = [&]() {
    if constexpr (!COPY) return;
    sync_all();                              // the positions are written
    const int shift = rows.hd <= 64 ? 3 : (rows.hd <= 128 ? 4 : 5);  // 16-byte pieces per row, rounded up
    const int share = (p.budget + nblocks - 1) / nblocks, slot0 = rank * share;
    const int total = max(min(share, p.budget - slot0), 0) << (shift + 1);
    const int h = (int)(bh - b * p.kv_heads);
    const uint16_t *k_in = rows.k + b * rows.k_seq + h * rows.k_head, *v_in = rows.v + b * rows.v_seq + h * rows.v_head;
    uint16_t *k_to = rows.k_out + b * rows.ko_seq + h * rows.ko_head, *v_to = rows.v_out + b * rows.vo_seq + h * rows.vo_head;
    constexpr int kUnroll = 4;
    for (int u0 = tid; u0 < total; u0 += kUnroll * kThreads) {
      uint4 x[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int u = u0 + q * kThreads, piece = u & ((1 << shift) - 1);
        x[q] = make_uint4(0u, 0u, 0u, 0u);
        if (u >= total || piece * 8 >= rows.hd) continue;
        const int64_t src = __ldcg(pos + slot0 + (u >> (shift + 1)));
        const uint16_t* at = (u >> shift) & 1 ? v_in + src * rows.v_row : k_in + src * rows.k_row;
        if (src >= 0) x[q] = load_once(at + piece * 8);
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int u = u0 + q * kThreads, piece = u & ((1 << shift) - 1);
        if (u >= total || piece * 8 >= rows.hd) continue;
        const int64_t to = slot0 + (u >> (shift + 1));
        uint16_t* at = (u >> shift) & 1 ? v_to + to * rows.vo_row : k_to + to * rows.ko_row;
        *reinterpret_cast<uint4*>(at + piece * 8) = x[q];
      }
    }
  };
  if (n <= p.budget) {  // uniform over the cluster
    for (int i = rank * kThreads + tid; i < n; i += nblocks * kThreads) {
      w_out[i] = w[i];
      pos[i] = i;
    }
    copy_rows();
    return;
  }
  const int old = n - p.recent;              // rows below `old` compete
  const int need = p.budget - p.recent;      // for this many places
  // the recent rows take the last slots
  for (int i = rank * kThreads + tid; i < p.recent; i += nblocks * kThreads) {
    w_out[need + i] = __ldg(w + old + i);
    pos[need + i] = old + i;
  }
  const int64_t first = (int64_t)my_warp * 32 * p.per + lane;  // rows first + 32 j
  uint32_t key[KPT > 0 ? KPT : 1];           // 0: a row that does not compete
  auto key_of = [&](int j) -> uint32_t {
    const int64_t i = first + 32 * j;
    return i < old ? weight_key(__ldg(w + i)) : 0u;
  };
  if constexpr (KPT > 0) {
#pragma unroll
    for (int j = 0; j < KPT; ++j) key[j] = j < p.per ? key_of(j) : 0u;
  }
  // f(j, key) for this thread's rows, in order (a few keys of 0 at the end)
  auto each = [&](auto&& f) {
    if constexpr (KPT > 0) {
      constexpr int kGroup = KPT < 4 ? KPT : 4;
#pragma unroll
      for (int j0 = 0; j0 < KPT; j0 += kGroup)
        if (j0 < p.per) {
#pragma unroll
          for (int j = j0; j < j0 + kGroup; ++j) f(j, key[j]);
        }
    } else {
      for (int j = 0; j < p.per; ++j) f(j, key_of(j));
    }
  };
  constexpr uint32_t kZero = 0x80000000u, kLowest = 0x007fffffu;  // keys of 0 and of -infinity
  uint32_t top = 0u, low = 0xffffffffu, positive = 0u, nonnegative = 0u;
  each([&](int, uint32_t k) {
    top = max(top, k);
    low = min(low, k > kZero ? k : 0xffffffffu);
    positive += k > kZero;
    nonnegative += k >= kZero;
  });
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  positive = __reduce_add_sync(0xffffffffu, positive);
  nonnegative = __reduce_add_sync(0xffffffffu, nonnegative);
  if (lane == 0) s_first[warp] = make_uint4(top, low, positive, nonnegative);
  if (tid == 0) s_listed = 0;
  sync_all();                                // every block runs: its shared memory may be used

  uint32_t cut = 0xffffffffu;                // need == 0: nothing competes
  int ties = 0;
  if (need > 0) {
    // Where the search starts: the positive weights' range, the zeros (which caches of
    // rows that nothing attends hold in number), or all that is negative.
    top = positive = nonnegative = 0u, low = 0xffffffffu;
    for (int i = lane; i < nwarps; i += 32) {
      const uint4 v = *cluster.map_shared_rank(&s_first[i % kWarpsPerBlock], i / kWarpsPerBlock);
      top = max(top, v.x);
      low = min(low, v.y);
      positive += v.z;
      nonnegative += v.w;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    const int n_positive = (int)__reduce_add_sync(0xffffffffu, positive);
    const int n_nonnegative = (int)__reduce_add_sync(0xffffffffu, nonnegative);
    Cut x = n_positive >= need      ? Cut{low, top - low + 1u, n_positive, 0}
            : n_nonnegative >= need ? Cut{kZero, 1u, n_nonnegative, n_positive}
                                    : Cut{kLowest, kZero - kLowest, old, n_nonnegative};
    int parity = 0;
#pragma unroll 1
    while (x.span > 1u && x.at != need && x.at - x.above > kList) {
      const uint32_t t1 = x.lo + x.step(), t2 = t1 + x.step(), t3 = t2 + x.step();
      uint32_t c1 = 0, c2 = 0, c3 = 0;
      each([&](int, uint32_t k) {            // (keys of 0 are below every candidate)
        c1 += k >= t1;
        c2 += k >= t2;
        c3 += k >= t3;
      });
      if constexpr (KPT > 0) {
        // a warp's three counts share one word
        c1 = __reduce_add_sync(0xffffffffu, c1 | c2 << 10 | c3 << 20);
        if (lane < nblocks) *cluster.map_shared_rank(&s_count[parity][0][my_warp], lane) = c1;
      } else {
        c1 = __reduce_add_sync(0xffffffffu, c1);
        c2 = __reduce_add_sync(0xffffffffu, c2);
        c3 = __reduce_add_sync(0xffffffffu, c3);
        if (lane < nblocks) {
          *cluster.map_shared_rank(&s_count[parity][0][my_warp], lane) = c1;
          *cluster.map_shared_rank(&s_count[parity][1][my_warp], lane) = c2;
          *cluster.map_shared_rank(&s_count[parity][2][my_warp], lane) = c3;
        }
      }
      sync_all();
      c1 = c2 = c3 = 0;
      for (int i = lane; i < nwarps; i += 32) {
        const uint32_t v = s_count[parity][0][i];
        c1 += KPT > 0 ? v & 1023u : v;
        c2 += KPT > 0 ? (v >> 10) & 1023u : s_count[parity][1][i];
        c3 += KPT > 0 ? v >> 20 : s_count[parity][2][i];
      }
      x.take((int)__reduce_add_sync(0xffffffffu, c1), (int)__reduce_add_sync(0xffffffffu, c2),
             (int)__reduce_add_sync(0xffffffffu, c3), need);
      parity ^= 1;
    }
    if (x.span > 1u && x.at != need) {
      // the keys in [lo, lo + span), collected by the first block
      uint32_t* list = cluster.map_shared_rank(s_list, 0);
      int* listed = cluster.map_shared_rank(&s_listed, 0);
      int mine = 0;
      each([&](int, uint32_t k) { mine += k - x.lo < x.span; });
      int at = mine;                         // of this warp's lanes up to this one, then of those before it
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += v;
      }
      int base = 0;
      if (lane == 31 && at > 0) base = atomicAdd(listed, at);
      at += __shfl_sync(0xffffffffu, base, 31) - mine;
      each([&](int, uint32_t k) {
        if (k - x.lo < x.span) list[at++] = k;
      });
      sync_all();
      const int count = x.at - x.above;
      const uint32_t k0 = tid < count ? list[tid] : 0u, k1 = tid + kThreads < count ? list[tid + kThreads] : 0u;
      const int outside = x.above;           // keys above every listed one
#pragma unroll 1
      do {
        const uint32_t t1 = x.lo + x.step(), t2 = t1 + x.step(), t3 = t2 + x.step();
        uint32_t c = ((k0 >= t1) + (k1 >= t1)) | ((k0 >= t2) + (k1 >= t2)) << 10 | ((k0 >= t3) + (k1 >= t3)) << 20;
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) s_count[parity][0][warp] = c;
        __syncthreads();
        c = lane < kWarpsPerBlock ? s_count[parity][0][lane] : 0u;
        // at most 64 keys a warp, 1024 a block: two counts to a word
        const uint32_t lo = __reduce_add_sync(0xffffffffu, (c & 1023u) | ((c >> 10) & 1023u) << 16);
        const uint32_t hi = __reduce_add_sync(0xffffffffu, c >> 20);
        x.take(outside + (int)(lo & 0xffffu), outside + (int)(lo >> 16), outside + (int)hi, need);
        parity ^= 1;
      } while (x.span > 1u && x.at != need);
    }
    if (x.at == need) cut = x.lo - 1u;       // exactly the keys >= lo stay
    else cut = x.lo, ties = need - x.above;  // the key is found: rows equal to it fill up
  }

  // This warp's rows above and equal to the cut, then those of the warps before it.
  uint32_t a = 0, e = 0;
  each([&](int, uint32_t k) {
    a += k > cut;
    e += k == cut;
  });
  a = __reduce_add_sync(0xffffffffu, a);
  e = __reduce_add_sync(0xffffffffu, e);
  if (lane < nblocks) *cluster.map_shared_rank(&s_total[my_warp], lane) = (uint64_t)a << 32 | e;
  sync_all();                                // (also: no block leaves while its list is read)
  uint64_t before = 0;
  for (int i = lane; i < my_warp; i += 32) before += s_total[i];
  before = warp_sum(before);
  a = (uint32_t)(before >> 32);
  e = (uint32_t)before;
  const uint32_t lower = (1u << lane) - 1u;
  auto put = [&](int j, uint32_t k, uint32_t slot) {
    const int i = (int)first + 32 * j;
    float v;                                 // a load here would hold up the warp at every row
    if (!weight_of(k, &v)) v = __ldg(w + i);
    pos[slot] = i;
    w_out[slot] = v;
  };
  if (ties == 0) {                           // uniform over the cluster
    each([&](int j, uint32_t k) {
      const uint32_t ab = __ballot_sync(0xffffffffu, k > cut);
      if (k > cut) put(j, k, a + __popc(ab & lower));
      a += __popc(ab);
    });
  } else {
    each([&](int j, uint32_t k) {
      const bool above = k > cut, equal = k == cut;
      const uint32_t ab = __ballot_sync(0xffffffffu, above), eb = __ballot_sync(0xffffffffu, equal);
      const uint32_t e_before = e + __popc(eb & lower);
      if (above || (equal && e_before < (uint32_t)ties)) put(j, k, a + __popc(ab & lower) + min((uint32_t)ties, e_before));
      a += __popc(ab);
      e += __popc(eb);
    });
  }
  copy_rows();
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

template <int KPT, bool COPY>
int launch_choose(const ChooseParams& p, const CopyParams& rows, int64_t caches, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(caches * cluster));
  cfg.blockDim = dim3(kThreads);
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
  TTJ_CUDA_TRY(cudaLaunchKernelEx(&cfg, choose_kernel<KPT, COPY>, p, rows));
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
  while (cluster < kMaxCluster && (int64_t)cluster * kBlockKeys < a.capacity) cluster *= 2;
  // Few caches get larger clusters where their blocks can then copy the rows (one of 8
  // heads of 128 cut to 512 of 1000 rows: 13.7 us against 18.5).
  const int64_t kept_bytes = a.head_dim * a.budget * 4;
  int wide = cluster;
  while (wide < kMaxCluster && kept_bytes > wide * kCopyBytes && caches * wide <= sm_count()) wide *= 2;
  const bool copy = kept_bytes <= wide * kCopyBytes;
  if (copy) cluster = wide;
  if (caches * cluster >= (int64_t)1 << 31) return fail(TTJ_ERR_UNSUPPORTED, "too many caches");
  const int64_t threads = (int64_t)cluster * kThreads;
  c.per = (int)std::max<int64_t>(1, (a.capacity + threads - 1) / threads);
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
  auto choose = [&](auto kpt) {
    constexpr int n = decltype(kpt)::value;
    return copy ? launch_choose<n, true>(c, p, caches, cluster, stream)
                : launch_choose<n, false>(c, p, caches, cluster, stream);
  };
  const int rc = c.per <= 2                   ? choose(std::integral_constant<int, 2>())
                 : c.per <= 8                 ? choose(std::integral_constant<int, 8>())
                 : c.per <= kMaxKeysPerThread ? choose(std::integral_constant<int, kMaxKeysPerThread>())
                                              : choose(std::integral_constant<int, 0>());
  if (rc || copy) return rc;
  const int64_t blocks = (p.rows + 255) / 256;
  if (blocks >= (int64_t)1 << 31) return fail(TTJ_ERR_UNSUPPORTED, "too many cache rows");
  const dim3 grid((unsigned)blocks);
  if (p.hd <= 64) TTJ_CUDA_TRY(launch_pdl(copy_rows_kernel<8>, grid, dim3(256), 0, stream, p));
  else if (p.hd <= 128) TTJ_CUDA_TRY(launch_pdl(copy_rows_kernel<16>, grid, dim3(256), 0, stream, p));
  else TTJ_CUDA_TRY(launch_pdl(copy_rows_kernel<32>, grid, dim3(256), 0, stream, p));
  return TTJ_OK;
}

}  // namespace ttj
