// Eviction from per-sequence caches by accumulated attention weight.
//
// One block per (sequence, key / value head).  Weights compare as 32-bit
// unsigned keys in the order of their values; the block finds the key of the
// last row to keep by bisection on its 32 bits (one count over the candidates
// per bit), then walks the rows in order, keeps those above it and the first few
// equal to it, and copies each kept row to the next free slot.
#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace ttj {
namespace {

constexpr int kThreads = 256;

// Ascending unsigned order of the weights; NaN as -infinity, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int block_sum(int v, int* shared) {
  __syncthreads();  // all threads have read the previous result
  if (threadIdx.x == 0) *shared = 0;
  __syncthreads();
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
  if ((threadIdx.x & 31) == 0) atomicAdd(shared, v);
  __syncthreads();
  return *shared;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(const ttj_cache_evict_args a) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ int s_sum, s_warp[2][kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.x / a.num_kv_heads;
  const int h = (int)(blockIdx.x % a.num_kv_heads);
  const int64_t bh = blockIdx.x;
  const int n = (int)min((int64_t)max(a.lengths[b], 0), a.capacity);
  const int budget = (int)a.budget, kept = min(n, budget);
  const float* w = a.key_weights + bh * a.capacity;
  const int old = n - min(n, (int)a.recent);       // rows below `old` compete
  int need = budget - (int)a.recent;               // rows of them to keep
  uint32_t cut = 0;                                // key of the last row kept
  int ties = 0;                                    // rows equal to it that are kept
  if (n > budget && need > 0) {
    for (int bit = 31; bit >= 0; --bit) {          // largest cut with at least `need` keys >= cut
      const uint32_t t = cut | (1u << bit);
      int c = 0;
      for (int i = tid; i < old; i += kThreads) c += weight_key(w[i]) >= t;
      if (block_sum(c, &s_sum) >= need) cut = t;
    }
    int c = 0;
    for (int i = tid; i < old; i += kThreads) c += weight_key(w[i]) > cut;
    ties = need - block_sum(c, &s_sum);
  }
  const int words = (int)a.head_dim / 8;
  auto copy_row = [&](int64_t to, int64_t from) {
    const uint16_t* ks = static_cast<const uint16_t*>(a.k_cache) + b * a.k_seq_stride + from * a.k_row_stride + h * a.k_head_stride;
    const uint16_t* vs = static_cast<const uint16_t*>(a.v_cache) + b * a.v_seq_stride + from * a.v_row_stride + h * a.v_head_stride;
    uint16_t* kd = static_cast<uint16_t*>(a.k_out) + b * a.k_out_seq_stride + to * a.k_out_row_stride + h * a.k_out_head_stride;
    uint16_t* vd = static_cast<uint16_t*>(a.v_out) + b * a.v_out_seq_stride + to * a.v_out_row_stride + h * a.v_out_head_stride;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int i = 0; i < words; ++i) {
      reinterpret_cast<uint4*>(kd)[i] = from >= 0 ? reinterpret_cast<const uint4*>(ks)[i] : zero;
      reinterpret_cast<uint4*>(vd)[i] = from >= 0 ? reinterpret_cast<const uint4*>(vs)[i] : zero;
    }
    a.weights_out[bh * a.budget + to] = from >= 0 ? w[from] : 0.f;
    a.positions_out[bh * a.budget + to] = (int32_t)from;
  };
  int slot0 = 0, tie0 = 0;                         // rows kept, and equal rows seen, before this chunk
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + tid;
    bool above = false, equal = false;
    if (i < n) {
      if (n <= budget || i >= old) {
        above = true;
      } else if (need > 0) {
        const uint32_t key = weight_key(w[i]);
        above = key > cut;
        equal = key == cut;
      }
    }
    const uint32_t eq = __ballot_sync(0xffffffffu, equal);
    if (lane == 0) s_warp[0][warp] = __popc(eq);
    __syncthreads();
    int before = tie0 + __popc(eq & ((1u << lane) - 1));
    for (int j = 0; j < kThreads / 32; ++j) {
      if (j < warp) before += s_warp[0][j];
      tie0 += s_warp[0][j];
    }
    const bool keep = above || (equal && before < ties);
    const uint32_t kp = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) s_warp[1][warp] = __popc(kp);
    __syncthreads();
    int slot = slot0 + __popc(kp & ((1u << lane) - 1));
    for (int j = 0; j < kThreads / 32; ++j) {
      if (j < warp) slot += s_warp[1][j];
      slot0 += s_warp[1][j];
    }
    if (keep) copy_row(slot, i);
  }
  for (int i = kept + tid; i < budget; i += kThreads) copy_row(i, -1);
  if (h == 0 && tid == 0) a.lengths_out[b] = kept;
}

}  // namespace

int launch_cache_evict(const ttj_cache_evict_args& a, cudaStream_t stream) {
  TTJ_CUDA_TRY(launch_pdl(evict_kernel, dim3((unsigned)(a.batch * a.num_kv_heads)), dim3(kThreads), 0, stream, a));
  return TTJ_OK;
}

}  // namespace ttj
