// Causal attention over packed prompts of different lengths with grouped heads.
//
// One warp per (token, query head) row: the lanes hold eight of the row's
// dimensions each, a key's score is a warp sum, and the running maximum, sum and
// output follow the softmax recurrence key by key (one pass over the keys).
#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace ttj {
namespace {

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = Pack<T>::unpack(ws[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) prompt_rows_kernel(const ttj_prompt_attn_args a) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int hd = (int)a.head_dim;
  const int group = (int)(a.num_heads / a.num_kv_heads);
  const int64_t item = blockIdx.x;
  const int kvh = (int)(item % a.num_kv_heads);
  const PlanEntry e = reinterpret_cast<const PlanEntry*>(a.plan)[item / a.num_kv_heads];
  const bool live = lane * 8 < hd;
  const T* k = static_cast<const T*>(a.k) + e.k_row * a.k_token_stride + kvh * a.k_head_stride + lane * 8;
  const T* v = static_cast<const T*>(a.v) + e.k_row * a.v_token_stride + kvh * a.v_head_stride + lane * 8;
  for (int r = threadIdx.x >> 5; r < e.rows * group; r += blockDim.x >> 5) {
    const int64_t row = e.q_row + r / group;
    const int h = kvh * group + r % group;
    float q[8] = {}, o[8] = {}, x[8];
    if (live) load8<T>(static_cast<const T*>(a.q) + row * a.q_token_stride + h * a.q_head_stride + lane * 8, q);
    float m = -INFINITY, l = 0.f;
    for (int64_t u = 0; u <= row - e.k_row; ++u) {
      float s = 0.f;
      if (live) {
        load8<T>(k + u * a.k_token_stride, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(q[j], x[j], s);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= a.scale;
      const float mn = fmaxf(m, s);
      const float keep = m == -INFINITY ? 0.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
      l = l * keep + p;
      m = mn;
      if (live) {
        load8<T>(v + u * a.v_token_stride, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = fmaf(p, x[j], o[j] * keep);
      }
    }
    const float inv = 1.f / l;
    if (live) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = Pack<T>::two(o[2 * j] * inv, o[2 * j + 1] * inv);
      *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (row * a.num_heads + h) * hd + lane * 8) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (a.lse != nullptr && lane == 0) a.lse[row * a.num_heads + h] = m + logf(l);
  }
}

}  // namespace

int launch_prompt_attn(const ttj_prompt_attn_args& a, cudaStream_t stream) {
  const dim3 grid((unsigned)(a.plan_entries * a.num_kv_heads));
  if (a.dtype == TTJ_F16) TTJ_CUDA_TRY(launch_pdl(prompt_rows_kernel<__half>, grid, dim3(256), 0, stream, a));
  else TTJ_CUDA_TRY(launch_pdl(prompt_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, a));
  return TTJ_OK;
}

}  // namespace ttj
