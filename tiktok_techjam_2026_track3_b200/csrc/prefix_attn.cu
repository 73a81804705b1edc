// One decode step over a prefix shared by the batch and each sequence's own
// cache, with grouped heads and, on request, the step's attention weights added
// to each cached key's running sum.
//
// One warp per (sequence, query head): the softmax recurrence over the prefix
// rows, then the cache rows.  The weights follow in a second pass over the
// cache with each row's maximum and sum.
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

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  return s;
}

template <typename T>
__global__ void __launch_bounds__(128) decode_rows_kernel(const ttj_shared_prefix_attn_args a) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int hd = (int)a.head_dim;
  const int group = (int)(a.num_heads / a.num_kv_heads);
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= a.batch * a.num_heads) return;
  const int64_t b = r / a.num_heads;
  const int h = (int)(r % a.num_heads), kvh = h / group;
  const bool live = lane * 8 < hd;
  float q[8] = {}, o[8] = {}, x[8];
  if (live) load8<T>(static_cast<const T*>(a.q) + b * a.q_seq_stride + h * a.q_head_stride + lane * 8, q);
  float m = -INFINITY, l = 0.f;
  const int64_t n = min((int64_t)max(a.lengths[b], 0), a.capacity);
  for (int64_t u = 0; u < a.prefix_len + n; ++u) {
    const int64_t c = u - a.prefix_len;
    const T* k = c < 0 ? static_cast<const T*>(a.prefix_k) + u * a.prefix_k_row_stride + kvh * a.prefix_k_head_stride
                       : static_cast<const T*>(a.k_cache) + b * a.k_seq_stride + c * a.k_row_stride + kvh * a.k_head_stride;
    const T* v = c < 0 ? static_cast<const T*>(a.prefix_v) + u * a.prefix_v_row_stride + kvh * a.prefix_v_head_stride
                       : static_cast<const T*>(a.v_cache) + b * a.v_seq_stride + c * a.v_row_stride + kvh * a.v_head_stride;
    float s = 0.f;
    if (live) {
      load8<T>(k + lane * 8, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(q[j], x[j], s);
    }
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
    l = l * keep + p;
    m = mn;
    if (live) {
      load8<T>(v + lane * 8, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(p, x[j], o[j] * keep);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (live) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = Pack<T>::two(o[2 * j] * inv, o[2 * j + 1] * inv);
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + r * hd + lane * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (a.key_weights != nullptr && lane == 0) static_cast<float*>(a.workspace)[r] = l > 0.f ? m + logf(l) : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256) key_weights_kernel(const ttj_shared_prefix_attn_args a) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int group = (int)(a.num_heads / a.num_kv_heads);
  const int64_t b = blockIdx.x / a.num_kv_heads;
  const int kvh = (int)(blockIdx.x % a.num_kv_heads);
  const bool live = lane * 8 < (int)a.head_dim;
  const float* lse = static_cast<const float*>(a.workspace) + b * a.num_heads + kvh * group;
  const int64_t n = min((int64_t)max(a.lengths[b], 0), a.capacity);
  for (int64_t c = threadIdx.x >> 5; c < a.capacity; c += 8) {
    const int64_t at = (b * a.num_kv_heads + kvh) * a.capacity + c;
    float sum = 0.f;
    if (c < n) {
      float x[8] = {}, q[8];
      if (live)
        load8<T>(static_cast<const T*>(a.k_cache) + b * a.k_seq_stride + c * a.k_row_stride + kvh * a.k_head_stride +
                     lane * 8, x);
      for (int i = 0; i < group; ++i) {
        float s = 0.f;
        if (live) {
          load8<T>(static_cast<const T*>(a.q) + b * a.q_seq_stride + (kvh * group + i) * a.q_head_stride + lane * 8, q);
#pragma unroll
          for (int j = 0; j < 8; ++j) s = fmaf(q[j], x[j], s);
        }
        sum += expf(warp_sum(s) * a.scale - lse[i]);
      }
    }
    if (lane == 0) a.key_weights_out[at] = c < n ? a.key_weights[at] + sum : a.key_weights[at];
  }
}

template <typename T>
int launch_decode(const ttj_shared_prefix_attn_args& a, cudaStream_t stream) {
  const int64_t rows = a.batch * a.num_heads;
  TTJ_CUDA_TRY(launch_pdl(decode_rows_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, a));
  if (a.key_weights != nullptr && a.capacity > 0)
    TTJ_CUDA_TRY(launch_pdl(key_weights_kernel<T>, dim3((unsigned)(a.batch * a.num_kv_heads)), dim3(256), 0, stream, a));
  return TTJ_OK;
}

}  // namespace

size_t shared_prefix_attn_workspace(int64_t batch, int64_t, int64_t, int64_t num_heads, int64_t, int64_t,
                                    bool with_key_weights) {
  return with_key_weights ? (size_t)batch * num_heads * sizeof(float) : 0;
}

int launch_shared_prefix_attn(const ttj_shared_prefix_attn_args& a, cudaStream_t stream) {
  return a.dtype == TTJ_F16 ? launch_decode<__half>(a, stream) : launch_decode<__nv_bfloat16>(a, stream);
}

}  // namespace ttj
