// extern "C" entry points of the serving operators (declared in
// include/ttj_attn.h): argument validation and the host-built prompt plan.  No
// entry point allocates, synchronises or throws.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <utility>

#include "ttj_internal.h"

using ttj::aligned16;
using ttj::check_dtype;
using ttj::fail;

namespace {

constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 1;      // tokens, batch
constexpr int64_t kMaxCache = (int64_t)1 << 30;           // prefix rows, cache rows
constexpr int64_t kMaxExtent = (int64_t)1 << 46;          // elements a stride may span
constexpr int64_t kMaxStride = ((int64_t)1 << 38) - 1;    // elements (tensor maps: bytes below 2^40)

int check_heads(int64_t num_heads, int64_t num_kv_heads, int64_t head_dim) {
  if (num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0)
    return fail(TTJ_ERR_INVALID_ARG, "num_heads, num_kv_heads and head_dim must be positive");
  if (num_heads > ttj::kMaxDModel) return fail(TTJ_ERR_UNSUPPORTED, "num_heads above the supported maximum");
  if (num_heads % num_kv_heads != 0)
    return fail(TTJ_ERR_INVALID_ARG, "num_heads must be a multiple of num_kv_heads");
  if (num_heads / num_kv_heads > ttj::kMaxGroup)
    return fail(TTJ_ERR_UNSUPPORTED, "at most 128 query heads per key / value head");
  if (head_dim % 8 != 0 || head_dim > 256)
    return fail(TTJ_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 256");
  return TTJ_OK;
}

// A strided dimension: `size` steps of `stride` elements, 16-byte multiples.
bool stride_ok(int64_t size, int64_t stride) {
  return stride > 0 && stride % 8 == 0 && stride <= kMaxStride && (size <= 1 || size - 1 <= kMaxExtent / stride);
}

int check_strides(const char* what, std::initializer_list<std::pair<int64_t, int64_t>> dims) {
  for (const auto& d : dims)
    if (!stride_ok(d.first, d.second))
      return fail(TTJ_ERR_UNSUPPORTED, std::string(what) + " strides must be positive multiples of 8 elements");
  return TTJ_OK;
}

int check_plan_args(const int64_t* seq_lens, int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads,
                    int64_t head_dim) {
  if (int rc = check_heads(num_heads, num_kv_heads, head_dim)) return rc;
  TTJ_CHECK_ARG(num_seqs >= 0 && (num_seqs == 0 || seq_lens != nullptr), TTJ_ERR_INVALID_ARG,
                "seq_lens must hold num_seqs lengths");
  int64_t total = 0;
  for (int64_t i = 0; i < num_seqs; ++i) {
    TTJ_CHECK_ARG(seq_lens[i] >= 0, TTJ_ERR_INVALID_ARG, "prompt lengths must not be negative");
    TTJ_CHECK_ARG(seq_lens[i] <= ttj::kMaxSeqLen, TTJ_ERR_UNSUPPORTED, "prompt above the supported length");
    total += seq_lens[i];
    TTJ_CHECK_ARG(total <= kMaxRows, TTJ_ERR_UNSUPPORTED, "more than 2^31 - 1 packed tokens");
  }
  return TTJ_OK;
}

// Byte ranges of two strided tensors intersect (a conservative test on their hulls).
struct Span {
  uintptr_t lo, hi;
};
Span span_of(const void* p, int64_t elem_bytes, int64_t inner, std::initializer_list<std::pair<int64_t, int64_t>> dims) {
  int64_t last = inner;
  for (const auto& d : dims) last += (d.first - 1) * d.second;
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, lo + (uintptr_t)(last * elem_bytes)};
}
bool overlap(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }

}  // namespace

extern "C" {

int64_t ttj_prompt_plan_entries(const int64_t* seq_lens, int64_t num_seqs, int64_t num_heads,
                                int64_t num_kv_heads, int64_t head_dim) {
  if (int rc = check_plan_args(seq_lens, num_seqs, num_heads, num_kv_heads, head_dim)) return rc;
  const int64_t step = ttj::plan_positions(num_heads / num_kv_heads, head_dim);
  int64_t n = 0;
  for (int64_t i = 0; i < num_seqs; ++i) n += (seq_lens[i] + step - 1) / step;
  return n;
}

int ttj_prompt_plan_build(const int64_t* seq_lens, int64_t num_seqs, int64_t num_heads, int64_t num_kv_heads,
                          int64_t head_dim, int32_t* plan, int64_t plan_entries) {
  const int64_t need = ttj_prompt_plan_entries(seq_lens, num_seqs, num_heads, num_kv_heads, head_dim);
  if (need < 0) return (int)need;
  TTJ_CHECK_ARG(plan_entries == need, TTJ_ERR_INVALID_ARG, "plan_entries must be ttj_prompt_plan_entries()");
  TTJ_CHECK_ARG(need == 0 || plan != nullptr, TTJ_ERR_INVALID_ARG, "plan is NULL");
  const int64_t step = ttj::plan_positions(num_heads / num_kv_heads, head_dim);
  ttj::PlanEntry* e = reinterpret_cast<ttj::PlanEntry*>(plan);
  int64_t n = 0, first = 0;
  for (int64_t i = 0; i < num_seqs; ++i) {
    for (int64_t p = 0; p < seq_lens[i]; p += step)
      e[n++] = {(int32_t)(first + p), (int32_t)std::min(step, seq_lens[i] - p), (int32_t)first, 0};
    first += seq_lens[i];
  }
  // Longest key range first, so that the work dealt out last is the shortest.
  std::sort(e, e + n, [](const ttj::PlanEntry& a, const ttj::PlanEntry& b) {
    const int32_t ka = a.q_row + a.rows - a.k_row, kb = b.q_row + b.rows - b.k_row;
    return ka != kb ? ka > kb : a.q_row < b.q_row;
  });
  return TTJ_OK;
}

int ttj_prompt_attn_fwd(const ttj_prompt_attn_args* a, ttj_stream_t stream) {
  TTJ_CHECK_ARG(a != nullptr, TTJ_ERR_INVALID_ARG, "args is NULL");
  if (int rc = check_dtype(a->dtype)) return rc;
  if (int rc = check_heads(a->num_heads, a->num_kv_heads, a->head_dim)) return rc;
  TTJ_CHECK_ARG(a->tokens >= 0 && a->plan_entries >= 0, TTJ_ERR_INVALID_ARG,
                "tokens and plan_entries must not be negative");
  TTJ_CHECK_ARG(a->tokens <= kMaxRows, TTJ_ERR_UNSUPPORTED, "more than 2^31 - 1 packed tokens");
  TTJ_CHECK_ARG((a->tokens == 0) == (a->plan_entries == 0) && a->plan_entries <= a->tokens, TTJ_ERR_INVALID_ARG,
                "the plan does not belong to this many tokens");
  if (a->tokens == 0) return TTJ_OK;
  TTJ_CHECK_ARG(a->plan_entries < (((int64_t)1 << 31) - 65536) / a->num_kv_heads, TTJ_ERR_UNSUPPORTED,
                "too many attention work items");
  TTJ_CHECK_ARG(a->q && a->k && a->v && a->out && a->plan, TTJ_ERR_INVALID_ARG,
                "q, k, v, out and plan must be non-NULL");
  TTJ_CHECK_ARG(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->out) && aligned16(a->plan),
                TTJ_ERR_ALIGNMENT, "q, k, v, out and plan must be 16-byte aligned");
  const int64_t t = a->tokens, hq = a->num_heads, hkv = a->num_kv_heads, hd = a->head_dim;
  if (int rc = check_strides("q", {{t, a->q_token_stride}, {hq, a->q_head_stride}})) return rc;
  if (int rc = check_strides("k", {{t, a->k_token_stride}, {hkv, a->k_head_stride}})) return rc;
  if (int rc = check_strides("v", {{t, a->v_token_stride}, {hkv, a->v_head_stride}})) return rc;
  TTJ_CHECK_ARG(t <= kMaxExtent / (hq * hd), TTJ_ERR_UNSUPPORTED, "tensor too large");
  TTJ_CHECK_ARG(a->scale > 0.f && std::isfinite(a->scale), TTJ_ERR_INVALID_ARG, "scale must be positive and finite");
  const Span out = span_of(a->out, 2, hd, {{t, hq * hd}, {hq, hd}});
  TTJ_CHECK_ARG(!overlap(out, span_of(a->q, 2, hd, {{t, a->q_token_stride}, {hq, a->q_head_stride}})) &&
                    !overlap(out, span_of(a->k, 2, hd, {{t, a->k_token_stride}, {hkv, a->k_head_stride}})) &&
                    !overlap(out, span_of(a->v, 2, hd, {{t, a->v_token_stride}, {hkv, a->v_head_stride}})),
                TTJ_ERR_INVALID_ARG, "out must not alias q, k or v");
  return ttj::launch_prompt_attn(*a, (cudaStream_t)stream);
}

size_t ttj_shared_prefix_attn_workspace_size(int64_t batch, int64_t prefix_len, int64_t capacity,
                                             int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                             int with_key_weights) {
  if (check_heads(num_heads, num_kv_heads, head_dim) != TTJ_OK) return 0;
  if (batch <= 0 || prefix_len < 0 || capacity < 0 || batch > kMaxRows || prefix_len > kMaxCache ||
      capacity > kMaxCache || batch > kMaxExtent / (num_heads * 256) / (capacity + 1))
    return 0;
  return ttj::shared_prefix_attn_workspace(batch, prefix_len, capacity, num_heads, num_kv_heads, head_dim,
                                           with_key_weights != 0);
}

int ttj_shared_prefix_attn_fwd(const ttj_shared_prefix_attn_args* a, ttj_stream_t stream) {
  TTJ_CHECK_ARG(a != nullptr, TTJ_ERR_INVALID_ARG, "args is NULL");
  if (int rc = check_dtype(a->dtype)) return rc;
  if (int rc = check_heads(a->num_heads, a->num_kv_heads, a->head_dim)) return rc;
  TTJ_CHECK_ARG(a->batch >= 0 && a->prefix_len >= 0 && a->capacity >= 0, TTJ_ERR_INVALID_ARG,
                "batch, prefix_len and capacity must not be negative");
  if (a->batch == 0) return TTJ_OK;
  const int64_t b = a->batch, p = a->prefix_len, c = a->capacity;
  const int64_t hq = a->num_heads, hkv = a->num_kv_heads, hd = a->head_dim;
  TTJ_CHECK_ARG(b <= kMaxRows && p <= kMaxCache && c <= kMaxCache && b <= kMaxExtent / (hq * 256) / (c + 1),
                TTJ_ERR_UNSUPPORTED, "batch, prefix_len or capacity above the supported maximum");
  TTJ_CHECK_ARG(b * hkv < ((int64_t)1 << 31) - 65536, TTJ_ERR_UNSUPPORTED, "too many attention work items");
  TTJ_CHECK_ARG(a->q && a->out && a->lengths && (p == 0 || (a->prefix_k && a->prefix_v)) &&
                    (c == 0 || (a->k_cache && a->v_cache)),
                TTJ_ERR_INVALID_ARG, "q, the used keys and values, lengths and out must be non-NULL");
  TTJ_CHECK_ARG((a->key_weights == nullptr) == (a->key_weights_out == nullptr), TTJ_ERR_INVALID_ARG,
                "key_weights and key_weights_out go together");
  TTJ_CHECK_ARG(aligned16(a->q) && aligned16(a->out) && (p == 0 || (aligned16(a->prefix_k) && aligned16(a->prefix_v))) &&
                    (c == 0 || (aligned16(a->k_cache) && aligned16(a->v_cache))),
                TTJ_ERR_ALIGNMENT, "q, keys, values and out must be 16-byte aligned");
  if (int rc = check_strides("q", {{b, a->q_seq_stride}, {hq, a->q_head_stride}})) return rc;
  if (p > 0) {
    if (int rc = check_strides("prefix_k", {{p, a->prefix_k_row_stride}, {hkv, a->prefix_k_head_stride}})) return rc;
    if (int rc = check_strides("prefix_v", {{p, a->prefix_v_row_stride}, {hkv, a->prefix_v_head_stride}})) return rc;
  }
  if (c > 0) {
    if (int rc = check_strides("k_cache", {{b, a->k_seq_stride}, {c, a->k_row_stride}, {hkv, a->k_head_stride}}))
      return rc;
    if (int rc = check_strides("v_cache", {{b, a->v_seq_stride}, {c, a->v_row_stride}, {hkv, a->v_head_stride}}))
      return rc;
  }
  TTJ_CHECK_ARG(a->scale > 0.f && std::isfinite(a->scale), TTJ_ERR_INVALID_ARG, "scale must be positive and finite");
  const Span out = span_of(a->out, 2, hd, {{b, hq * hd}, {hq, hd}});
  TTJ_CHECK_ARG(!overlap(out, span_of(a->q, 2, hd, {{b, a->q_seq_stride}, {hq, a->q_head_stride}})),
                TTJ_ERR_INVALID_ARG, "out must not alias q");
  if (a->key_weights != nullptr && c > 0)
    TTJ_CHECK_ARG(!overlap(span_of(a->key_weights, 4, c, {{b * hkv, c}}), span_of(a->key_weights_out, 4, c, {{b * hkv, c}})),
                  TTJ_ERR_INVALID_ARG, "key_weights_out must not alias key_weights");
  const size_t need = ttj::shared_prefix_attn_workspace(b, p, c, hq, hkv, hd, a->key_weights != nullptr);
  TTJ_CHECK_ARG(need == 0 || (a->workspace != nullptr && a->workspace_bytes >= need), TTJ_ERR_WORKSPACE,
                "workspace missing or smaller than ttj_shared_prefix_attn_workspace_size()");
  TTJ_CHECK_ARG(aligned16(a->workspace), TTJ_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  return ttj::launch_shared_prefix_attn(*a, (cudaStream_t)stream);
}

int ttj_cache_evict(const ttj_cache_evict_args* a, ttj_stream_t stream) {
  TTJ_CHECK_ARG(a != nullptr, TTJ_ERR_INVALID_ARG, "args is NULL");
  const int64_t b = a->batch, c = a->capacity, hkv = a->num_kv_heads, hd = a->head_dim, n = a->budget;
  if (int rc = check_heads(hkv, hkv, hd)) return rc;
  TTJ_CHECK_ARG(b >= 0 && c >= 0, TTJ_ERR_INVALID_ARG, "batch and capacity must not be negative");
  TTJ_CHECK_ARG(n > 0, TTJ_ERR_INVALID_ARG, "budget must be positive");
  TTJ_CHECK_ARG(a->recent >= 0 && a->recent <= n, TTJ_ERR_INVALID_ARG, "recent must lie in 0 .. budget");
  if (b == 0) return TTJ_OK;
  TTJ_CHECK_ARG(b <= kMaxRows && c <= kMaxCache && n <= kMaxCache && b <= kMaxExtent / (hkv * 256) / (c + n),
                TTJ_ERR_UNSUPPORTED, "batch, capacity or budget above the supported maximum");
  TTJ_CHECK_ARG(b * hkv < ((int64_t)1 << 31) - 65536, TTJ_ERR_UNSUPPORTED, "too many caches");
  TTJ_CHECK_ARG((c == 0 || (a->k_cache && a->v_cache && a->key_weights)) && a->lengths && a->k_out && a->v_out &&
                    a->weights_out && a->lengths_out && a->positions_out,
                TTJ_ERR_INVALID_ARG, "caches, weights, lengths and outputs must be non-NULL");
  TTJ_CHECK_ARG((c == 0 || (aligned16(a->k_cache) && aligned16(a->v_cache))) && aligned16(a->k_out) && aligned16(a->v_out),
                TTJ_ERR_ALIGNMENT, "caches must be 16-byte aligned");
  if (c > 0) {
    if (int rc = check_strides("k_cache", {{b, a->k_seq_stride}, {c, a->k_row_stride}, {hkv, a->k_head_stride}}))
      return rc;
    if (int rc = check_strides("v_cache", {{b, a->v_seq_stride}, {c, a->v_row_stride}, {hkv, a->v_head_stride}}))
      return rc;
  }
  if (int rc = check_strides("k_out", {{b, a->k_out_seq_stride}, {n, a->k_out_row_stride}, {hkv, a->k_out_head_stride}}))
    return rc;
  if (int rc = check_strides("v_out", {{b, a->v_out_seq_stride}, {n, a->v_out_row_stride}, {hkv, a->v_out_head_stride}}))
    return rc;
  const Span ko = span_of(a->k_out, 2, hd, {{b, a->k_out_seq_stride}, {n, a->k_out_row_stride}, {hkv, a->k_out_head_stride}});
  const Span vo = span_of(a->v_out, 2, hd, {{b, a->v_out_seq_stride}, {n, a->v_out_row_stride}, {hkv, a->v_out_head_stride}});
  const Span wo = span_of(a->weights_out, 4, n, {{b * hkv, n}});
  // k_out and v_out may be interleaved row by row in one allocation.
  const int64_t row = (hkv - 1) * a->k_out_head_stride + hd;
  const int64_t gap = std::abs((int64_t)(ko.lo - vo.lo)) / 2;
  const bool interleaved = a->k_out_seq_stride == a->v_out_seq_stride && a->k_out_row_stride == a->v_out_row_stride &&
                           a->k_out_head_stride == a->v_out_head_stride && gap >= row && gap + row <= a->k_out_row_stride;
  TTJ_CHECK_ARG(interleaved || !overlap(ko, vo), TTJ_ERR_INVALID_ARG, "k_out and v_out must not alias");
  // One head's blocks write a sequence's new length while the others' still read it.
  TTJ_CHECK_ARG(!overlap(span_of(a->lengths, 4, b, {}), span_of(a->lengths_out, 4, b, {})), TTJ_ERR_INVALID_ARG,
                "lengths_out must not alias lengths");
  if (c > 0) {
    const Span ki = span_of(a->k_cache, 2, hd, {{b, a->k_seq_stride}, {c, a->k_row_stride}, {hkv, a->k_head_stride}});
    const Span vi = span_of(a->v_cache, 2, hd, {{b, a->v_seq_stride}, {c, a->v_row_stride}, {hkv, a->v_head_stride}});
    const Span wi = span_of(a->key_weights, 4, c, {{b * hkv, c}});
    TTJ_CHECK_ARG(!overlap(ko, ki) && !overlap(ko, vi) && !overlap(vo, ki) && !overlap(vo, vi) && !overlap(wo, wi),
                  TTJ_ERR_INVALID_ARG, "outputs must not alias the cache");
  }
  return ttj::launch_cache_evict(*a, (cudaStream_t)stream);
}

}  // extern "C"
