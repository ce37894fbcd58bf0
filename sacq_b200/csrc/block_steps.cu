// C ABI of the steps between a block's quantized projections: attention over packed sequences, rotary positions, norms
// around a block.  Argument checks and the choice of the kernel.
#include <math.h>

#include "attention.cuh"
#include "common.cuh"

namespace sacq {

int launch_rotate_heads(const sacq_rotary_desc& d, cudaStream_t s);
int launch_residual_norm(const sacq_residual_norm_desc& d, cudaStream_t s);
int residual_norm_status(int* out);

namespace {

int check_size(const void* desc, uint32_t size, size_t want, const char* what) {
  if (desc == nullptr) return set_error(SACQ_ERR_INVALID_ARGUMENT, "null argument");
  if (size != want)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "%s.struct_size is %u, this library expects %zu", what, size, want);
  return SACQ_OK;
}

}  // namespace

}  // namespace sacq

using namespace sacq;

SACQ_API int sacq_rotate_heads(const sacq_rotary_desc* d, void* stream) {
  if (int rc = check_size(d, d ? d->struct_size : 0, sizeof(*d), "sacq_rotary_desc")) return rc;
  if (d->tokens < 0 || d->q.heads < 0 || d->k.heads < 0 || d->head_dim <= 0)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "bad geometry (tokens=%lld heads=%d,%d head_dim=%d)", (long long)d->tokens,
                     d->q.heads, d->k.heads, d->head_dim);
  if (d->rotary_dim <= 0 || d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "rotary_dim=%d is not an even number up to head_dim=%d", d->rotary_dim, d->head_dim);
  if (d->layout != SACQ_ROTARY_HALF && d->layout != SACQ_ROTARY_INTERLEAVED)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "unknown layout %d", d->layout);
  if (d->position_bytes != 4 && d->position_bytes != 8)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "positions of %d bytes", d->position_bytes);
  if (d->head_dim > 4096 || d->q.heads > 65536 || d->k.heads > 65536 ||
      (int64_t)(d->q.heads + d->k.heads) * d->head_dim > (1 << 22))
    return set_error(SACQ_ERR_UNSUPPORTED, "heads of a token beyond 2^22 elements, or of more than 4,096");
  if (d->tokens == 0 || d->q.heads + d->k.heads == 0) return SACQ_OK;
  if (d->positions == nullptr || d->inv_freq == nullptr || (d->q.heads > 0 && (d->q.in == nullptr || d->q.out == nullptr)) ||
      (d->k.heads > 0 && (d->k.in == nullptr || d->k.out == nullptr)))
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "null argument");
  return launch_rotate_heads(*d, static_cast<cudaStream_t>(stream));
}

SACQ_API int sacq_residual_norm(const sacq_residual_norm_desc* d, void* stream) {
  if (int rc = check_size(d, d ? d->struct_size : 0, sizeof(*d), "sacq_residual_norm_desc")) return rc;
  if (d->M < 0 || d->K < 0) return set_error(SACQ_ERR_INVALID_ARGUMENT, "negative size (M=%lld K=%lld)", (long long)d->M,
                                             (long long)d->K);
  if (d->M == 0) return SACQ_OK;
  if (d->K == 0) return set_error(SACQ_ERR_INVALID_ARGUMENT, "K must be positive");
  if (d->branch == nullptr || d->residual == nullptr || d->residual_out == nullptr)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "null argument");
  if ((d->q_out == nullptr) != (d->scale_out == nullptr))
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "8-bit rows need both q_out and scale_out");
  if (d->q_out == nullptr && d->normalized_out == nullptr)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "neither q_out nor normalized_out is given");
  if (d->norm != SACQ_NORM_RMS && d->norm != SACQ_NORM_LAYER)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "unknown norm %d", d->norm);
  if (d->post_norm != SACQ_NORM_NONE && d->post_norm != SACQ_NORM_RMS && d->post_norm != SACQ_NORM_LAYER)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "unknown post_norm %d", d->post_norm);
  if (d->post_norm == SACQ_NORM_NONE && (d->post_weight != nullptr || d->post_bias != nullptr))
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "post_weight and post_bias need a post_norm");
  if ((d->mod_scale == nullptr) != (d->mod_shift == nullptr))
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "modulation needs both its scale and its shift vectors");
  if (d->vector_rows != nullptr && d->vectors <= 0)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "vector_rows without a number of vectors");
  if (d->branch_pitch < d->K || d->residual_pitch < d->K)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "row pitch smaller than K=%lld", (long long)d->K);
  if (!(d->eps >= 0.f)) return set_error(SACQ_ERR_INVALID_ARGUMENT, "eps must be non-negative");
  return launch_residual_norm(*d, static_cast<cudaStream_t>(stream));
}

namespace {

int check_attention(const sacq_attention_desc* d) {
  if (int rc = check_size(d, d ? d->struct_size : 0, sizeof(*d), "sacq_attention_desc")) return rc;
  if (d->tokens_q < 0 || d->tokens_k < 0 || d->sequences < 0 || d->heads <= 0 || d->kv_heads <= 0 || d->head_dim <= 0)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "bad geometry (tokens=%lld,%lld sequences=%d heads=%d,%d head_dim=%d)",
                     (long long)d->tokens_q, (long long)d->tokens_k, d->sequences, d->heads, d->kv_heads, d->head_dim);
  if (d->heads % d->kv_heads != 0)
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "%d heads are no multiple of %d key-value heads", d->heads, d->kv_heads);
  if (d->head_dim > 256) return set_error(SACQ_ERR_UNSUPPORTED, "head_dim=%d above 256", d->head_dim);
  if (d->tokens_q > 2147480000LL || d->tokens_k > 2147480000LL || d->heads > 65536)
    return set_error(SACQ_ERR_UNSUPPORTED, "more than 2,147,480,000 tokens or 65,536 heads");
  if (!(d->scale > 0.f) || isinf(d->scale)) return set_error(SACQ_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  return SACQ_OK;
}

}  // namespace

namespace {

AttnParams attention_params(const sacq_attention_desc* d) {
  AttnParams p = {};
  p.q = static_cast<const uint16_t*>(d->q);
  p.k = static_cast<const uint16_t*>(d->k);
  p.v = static_cast<const uint16_t*>(d->v);
  p.out = static_cast<uint16_t*>(d->out);
  p.lse = d->lse;
  p.q_token = d->q_token; p.q_head = d->q_head;
  p.k_token = d->k_token; p.k_head = d->k_head;
  p.v_token = d->v_token; p.v_head = d->v_head;
  p.out_token = d->out_token; p.out_head = d->out_head;
  p.cu_q = d->cu_q; p.cu_k = d->cu_k;
  p.tokens_q = d->tokens_q; p.tokens_k = d->tokens_k;
  p.sequences = d->sequences; p.heads = d->heads; p.kv_heads = d->kv_heads; p.dim = d->head_dim;
  p.causal = d->causal != 0;
  p.scale = d->scale;
  return p;
}

}  // namespace

namespace {

enum { kByRows, kShort, kTmem };
// Sequences of few rows (queries x heads of a group) are bound by reading their keys: a kernel of 16-row tiles for them.  Only the
// average is known here.
int attention_kernel(const AttnParams& p) {
  if (!attention_tma_supported(p)) return kByRows;
  const int64_t rows = p.tokens_q * (p.heads / p.kv_heads);
  return rows <= 32 * (int64_t)p.sequences && rows < (1ll << 31) - 64 ? kShort : kTmem;
}
AttnSplit split_for(const AttnParams& p, int kernel, void* workspace) {
  return kernel == kShort ? attention_short_split(p, workspace) : attention_tmem_split(p, workspace);
}

}  // namespace

SACQ_API int64_t sacq_attention_workspace_bytes(const sacq_attention_desc* d) {
  if (int rc = check_attention(d)) return rc;
  if (d->tokens_q == 0 || d->sequences == 0) return 0;
  const AttnParams p = attention_params(d);
  const int kernel = attention_kernel(p);
  return kernel == kByRows ? 0 : attention_split_bytes(p, split_for(p, kernel, nullptr));
}

SACQ_API int sacq_attention_packed(const sacq_attention_desc* d, void* stream) {
  if (int rc = check_attention(d)) return rc;
  if (d->tokens_q == 0 || d->sequences == 0) return SACQ_OK;
  if (d->q == nullptr || d->out == nullptr || d->cu_q == nullptr || d->cu_k == nullptr ||
      (d->tokens_k > 0 && (d->k == nullptr || d->v == nullptr)))
    return set_error(SACQ_ERR_INVALID_ARGUMENT, "null argument");
  const AttnParams p = attention_params(d);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kernel = attention_kernel(p);
  if (kernel == kByRows) return launch_attention_rows(p, s);
  const AttnSplit split = split_for(p, kernel, d->workspace);
  const int64_t need = attention_split_bytes(p, split);
  if (need > 0) {
    if (d->workspace == nullptr || d->workspace_bytes < need)
      return set_error(SACQ_ERR_WORKSPACE, "workspace of %lld bytes, %lld are needed", (long long)(d->workspace ? d->workspace_bytes : 0), (long long)need);
    if (reinterpret_cast<uintptr_t>(d->workspace) % 256 != 0) return set_error(SACQ_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  }
  if (int rc = kernel == kShort ? launch_attention_short(p, split, s) : launch_attention_tmem(p, split, s)) return rc;
  return split.chunks_most > 1 ? launch_attention_join(p, split, s) : SACQ_OK;
}

SACQ_API int sacq_block_steps_status(int* status_out) {
  if (status_out == nullptr) return set_error(SACQ_ERR_INVALID_ARGUMENT, "null argument");
  int norm = 0;
  if (int rc = attention_status(status_out)) return rc;
  if (int rc = residual_norm_status(&norm)) return rc;
  *status_out |= norm;
  return SACQ_OK;
}
