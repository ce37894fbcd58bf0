// Attention over packed sequences: what its kernels share.
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  lse_i = m_i + ln sum_j p_ij
// over the keys j that query i sees: those of its sequence, with `causal` up to the query's own place when both ends are
// aligned (j <= i + keys - queries).  A query that sees none has out = 0 and lse = -inf.
#pragma once

#include "common.cuh"

namespace sacq {

struct AttnParams {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  float* lse;                      // [tokens_q, heads] or null
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;   // strides, elements
  const int32_t *cu_q, *cu_k;      // [sequences + 1]
  int64_t tokens_q, tokens_k;
  int sequences, heads, kv_heads, dim;
  int causal;
  float scale;
};

// Rows of sequence s.  Offsets that lie outside of the tensor or go backwards are cut to it: no access leaves it.
struct Span {
  int64_t begin, length;
};
__device__ __forceinline__ Span span_of(const int32_t* cu, int s, int64_t tokens) {
  const int64_t a = min(max((int64_t)cu[s], (int64_t)0), tokens), b = min(max((int64_t)cu[s + 1], (int64_t)0), tokens);
  return {a, b > a ? b - a : 0};
}

// One query row by one warp, key after key with a running maximum: lane l holds elements l, l + 32, ...  Returns the
// row's 1 / sum and leaves the sums in acc.
template <int E>
struct RowState {
  float acc[E];
  float m, l;
};
template <int E>
__device__ void attend_row(const AttnParams& p, const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t keys, RowState<E>& st) {
  const int lane = threadIdx.x & 31;
  float qe[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qe[e] = lane + 32 * e < p.dim ? bf16_bits_to_float(q[lane + 32 * e]) * p.scale : 0.f;
    st.acc[e] = 0.f;
  }
  st.m = -INFINITY;
  st.l = 0.f;
  for (int64_t j = 0; j < keys; ++j) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < p.dim) s = fmaf(qe[e], bf16_bits_to_float(k[j * p.k_token + lane + 32 * e]), s);
    s = warp_sum(s);
    const float m = fmaxf(st.m, s), base = m == -INFINITY ? 0.f : m;
    const float keep = expf(st.m - base), w = expf(s - base);
    st.m = m;
    st.l = st.l * keep + w;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < p.dim) st.acc[e] = fmaf(st.acc[e], keep, w * bf16_bits_to_float(v[j * p.v_token + lane + 32 * e]));
  }
}

int launch_attention_rows(const AttnParams& p, cudaStream_t s);          // any head dim up to 256, any alignment

// Tensor cores: head dims that are multiples of 8 up to 128, rows that TMA can read.
bool attention_tmem_supported(const AttnParams& p);
int64_t attention_tmem_workspace(const AttnParams& p);
int attention_tmem_status(int* out);
int launch_attention_tmem(const AttnParams& p, void* workspace, int64_t workspace_bytes, cudaStream_t s);

}  // namespace sacq
