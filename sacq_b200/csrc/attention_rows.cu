// Attention over packed sequences for any head dim up to 256 and any alignment: a warp per query row and head.
// Every query reads its keys by itself, so it is bound by L2 traffic and by 12 instructions per key and 32 elements.
#include "attention.cuh"

namespace sacq {

namespace {

constexpr int kRowWarps = 4;

template <int E>
__global__ void __launch_bounds__(kRowWarps * 32) attention_rows_kernel(const __grid_constant__ AttnParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int64_t token = item / p.heads;
  const int head = (int)(item - token * p.heads);
  if (token >= p.tokens_q) return;
  const int sequence = sequence_of(p.cu_q, p.sequences, p.tokens_q, token);
  if (sequence < 0) return;
  const Span sq = span_of(p.cu_q, sequence, p.tokens_q), sk = span_of(p.cu_k, sequence, p.tokens_k);
  int64_t keys = sk.length;
  if (p.causal) keys = min(keys, max((int64_t)0, token - sq.begin + 1 + sk.length - sq.length));
  const int kv = head / (p.heads / p.kv_heads);
  RowState<E> st;
  attend_row<E>(p, p.q + token * p.q_token + head * p.q_head, p.k + sk.begin * p.k_token + kv * p.k_head,
                p.v + sk.begin * p.v_token + kv * p.v_head, keys, st);
  uint16_t* out = p.out + token * p.out_token + head * p.out_head;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < p.dim) out[lane + 32 * e] = float_to_bf16_bits(keys > 0 ? st.acc[e] / st.l : 0.f);
  if (p.lse != nullptr && lane == 0) p.lse[token * p.heads + head] = keys > 0 ? st.m + logf(st.l) : -INFINITY;
}

}  // namespace

int launch_attention_rows(const AttnParams& p, cudaStream_t s) {
  const int64_t grid = (p.tokens_q * p.heads + kRowWarps - 1) / kRowWarps;
  if (grid > 2147483647LL) return set_error(SACQ_ERR_UNSUPPORTED, "%lld queries exceed the grid limit", (long long)p.tokens_q);
  const int e = (p.dim + 31) / 32;
  const void* fn = e <= 2 ? (const void*)attention_rows_kernel<2> : e <= 4 ? (const void*)attention_rows_kernel<4>
                                                                          : (const void*)attention_rows_kernel<8>;
  void* args[] = {const_cast<AttnParams*>(&p)};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kRowWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SACQ_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
  count_launch();
  return SACQ_OK;
}

}  // namespace sacq
