// What the attention kernels share on the host, and the kernel that joins the chunks of a query.
#include "attention.cuh"
#include "umma.cuh"

namespace sacq {

namespace {

__device__ int g_attention_status;            // nonzero: a wait of an attention kernel ran out

// A warp per row and head; the chunks are taken in their order.
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ AttnParams a, const __grid_constant__ AttnSplit split) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t token = item / a.heads;
  const int head = (int)(item - token * a.heads);
  if (token >= a.tokens_q) return;
  const int sequence = sequence_of(a.cu_q, a.sequences, a.tokens_q, token);
  if (sequence < 0) return;
  const Span sq = span_of(a.cu_q, sequence, a.tokens_q), sk = span_of(a.cu_k, sequence, a.tokens_k);
  const int chunks = chunks_of(split, (int)sk.length);
  if (chunks == 1) return;                   // written by the attention kernel
  const int64_t stride = a.tokens_q * a.heads, at = token * a.heads + head;
  float m = -INFINITY;
  for (int i = lane; i < chunks; i += 32) m = fmaxf(m, split.part_lse[i * stride + at]);
  m = warp_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  const int d = lane * 4;
  const float* const src = split.part_o + at * a.dim + (d < a.dim ? d : 0);
  for (int first = 0; first < chunks; first += 32) {
    // this lane's chunk's weight: 0 where the query sees none of its keys or all of them score -inf, and the part is zeros
    const int n = min(32, chunks - first);
    const float f = lane < n ? exp2f((split.part_lse[(first + lane) * stride + at] - base) * kLog2e) : 0.f;
    for (int i = 0; i < n; i += 8) {         // eight parts are on their way at a time
      float4 v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const float4*>(src + (first + min(i + e, n - 1)) * stride * a.dim);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = __shfl_sync(0xffffffffu, f, min(i + e, 31));
        if (i + e >= n) break;
        l += w;
        o[0] = fmaf(v[e].x, w, o[0]);
        o[1] = fmaf(v[e].y, w, o[1]);
        o[2] = fmaf(v[e].z, w, o[2]);
        o[3] = fmaf(v[e].w, w, o[3]);
      }
    }
  }
  const bool some = a.causal ? token - sq.begin + sk.length - sq.length >= 0 : true;      // keys that the query sees: they may all score -inf
  if (d < a.dim) {
    const float inv = some ? 1.0f / l : 0.f;
    *reinterpret_cast<uint2*>(a.out + token * a.out_token + head * a.out_head + d) =
        make_uint2(bf16_pair(o[0] * inv, o[1] * inv), bf16_pair(o[2] * inv, o[3] * inv));
  }
  if (a.lse != nullptr && lane == 0) a.lse[at] = some ? base + logf(l) : -INFINITY;
}

bool strides_for_tma(int64_t token, int64_t head, int heads, int64_t tokens) {
  auto fine = [](int64_t s, int64_t n) { return n == 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
  return fine(head, heads) && fine(token, tokens);
}

int64_t lse_offset(const AttnParams& a, int64_t chunks) { return (chunks * a.tokens_q * a.heads * a.dim * 4 + 255) / 256 * 256; }

}  // namespace

int device_sms() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    sms[dev] = n;
  }
  return sms[dev];
}

int* attention_status_word() {
  static int* word[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (word[dev] == nullptr) {
    void* at = nullptr;
    if (cudaGetSymbolAddress(&at, g_attention_status) != cudaSuccess) return nullptr;
    word[dev] = static_cast<int*>(at);
  }
  return word[dev];
}

int attention_status(int* out) {
  SACQ_CUDA_TRY(cudaMemcpyFromSymbol(out, g_attention_status, sizeof(int)));
  return SACQ_OK;
}

bool attention_tma_supported(const AttnParams& a) {
  auto al = [](const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  return a.dim <= 128 && a.dim % 8 == 0 && a.tokens_k > 0 && al(a.q, 16) && al(a.k, 16) && al(a.v, 16) && al(a.out, 16) &&
         strides_for_tma(a.out_token, a.out_head, a.heads, a.tokens_q) && strides_for_tma(a.q_token, a.q_head, a.heads, a.tokens_q) &&
         strides_for_tma(a.k_token, a.k_head, a.kv_heads, a.tokens_k) && strides_for_tma(a.v_token, a.v_head, a.kv_heads, a.tokens_k);
}

AttnSplit attention_chunks(const AttnParams& a, int64_t chunk, void* workspace) {
  AttnSplit s = {};
  const int64_t tiles = (a.tokens_k + kKeyTile - 1) / kKeyTile;            // of the longest sequence there can be
  s.chunk = (int)(tiles < 1 ? 1 : tiles);
  s.chunks_most = 1;
  if (chunk > 0) {
    const int64_t most_bytes = 256ll << 20, row = a.tokens_q * a.heads * (a.dim + 1) * 4;
    while (chunk < tiles && (tiles + chunk - 1) / chunk * row > most_bytes) chunk *= 2;
    if (2 * chunk <= tiles + 1) {
      s.chunk = (int)chunk;
      s.chunks_most = (int)((tiles + chunk - 1) / chunk);
    }
  }
  if (s.chunks_most > 1) {
    s.part_o = static_cast<float*>(workspace);
    s.part_lse = workspace == nullptr ? nullptr : reinterpret_cast<float*>(static_cast<char*>(workspace) + lse_offset(a, s.chunks_most));
  }
  return s;
}

int64_t attention_split_bytes(const AttnParams& a, const AttnSplit& s) {
  return s.chunks_most == 1 ? 0 : lse_offset(a, s.chunks_most) + (int64_t)s.chunks_most * a.tokens_q * a.heads * 4;
}

namespace {
int heads_map(CUtensorMap* m, const AttnParams& a, const void* base, int64_t tokens, int heads, int64_t token, int64_t head, int box_heads, int box_tokens) {
  // the stride of a dimension of one element means nothing, but is checked
  const int64_t h = heads == 1 ? a.dim : head, t = tokens == 1 ? (int64_t)a.dim * heads : token;
  return encode_bf16_3d(m, base, (uint64_t)a.dim, (uint64_t)heads, (uint64_t)tokens, (uint64_t)h, (uint64_t)t, 64u, (uint32_t)box_heads,
                        (uint32_t)box_tokens, CU_TENSOR_MAP_SWIZZLE_128B);
}
}  // namespace

int attention_tensor_maps(const AttnParams& a, int q_box_heads, int q_box_tokens, int k_box_tokens, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v) {
  if (q != nullptr)
    if (int rc = heads_map(q, a, a.q, a.tokens_q, a.heads, a.q_token, a.q_head, q_box_heads, q_box_tokens)) return rc;
  if (int rc = heads_map(k, a, a.k, a.tokens_k, a.kv_heads, a.k_token, a.k_head, 1, k_box_tokens)) return rc;
  return heads_map(v, a, a.v, a.tokens_k, a.kv_heads, a.v_token, a.v_head, 1, k_box_tokens);
}

int attention_out_map(const AttnParams& a, int box_heads, int box_tokens, CUtensorMap* out) {
  return heads_map(out, a, a.out, a.tokens_q, a.heads, a.out_token, a.out_head, box_heads, box_tokens);
}

int launch_attention_join(const AttnParams& a, const AttnSplit& split, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.tokens_q * a.heads + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<AttnParams*>(&a), const_cast<AttnSplit*>(&split)};
  SACQ_CUDA_TRY(cudaLaunchKernelExC(&cfg, (const void*)attention_join_kernel, args));
  count_launch();
  return SACQ_OK;
}

}  // namespace sacq
