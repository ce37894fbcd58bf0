// Attention over packed sequences: what its kernels share.
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  lse_i = m_i + ln sum_j p_ij
// over the keys j that query i sees: those of its sequence, with `causal` up to the query's own place when both ends are
// aligned (j <= i + keys - queries).  A query that sees none has out = 0 and lse = -inf.
#pragma once

#include <cuda.h>

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

// The sequence that a query token lies in, by a whole warp; -1: none.  Offsets that never go down are bisected, in which the last sequence that
// begins at or in front of the token is found; where that one does not hold it, because sequences lie in another order, empty ones
// begin in front of it, or none does, all are looked at, 32 at a time.
__device__ __forceinline__ int sequence_of(const int32_t* cu_q, int sequences, int64_t tokens_q, int64_t token) {
  auto holds = [&](int s) {
    const Span q = span_of(cu_q, s, tokens_q);
    return token >= q.begin && token < q.begin + q.length;
  };
  int lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid] <= token) lo = mid; else hi = mid;
  }
  if (holds(lo)) return lo;
  for (int first = 0; first < sequences; first += 32) {
    const int s = first + (threadIdx.x & 31);
    const uint32_t found = __ballot_sync(0xffffffffu, s < sequences && holds(s));
    if (found != 0) return first + __ffs(found) - 1;
  }
  return -1;
}

// One query row by one warp, key after key with a running maximum: lane l holds elements l, l + 32, ... of the weighted sum in acc, every
// lane the maximum m and the sum of weights l.
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
  constexpr int kAtOnce = 4;                 // scores whose sums over the lanes run together
  for (int64_t j = 0; j < keys; j += kAtOnce) {
    float s[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      s[i] = 0.f;
      const uint16_t* const row = k + min(j + i, keys - 1) * p.k_token;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + 32 * e < p.dim) s[i] = fmaf(qe[e], bf16_bits_to_float(row[lane + 32 * e]), s[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    float m = st.m;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) m = fmaxf(m, s[i]);
    const float base = m == -INFINITY ? 0.f : m, keep = expf(st.m - base);
    st.m = m;
    st.l *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) st.acc[e] *= keep;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (j + i >= keys) break;
      const float w = expf(s[i] - base);
      st.l += w;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + 32 * e < p.dim) st.acc[e] = fmaf(w, bf16_bits_to_float(v[(j + i) * p.v_token + lane + 32 * e]), st.acc[e]);
    }
  }
}

// A call that is cut up: chunks of `chunk` key tiles whose results, with their own lse, a second kernel joins.
constexpr int kKeyTile = 128;
struct AttnSplit {
  int chunk, chunks_most;          // chunks of the longest sequence possible; 1: results go straight to out
  float* part_o;                   // [chunks_most][tokens_q][heads][dim]
  float* part_lse;                 // [chunks_most][tokens_q][heads]
};
__host__ __device__ __forceinline__ int key_tiles(int keys) { return (keys + kKeyTile - 1) / kKeyTile; }
__device__ __forceinline__ int chunks_of(const AttnSplit& s, int keys) {
  if (s.chunks_most == 1) return 1;
  const int n = (key_tiles(keys) + s.chunk - 1) / s.chunk;
  return n > 1 ? n : 1;
}

constexpr float kLog2e = 1.4426950408889634f;
// Waits of these kernels: a warp that makes 32 rows again (redo_rows) is at it for 60 clocks a row and key, a microsecond a key, and others wait meanwhile:
// long enough for 10 million keys.
constexpr uint64_t kWaitNs = 10000000000ull;
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}

// Rows that a value which is not finite got into with a weight of zero (0 x inf), one after another by a warp: each from the keys that it
// sees, row by row.  Each lane has a row: its token, head and number of keys `mine`, and whether it is one to be looked at; keys up to
// `end` were multiplied.  A row is made again only if such a value lies between its own end and that one: what is not finite among
// the keys that it sees is in its result by right.  5,000 causal tokens, the first with a NaN, 4 heads: 73 us at head dim 64 and 89 at 128, without
// the NaN 68 and 79; rows made again for what they see took 7.2 and 8.8 ms.  part: the chunk, or -1; elements [from, to) are written.
__device__ __noinline__ inline void redo_rows(const AttnParams& a, const AttnSplit& split, int k_row, int kv_head, int part, int64_t token, int head, int mine,
                                              bool again, int end, int from, int to) {
  const int lane = threadIdx.x & 31, pieces = a.dim / 8;
  const uint16_t* const k = a.k + k_row * a.k_token + kv_head * a.k_head;
  const uint16_t* const v = a.v + k_row * a.v_token + kv_head * a.v_head;
  const int first = __reduce_min_sync(0xffffffffu, again ? mine : end);
  int last = -1;                             // key whose value is not finite
  for (int i = lane; i < (end - first) * pieces; i += 32) {
    const int row = first + i / pieces;
    const uint4 u = *reinterpret_cast<const uint4*>(v + row * a.v_token + i % pieces * 8);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u) last = row;
  }
  last = __reduce_max_sync(0xffffffffu, last);
  for (uint32_t odd = __ballot_sync(0xffffffffu, again && mine <= last); odd != 0; odd &= odd - 1) {
    const int src = __ffs(odd) - 1, h = __shfl_sync(0xffffffffu, head, src);
    const int64_t t = __shfl_sync(0xffffffffu, token, src);
    RowState<4> st;
    attend_row<4>(a, a.q + t * a.q_token + h * a.q_head, k, v, __shfl_sync(0xffffffffu, mine, src), st);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      if (d >= a.dim || d < from || d >= to) continue;
      if (part < 0) a.out[t * a.out_token + h * a.out_head + d] = float_to_bf16_bits(st.acc[e] / st.l);
      else split.part_o[(((int64_t)part * a.tokens_q + t) * a.heads + h) * a.dim + d] = st.m == -INFINITY ? st.acc[e] : st.acc[e] / st.l;
    }
  }
}

// Items of work, sequence after sequence, listed by one warp: 32 sequences are looked at at a time.  count(queries, keys) is how
// many items a sequence has.
template <typename Count>
struct ItemList {
  const AttnParams& a;
  Count count;
  int window = 0;
  int64_t before = 0, mine = 0, upto = 0;      // items in front of the window; this lane's sequence's, and up to it
  Span sq = {0, 0}, sk = {0, 0};
  __device__ __forceinline__ void look() {
    const int lane = threadIdx.x & 31, s = window + lane;
    mine = 0;
    sq = sk = {0, 0};
    if (s < a.sequences) {
      sq = span_of(a.cu_q, s, a.tokens_q);
      sk = span_of(a.cu_k, s, a.tokens_k);
      mine = count((int)sq.length, (int)sk.length);
    }
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
  }
  // The sequence of item `index` (best not smaller than the last one asked for), and which of its items that is; false: there is none.
  __device__ __forceinline__ bool find(int64_t index, Span& q, Span& k, int64_t& which) {
    if (index < before) {
      before = 0;
      window = 0;
      look();
    }
    int64_t all = __shfl_sync(0xffffffffu, upto, 31);
    while (window < a.sequences && index >= before + all) {
      before += all;
      window += 32;
      look();
      all = __shfl_sync(0xffffffffu, upto, 31);
    }
    const uint32_t found = __ballot_sync(0xffffffffu, index < before + upto);
    if (window >= a.sequences || found == 0) return false;
    const int src = __ffs(found) - 1;
    q = {__shfl_sync(0xffffffffu, sq.begin, src), __shfl_sync(0xffffffffu, sq.length, src)};
    k = {__shfl_sync(0xffffffffu, sk.begin, src), __shfl_sync(0xffffffffu, sk.length, src)};
    which = index - (before + __shfl_sync(0xffffffffu, upto, src) - __shfl_sync(0xffffffffu, mine, src));
    return true;
  }
};

// The next digit of `r` in base `n`; r is left with the rest.  (A 64-bit division takes about 100 instructions.)
__device__ __forceinline__ int digit_of(int64_t& r, int n) {
  if (n == 1) return 0;
  if (r >> 32 == 0) {
    const uint32_t x = (uint32_t)r, y = x / (uint32_t)n;
    r = y;
    return (int)(x - y * (uint32_t)n);
  }
  const int d = (int)(r % n);
  r /= n;
  return d;
}

int launch_attention_rows(const AttnParams& p, cudaStream_t s);          // any head dim up to 256, any alignment
int launch_attention_join(const AttnParams& a, const AttnSplit& split, cudaStream_t s);

// Head dims that are multiples of 8 up to 128, rows that TMA can read.
bool attention_tma_supported(const AttnParams& p);
// A call in chunks of `chunk` key tiles, or of more where their results would not fit 256 MB; 0: not cut up.
AttnSplit attention_chunks(const AttnParams& a, int64_t chunk, void* workspace);
int64_t attention_split_bytes(const AttnParams& a, const AttnSplit& split);
int attention_tensor_maps(const AttnParams& a, int q_box_heads, int q_box_tokens, int k_box_tokens, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v);
int attention_out_map(const AttnParams& a, int box_heads, int box_tokens, CUtensorMap* out);

// Tensor cores by tcgen05: tiles of 128 query rows.
AttnSplit attention_tmem_split(const AttnParams& p, void* workspace);
int launch_attention_tmem(const AttnParams& p, const AttnSplit& split, cudaStream_t s);
// Tensor cores by mma.sync: tiles of 16 query rows.
AttnSplit attention_short_split(const AttnParams& p, void* workspace);
int launch_attention_short(const AttnParams& p, const AttnSplit& split, cudaStream_t s);
int attention_status(int* out);
int* attention_status_word();

}  // namespace sacq
