// The norms behind and before a block with its gate and residual, and the 8-bit rows of the projections that follow, in
// one pass over a row:
//   b = norm_post(branch) * post_weight + post_bias          (post_norm; else b = branch)
//   r = residual_scale * residual + gate * b                 -> r_out, bf16
//   h = norm(r) * weight + bias,  h = h (1 + mod_scale) + mod_shift
//   -> h_out, bf16, and / or scale = max|h| / 448, q = e4m3(h / scale)
// with norm(x) = x / sqrt(mean(x^2) + eps) ("rms") or (x - mean) / sqrt(var + eps) ("layer"), var around the mean.
// Everything between the loads and the stores is fp32; each result is rounded once, from the fp32 row (h and q from r
// before its rounding to bf16).
//
// 7 bytes per element with 8-bit rows.  A CTA holds its row in registers, in pairs for the f32x2 operations.  Many rows: a CTA
// takes row after row, and bulk copies bring the next ones into shared memory meanwhile (the sums of a row are three to
// five barriers, during which a CTA that loads its own row asks for nothing).  Few rows, and rows that are not 16-byte aligned: a
// CTA per row, straight from memory, everything asked for at once.
// 19,200 x 2,048, RMS on both sides, a gate of each request's own, 8-bit rows: 67 us, 4.1 TB/s, 63 % of the measured copy rate;
// 31 instructions per element (10 unpack bf16) fill 55 % of the issue slots of 16 warps, more warps do not fit the
// registers.  A warp per row, loading it itself: 180 us; a CTA per row, likewise: 98; teams of a CTA with named barriers: 82;
// two rows at a time: 73 to 89.
#include "common.cuh"
#include "encode.cuh"
#include "umma.cuh"

namespace sacq {

namespace {

using umma::mbar_init;
using umma::smem_u32;

constexpr int kSlots = 2;         // rows of a CTA in shared memory

struct NormParams {
  const uint16_t *branch, *residual;
  int64_t branch_pitch, residual_pitch;
  const uint16_t *post_weight, *post_bias, *gate, *weight, *bias, *mod_scale, *mod_shift;
  const int32_t* vector_rows;     // row of gate, mod_scale and mod_shift that a row of x takes; null: they are vectors
  int64_t vectors;
  int64_t M, K;
  int post, norm;                 // SACQ_NORM_*
  float eps, residual_scale, inv_count;
  uint16_t *r_out, *h_out;        // [M, K]; h_out may be null
  uint8_t* q;                     // [M, K] or null
  float* scale;
};

// 1 / sqrt(v): the approximation and one step of Newton's iteration, which leaves an error of an ulp.
__device__ __forceinline__ float inverse_root(float v) {
  const float y = rsqrtf(v);
  const float better = fmaf(0.5f * y, fmaf(-v * y, y, 1.0f), y);
  return v > 0.f && v < INFINITY ? better : y;
}

// Sums over the threads of a CTA: a warp's shuffles and one word per warp in shared memory, new words for each sum of a row.
struct RowReduce {
  float* words;
  int stride;
  template <typename V, typename F>
  __device__ __forceinline__ V all(V v, F f) {
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    V* const w = reinterpret_cast<V*>(words);
    if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = v;
    __syncthreads();
    v = w[0];
    for (int i = 1; i < warps; ++i) v = f(v, w[i]);
    words += stride;
    return v;
  }
  __device__ __forceinline__ float sum(float v) { return all(warp_sum(v), [](float x, float y) { return x + y; }); }
  __device__ __forceinline__ uint32_t most(uint32_t v) { return all(warp_max_bits(v), [](uint32_t x, uint32_t y) { return max(x, y); }); }
};

// What a row is made of.
enum { kPostWeight, kPostBias, kGate, kWeight, kBias, kModScale, kModShift, kVectors };
struct RowInputs {
  const uint16_t *branch, *residual;
  const uint16_t* vec[kVectors];  // null: none
  const uint16_t* own[kVectors];  // vectors of the row's own, in memory where vec lies in shared memory (gate, mod_scale, mod_shift)
  bool outside;                   // its vector row lies outside of the table: the whole row becomes NaN
};

// Row m.  CH chunks of 8 elements per thread; VEC: a chunk is 16 bytes, and K a multiple of 8; else its elements are a
// row's width of threads apart, at any alignment.  RING: inputs and vectors lie in shared memory, but for vectors of the row's own, and
// `read` is called when all threads have read the inputs.  Else everything is loaded up front, if a thread has one chunk: one
// latency instead of one behind each sum.  FULL: K is 8 CH elements of every thread.
template <int CH, bool VEC, bool RING, bool FULL, typename Read>
__device__ __forceinline__ void norm_row(const NormParams& p, int64_t m, const RowInputs& in, RowReduce& reduce, Read read) {
  constexpr bool EARLY = !RING && CH == 1;
  const int T = blockDim.x, tid = threadIdx.x, K = (int)p.K;
  auto begin = [&](int c) { return (c * T + tid) * 8; };                          // VEC: first element of a chunk
  auto at = [&](int c, int j) { return VEC ? begin(c) + j : (c * 8 + j) * T + tid; };
  auto inside = [&](int c, int j) { return FULL || at(c, j) < K; };
  auto fetch = [&](const uint16_t* row, int c) {
    if constexpr (FULL) return *reinterpret_cast<const uint4*>(row + begin(c));
    uint4 u = make_uint4(0, 0, 0, 0);
    if constexpr (VEC) {
      if (begin(c) < K) u = *reinterpret_cast<const uint4*>(row + begin(c));
    } else {
      uint32_t* w = &u.x;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (inside(c, j)) w[j >> 1] |= (uint32_t)row[at(c, j)] << (16 * (j & 1));
    }
    return u;
  };
  auto pair = [&](const uint4& u, int j) {
    const uint32_t w = (&u.x)[j];
    return f32x2(pair_lo(w), pair_hi(w));
  };
  auto store = [&](uint16_t* row, int c, const uint64_t (&v)[4]) {
    uint4 u;
    uint32_t* w = &u.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      halves_of(v[j], a, b);
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (VEC) {
      if (FULL || begin(c) < K) *reinterpret_cast<uint4*>(row + begin(c)) = u;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (inside(c, j)) row[at(c, j)] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  };
  // elements behind the row's end stay zero
  auto only_inside = [&](uint64_t v, int c, int j) {
    float a, b;
    if constexpr (FULL) return v;
    halves_of(v, a, b);
    return f32x2(inside(c, 2 * j) ? a : 0.f, inside(c, 2 * j + 1) ? b : 0.f);
  };
  uint64_t x[CH][4];
  auto each = [&](auto f) {                  // f(chunk, pair)
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) f(c, j);
  };
  auto total = [&](uint64_t v) {
    float a, b;
    halves_of(v, a, b);
    return reduce.sum(a + b);
  };
  // x -> norm(x) without its weight
  auto standardize = [&](int kind) {
    if (kind == SACQ_NORM_LAYER) {
      uint64_t sum = f32x2(0.f, 0.f);
      each([&](int c, int j) { sum = add2(sum, x[c][j]); });
      const float mean = total(sum) * p.inv_count;
      const uint64_t minus = f32x2(-mean, -mean);
      each([&](int c, int j) { x[c][j] = only_inside(add2(x[c][j], minus), c, j); });
    }
    uint64_t sq = f32x2(0.f, 0.f);
    each([&](int c, int j) { sq = fma2(x[c][j], x[c][j], sq); });
    const float rstd = inverse_root(fmaf(total(sq), p.inv_count, p.eps));
    const uint64_t both = f32x2(rstd, rstd);
    each([&](int c, int j) { x[c][j] = mul2(x[c][j], both); });
  };

  uint4 early_residual, early[EARLY ? kVectors : 1];
  uint4 gate[RING ? CH : 1];                 // one of the row's own comes from L2: asked for in front of the first sum
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint4 u = fetch(in.branch, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[c][j] = pair(u, j);
    if constexpr (RING)
      if (in.own[kGate] != nullptr) gate[c] = fetch(in.own[kGate], c);
  }
  if constexpr (EARLY) {
    early_residual = fetch(in.residual, 0);
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (in.vec[v] != nullptr) early[v] = fetch(in.vec[v], 0);
  }
  // f(chunk, pair, its pair of vector v)
  auto with = [&](int v, auto f) {
    if (in.vec[v] != nullptr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint4 u;
        if constexpr (EARLY) u = early[v]; else u = fetch(in.vec[v], c);
#pragma unroll
        for (int j = 0; j < 4; ++j) f(c, j, pair(u, j));
      }
    } else if (RING && in.own[v] != nullptr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const uint4 u = v == kGate ? gate[RING ? c : 0] : fetch(in.own[v], c);
#pragma unroll
        for (int j = 0; j < 4; ++j) f(c, j, pair(u, j));
      }
    }
  };
  auto times = [&](int v) { with(v, [&](int c, int j, uint64_t w) { x[c][j] = mul2(x[c][j], w); }); };
  auto plus = [&](int v) { with(v, [&](int c, int j, uint64_t w) { x[c][j] = add2(x[c][j], w); }); };

  if (p.post != SACQ_NORM_NONE) {
    standardize(p.post);
    times(kPostWeight);
    plus(kPostBias);
  }
  times(kGate);
  const uint64_t res_scale = f32x2(p.residual_scale, p.residual_scale);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    uint4 u;
    if constexpr (EARLY) u = early_residual; else u = fetch(in.residual, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[c][j] = fma2(pair(u, j), res_scale, x[c][j]);
  }
  if (in.outside) {
    const float nan = __uint_as_float(0x7fc00000u);
    each([&](int c, int j) { x[c][j] = only_inside(f32x2(nan, nan), c, j); });
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) store(p.r_out + m * K, c, x[c]);
  standardize(p.norm);                       // behind its barrier all threads have read the inputs
  read();
  times(kWeight);
  plus(kBias);
  if (p.mod_scale != nullptr) {
    const uint64_t one = f32x2(1.f, 1.f);
    with(kModScale, [&](int c, int j, uint64_t w) { x[c][j] = mul2(x[c][j], add2(w, one)); });
    plus(kModShift);
  }
  if (p.h_out != nullptr) {
#pragma unroll
    for (int c = 0; c < CH; ++c) store(p.h_out + m * K, c, x[c]);
  }
  if (p.q == nullptr) return;
  // the maximum drops a NaN: `odd` becomes one if an element is not finite
  float high = 0.f;
  uint64_t odd = f32x2(0.f, 0.f);
  each([&](int c, int j) {
    float a, b;
    halves_of(x[c][j], a, b);
    high = fmaxf(high, fmaxf(fabsf(a), fabsf(b)));
    odd = fma2(x[c][j], f32x2(0.f, 0.f), odd);
  });
  uint32_t top = __float_as_uint(high);
  float odd0, odd1;
  halves_of(odd, odd0, odd1);
  if (odd0 + odd1 != 0.f)
    each([&](int c, int j) {
      float a, b;
      halves_of(x[c][j], a, b);
      top = absmax_bits(absmax_bits(top, a), b);
    });
  const float big = __uint_as_float(reduce.most(top));
  const float scale = big > 0.f ? big * (1.0f / 448.0f) : 1.0f;       // a NaN row keeps 1, as in quantize_rows
  if (tid == 0) p.scale[m] = scale;
  // h / scale as h (r1 + r2), the reciprocal in two parts: an ordinary scale is one that leaves both ordinary
  const bool ordinary = scale > 8.3e-25f && scale < 1.2e24f;
  const float first = ordinary ? __fdividef(1.0f, scale) : 0.f, second = fmaf(-scale, first, 1.0f) * first;
  uint8_t* const qrow = p.q + m * K;
  const uint64_t r1 = f32x2(first, first), r2 = f32x2(second, second);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    uint32_t two[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      if (ordinary) {
        halves_of(quotient2(x[c][j], r1, r2), a, b);
      } else {
        halves_of(x[c][j], a, b);
        a = __fdiv_rn(a, scale);
        b = __fdiv_rn(b, scale);
      }
      two[j] = float2_to_e4m3x2(sat448(a), sat448(b));
    }
    if constexpr (VEC) {
      if (FULL || begin(c) < K) *reinterpret_cast<uint2*>(qrow + begin(c)) = make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (inside(c, j)) qrow[at(c, j)] = (uint8_t)(two[j >> 1] >> (8 * (j & 1)));
    }
  }
}

// A CTA per row.
template <int CH, bool VEC, int T>
__global__ void __launch_bounds__(T) residual_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[5][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  RowReduce reduce{&red[0][0], 32};
  const int64_t m = blockIdx.x;
  RowInputs in;
  const int32_t v = p.vector_rows == nullptr ? 0 : p.vector_rows[m];
  in.outside = v < 0 || v >= p.vectors;
  const int64_t at = in.outside ? 0 : v * p.K;
  auto table = [&](const uint16_t* t) { return t == nullptr ? t : t + at; };
  in.branch = p.branch + m * p.branch_pitch;
  in.residual = p.residual + m * p.residual_pitch;
  in.vec[kPostWeight] = p.post_weight;
  in.vec[kPostBias] = p.post_bias;
  in.vec[kWeight] = p.weight;
  in.vec[kBias] = p.bias;
  in.vec[kGate] = table(p.gate);
  in.vec[kModScale] = table(p.mod_scale);
  in.vec[kModShift] = table(p.mod_shift);
  norm_row<CH, VEC, false, false>(p, m, in, reduce, [] {});
}

// A CTA for the rows blockIdx.x, blockIdx.x + gridDim.x, ...  In shared memory: the vectors that all rows take, and two slots
// with branch and residual of a row.
template <int CH, bool FULL>
__global__ void __launch_bounds__(256) residual_norm_rows_kernel(const __grid_constant__ NormParams p, int* status) {
  extern __shared__ __align__(16) uint16_t rows[];
  __shared__ float red[2][5][8];                      // of two rows in turn: a word is used again behind the next row's barriers
  __shared__ __align__(8) uint64_t full[kSlots];
  __shared__ int abort_flag;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int K = (int)p.K;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(smem_u32(&full[s]), 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  RowInputs in;
  const bool tables = p.vector_rows != nullptr;
  const uint16_t* const vectors[kVectors] = {p.post_weight, p.post_bias, tables ? nullptr : p.gate, p.weight, p.bias,
                                             tables ? nullptr : p.mod_scale, tables ? nullptr : p.mod_shift};
  int used = 0;
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    in.vec[v] = vectors[v] == nullptr ? nullptr : rows + used;
    in.own[v] = nullptr;
    if (vectors[v] != nullptr) used += K;
  }
  const uint32_t bytes = (uint32_t)K * 2;
  auto copy = [&](int64_t m, int s, int extra) {      // by one thread
    const uint32_t bar = smem_u32(&full[s]), at = smem_u32(rows + used + s * 2 * K);
    umma::mbar_arrive_expect_tx(bar, 2 * bytes + extra);
    umma::bulk_load(at, p.branch + m * p.branch_pitch, bytes, bar);
    umma::bulk_load(at + bytes, p.residual + m * p.residual_pitch, bytes, bar);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      const int64_t m = blockIdx.x + (int64_t)s * gridDim.x;
      if (m < p.M) copy(m, s, s == 0 ? used * 2 : 0);
    }
    int off = 0;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (vectors[v] != nullptr) {
        umma::bulk_load(smem_u32(rows + off), vectors[v], bytes, smem_u32(&full[0]));
        off += K;
      }
  }
  int next = tables ? p.vector_rows[blockIdx.x] : 0;  // the vector row is read a row ahead
  uint32_t i = 0;
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x, ++i) {
    const int s = i % kSlots;
    // a wait that runs out leaves through the same barrier in every thread
    if (__syncthreads_or(!umma::mbar_wait(smem_u32(&full[s]), (i / kSlots) & 1, &abort_flag, status))) {
      for (uint32_t c = i; c < i + kSlots; ++c)       // copies in flight land before the CTA leaves
        if (m + (int64_t)(c - i) * gridDim.x < p.M)
          for (int t = 0; t < 100000 && !umma::mbar_try_wait(smem_u32(&full[c % kSlots]), (c / kSlots) & 1); ++t) {}
      return;
    }
    RowReduce reduce{&red[i & 1][0][0], 8};
    in.branch = rows + used + s * 2 * K;
    in.residual = in.branch + K;
    in.outside = false;
    if (tables) {
      in.outside = next < 0 || next >= p.vectors;
      const int64_t v = in.outside ? 0 : (int64_t)next * K;
      in.own[kGate] = p.gate == nullptr ? nullptr : p.gate + v;
      in.own[kModScale] = p.mod_scale == nullptr ? nullptr : p.mod_scale + v;
      in.own[kModShift] = p.mod_shift == nullptr ? nullptr : p.mod_shift + v;
      if (m + gridDim.x < p.M) next = p.vector_rows[m + gridDim.x];
    }
    norm_row<CH, true, true, FULL>(p, m, in, reduce, [&] {
      if (blockDim.x == 32) __syncwarp();
      const int64_t ahead = m + (int64_t)kSlots * gridDim.x;
      if (threadIdx.x == 0 && ahead < p.M) copy(ahead, s, 0);
    });
  }
}

__device__ int g_norm_status;                         // nonzero: a wait ran out

template <bool VEC>
const void* direct_instance(int chunks, unsigned threads) {
  switch (chunks) {
    case 1: return threads <= 512 ? (const void*)residual_norm_kernel<1, VEC, 512> : (const void*)residual_norm_kernel<1, VEC, 1024>;
    case 2: return (const void*)residual_norm_kernel<2, VEC, 1024>;
    case 3: return (const void*)residual_norm_kernel<3, VEC, 1024>;
    case 4: return (const void*)residual_norm_kernel<4, VEC, 1024>;
    default: return nullptr;
  }
}

template <bool FULL>
const void* rows_instance(int chunks) {
  switch (chunks) {
    case 1: return (const void*)residual_norm_rows_kernel<1, FULL>;
    case 2: return (const void*)residual_norm_rows_kernel<2, FULL>;
    case 3: return (const void*)residual_norm_rows_kernel<3, FULL>;
    case 4: return (const void*)residual_norm_rows_kernel<4, FULL>;
    default: return nullptr;
  }
}

}  // namespace

int residual_norm_status(int* out) {
  SACQ_CUDA_TRY(cudaMemcpyFromSymbol(out, g_norm_status, sizeof(int)));
  return SACQ_OK;
}

int launch_residual_norm(const sacq_residual_norm_desc& d, cudaStream_t s) {
  auto al = [](const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; };   // null: aligned
  const int64_t K = d.K;
  const bool vec = K % 8 == 0 && d.branch_pitch % 8 == 0 && d.residual_pitch % 8 == 0 && al(d.branch, 16) && al(d.residual, 16) &&
                   al(d.post_weight, 16) && al(d.post_bias, 16) && al(d.gate, 16) && al(d.weight, 16) && al(d.bias, 16) &&
                   al(d.mod_scale, 16) && al(d.mod_shift, 16) && al(d.residual_out, 16) && al(d.normalized_out, 16) && al(d.q_out, 8);
  NormParams p = {};
  p.branch = static_cast<const uint16_t*>(d.branch);
  p.residual = static_cast<const uint16_t*>(d.residual);
  p.branch_pitch = d.branch_pitch;
  p.residual_pitch = d.residual_pitch;
  p.post_weight = static_cast<const uint16_t*>(d.post_weight);
  p.post_bias = static_cast<const uint16_t*>(d.post_bias);
  p.gate = static_cast<const uint16_t*>(d.gate);
  p.weight = static_cast<const uint16_t*>(d.weight);
  p.bias = static_cast<const uint16_t*>(d.bias);
  p.mod_scale = static_cast<const uint16_t*>(d.mod_scale);
  p.mod_shift = static_cast<const uint16_t*>(d.mod_shift);
  p.vector_rows = d.vector_rows;
  p.vectors = d.vector_rows == nullptr ? 1 : d.vectors;
  p.M = d.M;
  p.K = K;
  p.post = d.post_norm;
  p.norm = d.norm;
  p.eps = d.eps;
  p.residual_scale = d.residual_scale;
  p.inv_count = (float)(1.0 / (double)K);
  p.r_out = static_cast<uint16_t*>(d.residual_out);
  p.h_out = static_cast<uint16_t*>(d.normalized_out);
  p.q = static_cast<uint8_t*>(d.q_out);
  p.scale = d.scale_out;
  const int64_t chunks = (K + 7) / 8;
  const bool many = vec && d.M >= 1024 && chunks <= 4 * 256;
  unsigned threads;
  int per;
  bool full = false;
  int64_t grid = d.M;
  size_t smem = 0;
  if (many) {
    // up to 4 chunks a thread (of 2,048-wide rows one took 99 us, two 68, four 67), as many as leave the fewest elements that are not
    // there; where there are none, nothing is checked
    const int64_t pieces = (chunks + 31) / 32, pieces4 = (pieces + 3) / 4;
    per = (int)((pieces + pieces4 - 1) / pieces4);
    if (chunks % 32 == 0)
      for (int c = 4; c >= 2 && pieces / c <= 8; --c)
        if (pieces % c == 0) {
          per = c;
          break;
        }
    threads = (unsigned)((pieces + per - 1) / per * 32);
    full = chunks == (int64_t)threads * per;
    const int all = (d.post_weight != nullptr) + (d.post_bias != nullptr) + (d.weight != nullptr) + (d.bias != nullptr) +
                    (d.vector_rows ? 0 : (d.gate != nullptr) + 2 * (d.mod_scale != nullptr));
    // as many CTAs as an SM's shared memory holds, of 64 registers a thread
    smem = (size_t)(kSlots * 2 + all) * K * 2;
    int64_t fit = (int64_t)(224 * 1024) / (int64_t)(smem + 2048);
    if (fit > 1024 / threads) fit = 1024 / threads;
    if (fit < 1) fit = 1;
    if (grid > fit * 148) grid = fit * 148;
  } else {
    threads = (unsigned)(chunks >= 1024 ? 1024 : (chunks + 31) / 32 * 32);
    per = (int)((chunks + threads - 1) / threads);
  }
  const void* fn = many ? (full ? rows_instance<true>(per) : rows_instance<false>(per)) : vec ? direct_instance<true>(per, threads) : direct_instance<false>(per, threads);
  if (fn == nullptr) return set_error(SACQ_ERR_UNSUPPORTED, "K=%lld: a row does not fit the registers of a CTA", (long long)K);
  if (grid > 2147483647LL) return set_error(SACQ_ERR_UNSUPPORTED, "M=%lld exceeds the grid limit", (long long)d.M);
  int* status = nullptr;
  if (many) {
    static int* word[64] = {};
    static bool configured[2][5][64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return set_error(SACQ_ERR_UNSUPPORTED, "device %d", dev);
    if (word[dev] == nullptr) {
      void* at = nullptr;
      SACQ_CUDA_TRY(cudaGetSymbolAddress(&at, g_norm_status));
      word[dev] = static_cast<int*>(at);
    }
    status = word[dev];
    if (!configured[full][per][dev]) {
      SACQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
      SACQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      configured[full][per][dev] = true;
    }
  }
  void* args[] = {&p, &status};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
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
