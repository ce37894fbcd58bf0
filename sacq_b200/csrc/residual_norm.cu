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
// 7 bytes per element with 8-bit rows.  A row is held in registers, in pairs for the f32x2 operations.  Many rows: a warp takes row
// after row (up to 2,048 elements; a CTA, wider ones), and bulk copies bring the next one into shared memory meanwhile, its gate from a
// table too.  Few rows, and rows that are not 16-byte aligned: a CTA per row, straight from memory, everything asked for at once.
// 19,200 x 2,048, RMS on both sides, a gate of each request's own, 8-bit rows: 49 us, 5.6 TB/s, 86 % of the measured copy rate.  A CTA per
// row from shared memory: 62 us (what a row costs beside its elements was twice the instructions); a warp per row with two rows ahead, 12
// warps instead of 15: 62; the gate by ordinary loads: 59; without bulk copies a warp per row 180, a CTA 98.  Scalar operations
// instead of pairs: 70 for 62.
#include <type_traits>

#include "common.cuh"
#include "encode.cuh"
#include "umma.cuh"

namespace sacq {

namespace {

using umma::mbar_init;
using umma::smem_u32;

constexpr int kSlots = 2;         // rows of a CTA in shared memory
// Warps of a CTA that take a row each, of up to 256 elements for each of `chunks`: as many as have registers for it (19,200 x 1,536: 20
// warps 37.3 us, 18 39.3; x 512: 28 13.8, 32 15.1, 24 17.0).
__host__ __device__ constexpr int row_warps(int chunks) {
  return chunks <= 2 ? 28 : chunks <= 4 ? 22 : chunks <= 6 ? 20 : 15;
}

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

// The largest of m, |a| and |b|, NaN if one is.
__device__ __forceinline__ float absmax_nan(float m, float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// Sums over the threads of a row: a warp's shuffles and one word per warp in shared memory, new words for each sum of a row.
struct RowReduce {
  float* words;
  int stride, warps;
  template <typename V, typename F>
  __device__ __forceinline__ V all(V v, F f) {
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
  bool late;                      // WARP: vectors that are used behind the norm lie with the inputs
};

// Row m.  CH chunks of 8 elements per thread; VEC: a chunk is 16 bytes, and K a multiple of 8; else its elements are a
// row's width of threads apart, at any alignment.  RING: inputs and vectors lie in shared memory, but for vectors of the row's own, and
// `read` is called when all threads have read the inputs.  Else everything is loaded up front, if a thread has one chunk: one
// latency instead of one behind each sum.  FULL: K is 8 CH elements of every thread.  WARP: a row is a warp's, else a CTA's.  LEAN: root
// mean squares only.
template <int CH, bool VEC, bool RING, bool FULL, bool WARP, bool LEAN, typename Read>
__device__ __forceinline__ void norm_row(const NormParams& p, int64_t m, const RowInputs& in, RowReduce& reduce, Read read) {
  constexpr bool EARLY = !RING && CH == 1;
  const int T = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x, K = (int)p.K;
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
    if (!LEAN && kind == SACQ_NORM_LAYER) {
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
  constexpr bool AHEAD = RING && !WARP;
  uint4 gate[AHEAD ? CH : 1];                 // one of the row's own comes from L2: asked for in front of the first sum
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint4 u = fetch(in.branch, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[c][j] = pair(u, j);
    if constexpr (AHEAD)
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
        const uint4 u = AHEAD && v == kGate ? gate[AHEAD ? c : 0] : fetch(in.own[v], c);
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
  if (!WARP || LEAN || !in.late) read();
  times(kWeight);
  plus(kBias);
  if (!LEAN && p.mod_scale != nullptr) {
    const uint64_t one = f32x2(1.f, 1.f);
    with(kModScale, [&](int c, int j, uint64_t w) { x[c][j] = mul2(x[c][j], add2(w, one)); });
    plus(kModShift);
  }
  if (WARP && !LEAN && in.late) read();      // vectors of the row's own lie with the inputs
  if (p.h_out != nullptr) {
#pragma unroll
    for (int c = 0; c < CH; ++c) store(p.h_out + m * K, c, x[c]);
  }
  if (p.q == nullptr) return;
  float high = 0.f;                          // NaN if an element is, which is more than infinity in bits
  each([&](int c, int j) {
    float a, b;
    halves_of(x[c][j], a, b);
    high = absmax_nan(high, a, b);
  });
  const float big = __uint_as_float(reduce.most(__float_as_uint(high)));
  // scale and quotients as in quantize_rows: a NaN row keeps 1
  const RowDivisor d = scale_of<false>(big);
  if (tid == 0) p.scale[m] = d.s;
  uint8_t* const qrow = p.q + m * K;
  const uint64_t r1 = f32x2(d.r, d.r), r2 = f32x2(d.r2, d.r2);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    uint32_t two[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      if (d.fast) {
        halves_of(quotient2(x[c][j], r1, r2), a, b);
      } else {
        halves_of(x[c][j], a, b);
        a = __fdiv_rn(a, d.s);
        b = __fdiv_rn(b, d.s);
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
  RowReduce reduce{&red[0][0], 32, (int)blockDim.x >> 5};
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
  norm_row<CH, VEC, false, false, false, false>(p, m, in, reduce, [] {});
}

// Rows wider than a warp holds: a CTA for the rows blockIdx.x, blockIdx.x + gridDim.x, ...  In shared memory: the vectors that all rows take, and two slots
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
    RowReduce reduce{&red[i & 1][0][0], 8, (int)blockDim.x >> 5};
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
    norm_row<CH, true, true, FULL, false, false>(p, m, in, reduce, [&] {
      const int64_t ahead = m + (int64_t)kSlots * gridDim.x;
      if (threadIdx.x == 0 && ahead < p.M) copy(ahead, s, 0);
    });
  }
}

// The same with a warp for each row: no barrier, and what a row costs beside its elements (three sums, the scale, the copies) is done by
// one warp.  In shared memory: the vectors that all rows take, once, and room for one row of each warp with its own vectors, which is
// asked for as soon as the last one is in registers.  LEAN: root mean squares, weights and a gate, nothing else (62.5 us became 59.7).
template <int CH, bool FULL, bool LEAN, bool TABLES>
__global__ void __launch_bounds__(row_warps(CH) * 32) residual_norm_warps_kernel(const __grid_constant__ NormParams p, int* status) {
  extern __shared__ __align__(16) uint16_t rows[];
  __shared__ __align__(8) uint64_t full[row_warps(CH)];
  __shared__ __align__(8) uint64_t vectors_full;
  __shared__ int abort_flag;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int K = (int)p.K, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (threadIdx.x == 0) {
    for (int w = 0; w < warps; ++w) mbar_init(smem_u32(&full[w]), 1);
    mbar_init(smem_u32(&vectors_full), 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  RowInputs in;
  const uint16_t* const vectors[kVectors] = {p.post_weight, LEAN ? nullptr : p.post_bias, TABLES ? nullptr : p.gate, p.weight,
                                             LEAN ? nullptr : p.bias, LEAN || TABLES ? nullptr : p.mod_scale,
                                             LEAN || TABLES ? nullptr : p.mod_shift};
  int used = 0;
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    in.vec[v] = vectors[v] == nullptr ? nullptr : rows + used;
    in.own[v] = nullptr;
    if (vectors[v] != nullptr) used += K;
  }
  // a row's inputs, and its own vectors where there are tables of them
  const uint16_t* const table[3] = {TABLES ? p.gate : nullptr, LEAN || !TABLES ? nullptr : p.mod_scale, LEAN || !TABLES ? nullptr : p.mod_shift};
  constexpr int kOwn[3] = {kGate, kModScale, kModShift};
  int parts = 2;
#pragma unroll
  for (int v = 0; v < 3; ++v) parts += table[v] != nullptr;
  const uint32_t bytes = (uint32_t)K * 2;
  uint16_t* const slot = rows + used + warp * parts * K;
  in.branch = slot;
  in.residual = slot + K;
  in.late = table[1] != nullptr;
#pragma unroll
  for (int v = 0, at = 2; v < 3; ++v)
    if (table[v] != nullptr) in.vec[kOwn[v]] = slot + at++ * K;
  auto inside = [&](int v) { return v >= 0 && v < p.vectors; };
  auto copy = [&](int64_t m, int vector_row) {        // by one lane
    const uint32_t bar = smem_u32(&full[warp]);
    uint32_t at = smem_u32(slot);
    umma::mbar_arrive_expect_tx(bar, parts * bytes);
    umma::bulk_load(at, p.branch + m * p.branch_pitch, bytes, bar);
    umma::bulk_load(at += bytes, p.residual + m * p.residual_pitch, bytes, bar);
    const int64_t v0 = inside(vector_row) ? (int64_t)vector_row * K : 0;
#pragma unroll
    for (int v = 0; v < 3; ++v)
      if (table[v] != nullptr) umma::bulk_load(at += bytes, table[v] + v0, bytes, bar);
  };
  const int64_t first = (int64_t)warp * gridDim.x + blockIdx.x, step = (int64_t)warps * gridDim.x;
  auto vector_row = [&](int64_t m) { return TABLES && m < p.M ? p.vector_rows[m] : 0; };
  int now = vector_row(first), next = vector_row(first + step);
  if (lane == 0) {
    if (first < p.M) copy(first, now);
    if (warp == 0) {
      umma::mbar_arrive_expect_tx(smem_u32(&vectors_full), (uint32_t)used * 2);
      int off = 0;
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
        if (vectors[v] != nullptr) {
          umma::bulk_load(smem_u32(rows + off), vectors[v], bytes, smem_u32(&vectors_full));
          off += K;
        }
    }
  }
  __syncwarp();
  bool ok = umma::mbar_wait_warp(smem_u32(&vectors_full), 0, &abort_flag, status);
  uint32_t i = 0;
  int64_t m = first;
  for (; ok && m < p.M; m += step, ++i) {
    ok = umma::mbar_wait_warp(smem_u32(&full[warp]), i & 1, &abort_flag, status);
    if (!ok) break;
    RowReduce reduce{nullptr, 0, 1};
    in.outside = !inside(now);
    const int after = vector_row(m + 2 * step);
    norm_row<CH, true, true, FULL, true, LEAN>(p, m, in, reduce, [&] {
      __syncwarp();
      if (lane == 0 && m + step < p.M) copy(m + step, next);
    });
    now = next;
    next = after;
  }
  if (!ok) {                                          // copies in flight land before the CTA leaves
    for (int t = 0; t < 100000 && !umma::mbar_try_wait(smem_u32(&vectors_full), 0); ++t) {}
    if (m < p.M)
      for (int t = 0; t < 100000 && !umma::mbar_try_wait(smem_u32(&full[warp]), i & 1); ++t) {}
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

template <bool FULL, bool LEAN, bool TABLES>
const void* warps_instance(int chunks) {
  switch (chunks) {
    case 1: return (const void*)residual_norm_warps_kernel<1, FULL, LEAN, TABLES>;
    case 2: return (const void*)residual_norm_warps_kernel<2, FULL, LEAN, TABLES>;
    case 3: return (const void*)residual_norm_warps_kernel<3, FULL, LEAN, TABLES>;
    case 4: return (const void*)residual_norm_warps_kernel<4, FULL, LEAN, TABLES>;
    case 5: return (const void*)residual_norm_warps_kernel<5, FULL, LEAN, TABLES>;
    case 6: return (const void*)residual_norm_warps_kernel<6, FULL, LEAN, TABLES>;
    case 7: return (const void*)residual_norm_warps_kernel<7, FULL, LEAN, TABLES>;
    case 8: return (const void*)residual_norm_warps_kernel<8, FULL, LEAN, TABLES>;
    default: return nullptr;
  }
}

template <bool FULL>
const void* rows_instance(int chunks) {
  switch (chunks) {
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
  // 900 rows of 2,048 take 5.6 us either way, 600 5.5 (many) and 4.7, 1,200 6.2 and 7.2
  const bool many = vec && d.M >= 1024 && chunks <= 4 * 256, warps = many && chunks <= 8 * 32;
  const int all = (d.post_weight != nullptr) + (d.post_bias != nullptr) + (d.weight != nullptr) + (d.bias != nullptr) +
                  (d.vector_rows ? 0 : (d.gate != nullptr) + 2 * (d.mod_scale != nullptr));
  const bool lean = d.norm == SACQ_NORM_RMS && d.post_norm != SACQ_NORM_LAYER && d.post_bias == nullptr && d.bias == nullptr && d.mod_scale == nullptr;
  unsigned threads;
  int per;
  bool full = false;
  int64_t grid = d.M;
  size_t smem = 0;
  if (warps) {
    per = (int)((chunks + 31) / 32);
    full = chunks == 32 * per;
    const int own = d.vector_rows ? (d.gate != nullptr) + 2 * (d.mod_scale != nullptr) : 0;
    int64_t fit = ((int64_t)(220 * 1024) - all * K * 2) / ((2 + own) * K * 2);
    if (fit > row_warps(per)) fit = row_warps(per);
    threads = (unsigned)fit * 32;
    smem = (size_t)(fit * (2 + own) + all) * K * 2;
    if (grid > device_sms()) grid = device_sms();
  } else if (many) {
    // up to 4 chunks a thread, as many as leave the fewest elements that are not there; where there are none, nothing is checked
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
    // as many CTAs as an SM's shared memory holds, of 64 registers a thread
    smem = (size_t)(kSlots * 2 + all) * K * 2;
    int64_t fit = (int64_t)(224 * 1024) / (int64_t)(smem + 2048);
    if (fit > 1024 / threads) fit = 1024 / threads;
    if (fit < 1) fit = 1;
    if (grid > fit * device_sms()) grid = fit * device_sms();
  } else {
    threads = (unsigned)(chunks >= 1024 ? 1024 : (chunks + 31) / 32 * 32);
    per = (int)((chunks + threads - 1) / threads);
  }
  const bool tables = d.vector_rows != nullptr;
  auto by_warps = [&](auto f, auto l) {
    return tables ? warps_instance<decltype(f)::value, decltype(l)::value, true>(per) : warps_instance<decltype(f)::value, decltype(l)::value, false>(per);
  };
  const std::true_type yes;
  const std::false_type no;
  const void* fn = warps ? (full ? (lean ? by_warps(yes, yes) : by_warps(yes, no)) : (lean ? by_warps(no, yes) : by_warps(no, no)))
                         : many ? (full ? rows_instance<true>(per) : rows_instance<false>(per)) : vec ? direct_instance<true>(per, threads) : direct_instance<false>(per, threads);
  if (fn == nullptr) return set_error(SACQ_ERR_UNSUPPORTED, "K=%lld: a row does not fit the registers of a CTA", (long long)K);
  if (grid > 2147483647LL) return set_error(SACQ_ERR_UNSUPPORTED, "M=%lld exceeds the grid limit", (long long)d.M);
  int* status = nullptr;
  if (many) {
    static int* word[64] = {};
    static bool configured[2][2][2][2][9][64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return set_error(SACQ_ERR_UNSUPPORTED, "device %d", dev);
    if (word[dev] == nullptr) {
      void* at = nullptr;
      SACQ_CUDA_TRY(cudaGetSymbolAddress(&at, g_norm_status));
      word[dev] = static_cast<int*>(at);
    }
    status = word[dev];
    if (!configured[warps][tables][lean][full][per][dev]) {
      SACQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
      SACQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
      configured[warps][tables][lean][full][per][dev] = true;
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
