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
// Bound by memory: 7 bytes per element with 8-bit rows.  The row stays in registers, 8 elements per thread and chunk: a
// warp takes a whole row where there are many (its sums are shuffles, and 8 KB of loads per warp are in flight),
// else a CTA does, one chunk per thread where it can.
#include "common.cuh"
#include "encode.cuh"

namespace sacq {

namespace {

struct NormParams {
  const uint16_t *branch, *residual;
  int64_t branch_pitch, residual_pitch;
  const uint16_t *post_weight, *post_bias, *gate, *weight, *bias, *mod_scale, *mod_shift;
  const int32_t* vector_rows;     // row of gate, mod_scale and mod_shift that a row of x takes; null: they are vectors
  int64_t vectors;
  int64_t M, K;
  int post, norm;                 // SACQ_NORM_*
  float eps, residual_scale;
  uint16_t *r_out, *h_out;        // [M, K]; h_out may be null
  uint8_t* q;                     // [M, K] or null
  float* scale;
};

// Sums over the threads of a row: a warp's shuffles, and for a CTA's row one word per warp in shared memory, a new slot
// for each sum.
template <bool CTA>
struct RowReduce {
  float (*slot)[32];
  int next = 0;
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    if constexpr (!CTA) return v;
    float* s = slot[next++];
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += s[i];
    return t;
  }
  __device__ __forceinline__ uint32_t most(uint32_t v) {
    v = warp_max_bits(v);
    if constexpr (!CTA) return v;
    float* s = slot[next++];
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = __uint_as_float(v);
    __syncthreads();
    uint32_t t = 0u;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t = max(t, __float_as_uint(s[i]));
    return t;
  }
};

// CH chunks of 8 elements per thread.  VEC: a chunk is 16 bytes, and K a multiple of 8; else its elements are a
// row's width of threads apart, at any alignment.
template <int CH, bool CTA, bool VEC>
__global__ void __launch_bounds__(CTA ? 1024 : 128)
residual_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float red[5][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int T = CTA ? blockDim.x : 32, tid = CTA ? threadIdx.x : threadIdx.x & 31;
  const int64_t m = CTA ? blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (!CTA && m >= p.M) return;
  const int K = (int)p.K;
  RowReduce<CTA> reduce{red};

  auto begin = [&](int c) { return (c * T + tid) * 8; };                          // VEC: first element of a chunk
  auto at = [&](int c, int j) { return VEC ? begin(c) + j : (c * 8 + j) * T + tid; };
  auto load = [&](const uint16_t* row, int c, float (&v)[8]) {
    if constexpr (VEC) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (begin(c) < K) u = *reinterpret_cast<const uint4*>(row + begin(c));
      const uint32_t* w = &u.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = pair_lo(w[j]);
        v[2 * j + 1] = pair_hi(w[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = at(c, j) < K ? bf16_bits_to_float(row[at(c, j)]) : 0.f;
    }
  };
  auto store = [&](uint16_t* row, int c, const float (&v)[8]) {
    if constexpr (VEC) {
      if (begin(c) >= K) return;
      uint4 u;
      uint32_t* w = &u.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(row + begin(c)) = u;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(c, j) < K) row[at(c, j)] = float_to_bf16_bits(v[j]);
    }
  };
  const float count = (float)K;
  // x -> x - mean (layer), and 1 / sqrt of the mean square + eps
  auto standardize = [&](float (&x)[CH][8], int kind) {
    if (kind == SACQ_NORM_LAYER) {
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += x[c][j];
      const float mean = reduce.sum(sum) / count;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[c][j] = at(c, j) < K ? x[c][j] - mean : 0.f;
    }
    float sq = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(x[c][j], x[c][j], sq);
    return 1.0f / sqrtf(reduce.sum(sq) / count + p.eps);
  };

  float x[CH][8], v[8];
#pragma unroll
  for (int c = 0; c < CH; ++c) load(p.branch + m * p.branch_pitch, c, x[c]);
  float res[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) load(p.residual + m * p.residual_pitch, c, res[c]);
  // a vector row outside of its table: the whole row becomes NaN
  int64_t vrow = 0;
  float poison = 0.f;
  if (p.vector_rows != nullptr) {
    vrow = p.vector_rows[m];
    if (vrow < 0 || vrow >= p.vectors) {
      vrow = 0;
      poison = __uint_as_float(0x7fc00000u);
    }
    vrow *= K;
  }
  if (p.post != SACQ_NORM_NONE) {
    const float rstd = standardize(x, p.post);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[c][j] *= rstd;
      if (p.post_weight != nullptr) {
        load(p.post_weight, c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[c][j] *= v[j];
      }
      if (p.post_bias != nullptr) {
        load(p.post_bias, c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[c][j] += v[j];
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (p.gate != nullptr) {
      load(p.gate + vrow, c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[c][j] *= v[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[c][j] = at(c, j) < K ? fmaf(p.residual_scale, res[c][j], x[c][j]) + poison : 0.f;
    store(p.r_out + m * K, c, x[c]);
  }
  const float rstd = standardize(x, p.norm);
  uint32_t mx = 0u;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[c][j] *= rstd;
    if (p.weight != nullptr) {
      load(p.weight, c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[c][j] *= v[j];
    }
    if (p.bias != nullptr) {
      load(p.bias, c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[c][j] += v[j];
    }
    if (p.mod_scale != nullptr) {
      float t[8];
      load(p.mod_scale + vrow, c, v);
      load(p.mod_shift + vrow, c, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[c][j] = fmaf(x[c][j], 1.0f + v[j], t[j]);
    }
    if (p.h_out != nullptr) store(p.h_out + m * K, c, x[c]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at(c, j) < K) mx = absmax_bits(mx, x[c][j]);
  }
  if (p.q == nullptr) return;
  const RowDivisor d = scale_of<false>(__uint_as_float(reduce.most(mx)));
  if (tid == 0) p.scale[m] = d.s;
  uint8_t* qrow = p.q + m * K;
  const uint64_t r = f32x2(d.r, d.r), r2 = f32x2(d.r2, d.r2);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    uint32_t two[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = x[c][2 * j], b = x[c][2 * j + 1];
      if (d.fast) halves_of(quotient2(f32x2(a, b), r, r2), a, b);
      else { a = __fdiv_rn(a, d.s); b = __fdiv_rn(b, d.s); }
      two[j] = float2_to_e4m3x2(sat448(a), sat448(b));
    }
    if constexpr (VEC) {
      if (begin(c) < K) *reinterpret_cast<uint2*>(qrow + begin(c)) = make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(c, j) < K) qrow[at(c, j)] = (uint8_t)(two[j >> 1] >> (8 * (j & 1)));
    }
  }
}

template <bool CTA, bool VEC>
const void* instance(int chunks) {
  switch (chunks) {
    case 1: return (const void*)residual_norm_kernel<1, CTA, VEC>;
    case 2: return (const void*)residual_norm_kernel<2, CTA, VEC>;
    case 3: return (const void*)residual_norm_kernel<3, CTA, VEC>;
    case 4: return (const void*)residual_norm_kernel<4, CTA, VEC>;
    case 5: return CTA ? nullptr : (const void*)residual_norm_kernel<CTA ? 1 : 5, CTA, VEC>;
    case 6: return CTA ? nullptr : (const void*)residual_norm_kernel<CTA ? 1 : 6, CTA, VEC>;
    case 7: return CTA ? nullptr : (const void*)residual_norm_kernel<CTA ? 1 : 7, CTA, VEC>;
    case 8: return CTA ? nullptr : (const void*)residual_norm_kernel<CTA ? 1 : 8, CTA, VEC>;
    default: return nullptr;
  }
}

}  // namespace

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
  p.vectors = d.vectors;
  p.M = d.M;
  p.K = K;
  p.post = d.post_norm;
  p.norm = d.norm;
  p.eps = d.eps;
  p.residual_scale = d.residual_scale;
  p.r_out = static_cast<uint16_t*>(d.residual_out);
  p.h_out = static_cast<uint16_t*>(d.normalized_out);
  p.q = static_cast<uint8_t*>(d.q_out);
  p.scale = d.scale_out;
  const int64_t chunks = (K + 7) / 8;
  const bool warp_rows = d.M >= 1024 && chunks <= 8 * 32;
  unsigned threads = 128;
  int per = (int)((chunks + 31) / 32);
  if (!warp_rows) {
    threads = (unsigned)(chunks >= 1024 ? 1024 : (chunks + 31) / 32 * 32);
    per = (int)((chunks + threads - 1) / threads);
  }
  const void* fn = warp_rows ? (vec ? instance<false, true>(per) : instance<false, false>(per))
                             : (vec ? instance<true, true>(per) : instance<true, false>(per));
  if (fn == nullptr) return set_error(SACQ_ERR_UNSUPPORTED, "K=%lld: a row does not fit the registers of a CTA", (long long)K);
  const int64_t grid = warp_rows ? (d.M + 3) / 4 : d.M;
  if (grid > 2147483647LL) return set_error(SACQ_ERR_UNSUPPORTED, "M=%lld exceeds the grid limit", (long long)d.M);
  void* args[] = {&p};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
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
