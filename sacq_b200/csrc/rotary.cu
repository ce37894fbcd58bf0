// Rotary positions of query and key heads, in one launch:
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i],  both times `amplitude`
// for the rotary_dim / 2 pairs of every head; what lies behind rotary_dim is copied.  A pair is (x[i], x[i + R/2])
// ("half") or (x[2i], x[2i + 1]) ("interleaved").
//
// Angles: a position of 10^6 times a frequency near 1 is right to 0.06 radians in fp32, so the product is made in
// double, in turns (inv_freq / 2 pi), reduced to half a turn either way there, and only then rounded: the
// rounding that is left is 2^-26 turns.  They are the same for all heads, so a CTA makes those of its tokens once, in
// shared memory, between its loads and its stores.
//
// Bound by memory: 4 bytes per element.  A thread holds what it loads (16-byte chunks, of "half" both of a pair) in
// registers while the angles are made.
#include "common.cuh"

namespace sacq {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;                       // per thread and step: loads in flight

struct RotaryParams {
  sacq_head_rows x[2];                          // query heads, key heads
  const void* positions;
  const double* inv_freq;
  int64_t tokens;
  int dim, half;                                // head dim; rotated pairs
  int per_head;                                 // units of a head: turned ones first, then copied ones
  int turned;
  int per_token;                                // units of a token, both tensors
  int tokens_per_cta;
  float amplitude;
  bool wide_positions;
};

__device__ __forceinline__ float2 turn_of(double position, double inv_freq, float amplitude) {
  const double t = position * (inv_freq * 0.15915494309189533577);   // turns
  float s, c;
  sincospif(2.0f * (float)(t - rint(t)), &s, &c);
  return make_float2(c * amplitude, s * amplitude);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight pairs: a in u, b in v ("half").
__device__ __forceinline__ void turn_half(uint4& u, uint4& v, const float2* cs) {
  uint32_t* a = &u.x;
  uint32_t* b = &v.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 c0 = cs[2 * j], c1 = cs[2 * j + 1];
    const float a0 = __uint_as_float(a[j] << 16), a1 = __uint_as_float(a[j] & 0xffff0000u);
    const float b0 = __uint_as_float(b[j] << 16), b1 = __uint_as_float(b[j] & 0xffff0000u);
    a[j] = pack2(a0 * c0.x - b0 * c0.y, a1 * c1.x - b1 * c1.y);
    b[j] = pack2(b0 * c0.x + a0 * c0.y, b1 * c1.x + a1 * c1.y);
  }
}

// Four neighbouring pairs ("interleaved").
__device__ __forceinline__ void turn_neighbours(uint4& u, const float2* cs) {
  uint32_t* w = &u.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = __uint_as_float(w[j] << 16), b = __uint_as_float(w[j] & 0xffff0000u);
    w[j] = pack2(a * cs[j].x - b * cs[j].y, b * cs[j].x + a * cs[j].y);
  }
}

// VEC: units of 16-byte chunks ("half": two of them where turned); else of single pairs and elements, at any alignment.
template <bool HALF, bool VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 turns[];             // [tokens_per_cta][half]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t first = (int64_t)blockIdx.x * p.tokens_per_cta;
  const int here = (int)min((int64_t)p.tokens_per_cta, p.tokens - first);
  const int units = here * p.per_token;

  struct Unit {
    const uint16_t* src;
    uint16_t* dst;
    int at, token;                              // unit of its head, token of the CTA
  };
  auto unit_of = [&](int u) {
    Unit r;
    r.token = u / p.per_token;
    u -= r.token * p.per_token;
    int head = u / p.per_head;
    r.at = u - head * p.per_head;
    const bool key = head >= p.x[0].heads;
    if (key) head -= p.x[0].heads;
    const sacq_head_rows& x = p.x[key];
    r.src = static_cast<const uint16_t*>(x.in) + (first + r.token) * x.in_token + head * x.in_head;
    r.dst = static_cast<uint16_t*>(x.out) + (first + r.token) * x.out_token + head * x.out_head;
    return r;
  };
  auto make_turns = [&] {
    for (int i = threadIdx.x; i < here * p.half; i += kThreads) {
      const int t = i / p.half, f = i - t * p.half;
      const double pos = p.wide_positions ? (double)static_cast<const int64_t*>(p.positions)[first + t]
                                          : (double)static_cast<const int32_t*>(p.positions)[first + t];
      turns[i] = turn_of(pos, p.inv_freq[f], p.amplitude);
    }
    __syncthreads();
  };

  if constexpr (VEC) {
    for (int base = 0; base < units; base += kThreads * kUnits) {
      Unit un[kUnits];
      uint4 a[kUnits], b[kUnits];
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = base + i * kThreads + threadIdx.x;
        if (u >= units) continue;
        un[i] = unit_of(u);
        const bool turned = un[i].at < p.turned;
        if constexpr (HALF) {
          // a turned unit is a chunk and the one half a rotary dim behind it; a copied one follows both halves
          const int off = turned ? un[i].at * 8 : 2 * p.half + (un[i].at - p.turned) * 8;
          un[i].src += off;
          un[i].dst += off;
          a[i] = *reinterpret_cast<const uint4*>(un[i].src);
          if (turned) b[i] = *reinterpret_cast<const uint4*>(un[i].src + p.half);
        } else {
          un[i].src += un[i].at * 8;
          un[i].dst += un[i].at * 8;
          a[i] = *reinterpret_cast<const uint4*>(un[i].src);
        }
      }
      if (base == 0) make_turns();
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = base + i * kThreads + threadIdx.x;
        if (u >= units) continue;
        const bool turned = un[i].at < p.turned;
        const float2* cs = turns + un[i].token * p.half + un[i].at * (HALF ? 8 : 4);
        if constexpr (HALF) {
          if (turned) {
            turn_half(a[i], b[i], cs);
            *reinterpret_cast<uint4*>(un[i].dst + p.half) = b[i];
          }
        } else {
          if (turned) turn_neighbours(a[i], cs);
        }
        *reinterpret_cast<uint4*>(un[i].dst) = a[i];
      }
    }
  } else {
    make_turns();
    for (int u = threadIdx.x; u < units; u += kThreads) {
      const Unit un = unit_of(u);
      if (un.at < p.turned) {
        const int i = HALF ? un.at : 2 * un.at, j = HALF ? un.at + p.half : i + 1;
        const float2 c = turns[un.token * p.half + un.at];
        const float x = bf16_bits_to_float(un.src[i]), y = bf16_bits_to_float(un.src[j]);
        un.dst[i] = float_to_bf16_bits(x * c.x - y * c.y);
        un.dst[j] = float_to_bf16_bits(y * c.x + x * c.y);
      } else {
        const int i = p.half + un.at;            // 2 * half + (at - half)
        un.dst[i] = un.src[i];
      }
    }
  }
}

bool chunks_of(const sacq_head_rows& x) {
  auto al = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  return x.heads == 0 || (al(x.in) && al(x.out) && x.in_token % 8 == 0 && x.in_head % 8 == 0 && x.out_token % 8 == 0 &&
                          x.out_head % 8 == 0);
}

}  // namespace

int launch_rotate_heads(const sacq_rotary_desc& d, cudaStream_t s) {
  const bool halves = d.layout == SACQ_ROTARY_HALF;
  RotaryParams p = {};
  p.x[0] = d.q;
  p.x[1] = d.k;
  p.positions = d.positions;
  p.inv_freq = d.inv_freq;
  p.tokens = d.tokens;
  p.dim = d.head_dim;
  p.half = d.rotary_dim / 2;
  p.amplitude = d.amplitude;
  p.wide_positions = d.position_bytes == 8;
  const bool vec = d.head_dim % 8 == 0 && chunks_of(d.q) && chunks_of(d.k) && d.rotary_dim % (halves ? 16 : 8) == 0;
  p.turned = !vec ? p.half : halves ? p.half / 8 : p.half / 4;
  p.per_head = p.turned + (vec ? (d.head_dim - d.rotary_dim) / 8 : d.head_dim - d.rotary_dim);
  p.per_token = p.per_head * (d.q.heads + d.k.heads);
  // tokens of a CTA: one step of its threads, fewer where the grid would not fill the GPU, and no more turns than 48 KB
  const int64_t step = (int64_t)kThreads * kUnits / p.per_token;
  int64_t per = step < 1 ? 1 : step;
  if (per > d.tokens / 148) per = d.tokens / 148 > 0 ? d.tokens / 148 : 1;
  const int64_t room = 48 * 1024 / 8 / p.half;
  if (per > room) per = room;
  p.tokens_per_cta = (int)per;
  const int64_t grid = (d.tokens + per - 1) / per;
  if (grid > 2147483647LL) return set_error(SACQ_ERR_UNSUPPORTED, "%lld tokens exceed the grid limit", (long long)d.tokens);
  const void* fn = halves ? (vec ? (const void*)rotary_kernel<true, true> : (const void*)rotary_kernel<true, false>)
                          : (vec ? (const void*)rotary_kernel<false, true> : (const void*)rotary_kernel<false, false>);
  void* args[] = {&p};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)per * p.half * sizeof(float2);
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
