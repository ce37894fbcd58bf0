// Rotary positions of query and key heads, in one launch:
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i],  both times `amplitude`
// for the rotary_dim / 2 pairs of every head; what lies behind rotary_dim is copied.  A pair is (x[i], x[i + R/2])
// ("half") or (x[2i], x[2i + 1]) ("interleaved").
//
// Angles: a position of 10^6 times a frequency near 1 is right to 0.06 radians in fp32, so the product is made in
// double, in turns (inv_freq / 2 pi), reduced to half a turn either way there, and only then rounded, to 2^-26 turns.
// The quotient, the product and the constant are rounded to 53 bits: 3 x 2^-53 of the angle, which is less than that up to
// angles of 2^28 radians and 2.9e-6 radians at 2^33.  They are the same for all heads, so a CTA makes those of its tokens once, in
// shared memory, between its loads and its stores.
//
// Bound by memory: 4 bytes per element.  A thread has one place in a token (16-byte chunks, of "half" both of a pair) and takes it in
// several tokens, so that nothing is divided; it holds what it loads in registers while the angles are made.
// 12,001 tokens of 24 heads of 128: 28 us, 5.3 TB/s (34 with units that each thread finds by division); 32,768 tokens, half of
// each head turned: 60 us, 6.7 TB/s, what a copy takes.
#include "common.cuh"

namespace sacq {

namespace {

constexpr int kMostThreads = 512;
constexpr int kTokens = 4;                      // of a thread at a time: loads in flight

struct RotaryParams {
  sacq_head_rows x[2];                          // query heads, key heads
  const void* positions;
  const double* inv_freq;
  int64_t tokens;
  int per_head;                                 // units of a head: turned ones first, then copied ones
  int turned;
  int per_token;                                // units of a token, both tensors
  int per_cta;                                  // tokens of a CTA, up to kTokens
  int half;                                     // rotated pairs
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

// Units of a token: 16-byte chunks (VEC; "half": two of them where turned), else single pairs and elements, at any alignment.
template <bool HALF, bool VEC>
__global__ void __launch_bounds__(kMostThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ __align__(16) float2 turns[];       // [per_cta][half]
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t first = (int64_t)blockIdx.x * p.per_cta;
  const int here = (int)min((int64_t)p.per_cta, p.tokens - first);

  struct Unit {
    const uint16_t* src;                        // in the CTA's first token
    uint16_t* dst;
    int64_t in_token, out_token;
    int at;                                     // unit of its head
  };
  auto unit_of = [&](int u) {
    Unit r;
    int head = u / p.per_head;
    r.at = u - head * p.per_head;
    const bool key = head >= p.x[0].heads;
    if (key) head -= p.x[0].heads;
    const sacq_head_rows& x = p.x[key];
    r.in_token = x.in_token;
    r.out_token = x.out_token;
    r.src = static_cast<const uint16_t*>(x.in) + first * x.in_token + head * x.in_head;
    r.dst = static_cast<uint16_t*>(x.out) + first * x.out_token + head * x.out_head;
    return r;
  };
  auto make_turns = [&] {
    for (int f = threadIdx.x; f < p.half * here; f += blockDim.x) {
      const int t = f / p.half, i = f - t * p.half;
      const double pos = p.wide_positions ? (double)static_cast<const int64_t*>(p.positions)[first + t]
                                          : (double)static_cast<const int32_t*>(p.positions)[first + t];
      turns[f] = turn_of(pos, p.inv_freq[i], p.amplitude);
    }
    __syncthreads();
  };

  if constexpr (VEC) {
    for (int base = 0; base < p.per_token; base += blockDim.x) {
      const bool real = base + (int)threadIdx.x < p.per_token;
      Unit un = {};
      bool turned = false;
      uint4 a[kTokens], b[kTokens];
      if (real) {
        un = unit_of(base + threadIdx.x);
        turned = un.at < p.turned;
        // "half": a turned unit is a chunk and the one half a rotary dim behind it; a copied one follows both halves
        const int off = !HALF || turned ? un.at * 8 : 2 * p.half + (un.at - p.turned) * 8;
        un.src += off;
        un.dst += off;
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
          if (t < here) {
            a[t] = *reinterpret_cast<const uint4*>(un.src + t * un.in_token);
            if (HALF && turned) b[t] = *reinterpret_cast<const uint4*>(un.src + t * un.in_token + p.half);
          }
      }
      if (base == 0) make_turns();
      if (!real) continue;
#pragma unroll
      for (int t = 0; t < kTokens; ++t)
        if (t < here) {
          if (turned) {
            const float2* const cs = turns + t * p.half + un.at * (HALF ? 8 : 4);
            if constexpr (HALF) {
              turn_half(a[t], b[t], cs);
              *reinterpret_cast<uint4*>(un.dst + t * un.out_token + p.half) = b[t];
            } else {
              turn_neighbours(a[t], cs);
            }
          }
          *reinterpret_cast<uint4*>(un.dst + t * un.out_token) = a[t];
        }
    }
  } else {
    make_turns();
    for (int u = threadIdx.x; u < p.per_token; u += blockDim.x) {
      const Unit un = unit_of(u);
      for (int t = 0; t < here; ++t) {
        const uint16_t* const src = un.src + t * un.in_token;
        uint16_t* const dst = un.dst + t * un.out_token;
        if (un.at < p.turned) {
          const int i = HALF ? un.at : 2 * un.at, j = HALF ? un.at + p.half : i + 1;
          const float2 c = turns[t * p.half + un.at];
          const float x = bf16_bits_to_float(src[i]), y = bf16_bits_to_float(src[j]);
          dst[i] = float_to_bf16_bits(x * c.x - y * c.y);
          dst[j] = float_to_bf16_bits(y * c.x + x * c.y);
        } else {
          const int i = p.half + un.at;          // 2 * half + (at - half)
          dst[i] = src[i];
        }
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
  p.half = d.rotary_dim / 2;
  p.amplitude = d.amplitude;
  p.wide_positions = d.position_bytes == 8;
  const bool vec = d.head_dim % 8 == 0 && chunks_of(d.q) && chunks_of(d.k) && d.rotary_dim % (halves ? 16 : 8) == 0;
  p.turned = !vec ? p.half : halves ? p.half / 8 : p.half / 4;
  p.per_head = p.turned + (vec ? (d.head_dim - d.rotary_dim) / 8 : d.head_dim - d.rotary_dim);
  p.per_token = p.per_head * (d.q.heads + d.k.heads);
  // few tokens are spread over the SMs
  const int64_t share = d.tokens / device_sms();
  p.per_cta = share < 1 ? 1 : share < kTokens ? (int)share : kTokens;
  const int room = 48 * 1024 / (int)sizeof(float2) / p.half;
  if (p.per_cta > room) p.per_cta = room;
  const int64_t grid = (d.tokens + p.per_cta - 1) / p.per_cta;
  if (grid > 2147483647LL) return set_error(SACQ_ERR_UNSUPPORTED, "%lld tokens exceed the grid limit", (long long)d.tokens);
  const void* fn = halves ? (vec ? (const void*)rotary_kernel<true, true> : (const void*)rotary_kernel<true, false>)
                          : (vec ? (const void*)rotary_kernel<false, true> : (const void*)rotary_kernel<false, false>);
  void* args[] = {&p};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)(p.per_token < kMostThreads ? (p.per_token + 31) / 32 * 32 : kMostThreads));
  cfg.dynamicSmemBytes = (size_t)p.per_cta * p.half * sizeof(float2);
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
