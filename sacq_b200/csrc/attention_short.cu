// Attention over packed sequences for few queries (single tokens, an action head's 16 steps), head dims up to 128.
//
// A tile is 16 rows: tokens x all heads of one key-value head's group.  What it costs is reading the keys and values, so
// everything is arranged for that: TMA brings 64 keys at a time (SWIZZLE_128B), two CTAs of an SM have up to 190 KB on their way.
// Two warps take the first 32 of the 64 keys and two the others, by mma.sync (m16n8k16); of each two, one has the first half of the
// head's output and one the second, and both make the weights.  Running maxima, sums and outputs are their own, in registers; the scores'
// accumulators are the next product's A operand as they lie.  At the end of an item the second two hand their results to the
// first through shared memory.
//
// Warp 4 lists the items and issues the copies, the queries of the next item among them.  Every mbarrier wait is bounded (status word + CTA-wide abort flag).
#include "attention.cuh"
#include "umma.cuh"

namespace sacq {

namespace {

using namespace umma;

constexpr int kRows = 16;
constexpr int kStep = 64;                    // keys of a copy
constexpr int kWarps = 4, kThreads = 32 * (kWarps + 1);

struct ShortParams {
  AttnParams a;
  AttnSplit split;
  int* status;
};

struct ShortItem {
  int last;
  int q_row, q_rows;                         // first token of the sequence; its rows (tokens x group)
  int first;                                 // first row of the tile
  int kv_head, k_row, keys, base;            // as in the kernel with 128-row tiles, base for the sequence's first token
  int steps;                                 // 64-key steps
  int part;
};

template <int DP>
struct ShortShape {
  static constexpr int kHalves = DP / 64, kHalfBytes = kStep * 128, kTensorBytes = kHalves * kHalfBytes, kStageBytes = 2 * kTensorBytes;
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int kQPitch = DP * 2 + 16, kQBytes = kRows * kQPitch;      // rows of 16 bytes more than 32 banks: ldmatrix meets each bank once
  static constexpr uint32_t kJoin = kStages * kStageBytes;              // two warps' [16 rows][DP / 2] sums
  static constexpr uint32_t kMl = kJoin + kRows * DP * 4;               // their [16][m, l]
  static constexpr uint32_t kQ = kMl + kRows * 8;                       // two items' rows of queries
  static constexpr uint32_t kItems = kQ + 2 * kQBytes;                  // two of 48 bytes
  static constexpr uint32_t kBars = kItems + 2 * 48;
  static constexpr uint32_t kAbort = kBars + 8 * 18;
  static constexpr uint32_t kTotal = kAbort + 16;
};
constexpr int ST_FULL = 0, ST_EMPTY = 6, IT_FULL = 12, IT_EMPTY = 14, JOIN = 16;      // mbarriers

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte of element (row, col) of a swizzled [rows][64] half of a tile.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

template <int DP>
__global__ void __launch_bounds__(kThreads, 2)
attention_short_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ShortParams p) {
  using Sh = ShortShape<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + Sh::kAbort);
  const uint32_t sm = smem_u32(smem);
  auto bar = [&](int i) { return sm + Sh::kBars + 8u * i; };
  auto item_at = [&](uint32_t i) { return reinterpret_cast<ShortItem*>(smem + Sh::kItems + (i & 1) * 48); };
  const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const AttnParams& a = p.a;
  const bool causal = a.causal != 0;
  const int group = a.heads / a.kv_heads;
  static_assert(sizeof(ShortItem) <= 48 && Sh::kStages <= 6, "item slots and mbarriers");

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < Sh::kStages; ++s) {
      mbar_init(bar(ST_FULL + s), 1);
      mbar_init(bar(ST_EMPTY + s), kWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(IT_FULL + s), 1);
      mbar_init(bar(IT_EMPTY + s), kWarps);
    }
    mbar_init(bar(JOIN), kWarps);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // what lies behind the head dim in the rows of queries is multiplied by zeros: no NaN
  for (uint32_t i = threadIdx.x; i < 2 * Sh::kQBytes / 16; i += kThreads) *reinterpret_cast<uint4*>(smem + Sh::kQ + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  if (warp == kWarps && lane == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == kWarps) {
    // ---- the list of items, and the copies they need
    const auto count = [&](int queries, int keys) -> int64_t {
      return ((int64_t)queries * group + kRows - 1) / kRows * chunks_of(p.split, keys) * a.kv_heads;
    };
    ItemList<decltype(count)> list{a, count};
    list.look();
    uint32_t c = 0, made = 0;
    bool ok = true;
    for (int64_t index = blockIdx.x; ok; index += gridDim.x) {
      ShortItem it = {};
      Span sq, sk;
      int64_t r;
      it.last = !list.find(index, sq, sk, r);
      if (!it.last) {
        const int lk = (int)sk.length, chunks = chunks_of(p.split, lk), tiles = key_tiles(lk);
        it.kv_head = digit_of(r, a.kv_heads);
        const int part = digit_of(r, chunks);
        it.first = (int)r * kRows;
        const int begin = chunks > 1 ? part * p.split.chunk : 0, n = chunks > 1 ? min(p.split.chunk, tiles - begin) : tiles;
        it.q_row = (int)sq.begin;
        it.q_rows = (int)sq.length * group;
        it.k_row = (int)sk.begin + begin * kKeyTile;
        it.keys = min(lk - begin * kKeyTile, n * kKeyTile);
        it.base = lk - (int)sq.length - begin * kKeyTile;
        it.part = chunks > 1 ? part : -1;
        const int most = causal ? min(it.keys, it.base + (min(it.first + kRows, it.q_rows) - 1) / group + 1) : it.keys;
        it.steps = most > 0 ? (most + kStep - 1) / kStep : 0;
      }
      ok = mbar_wait_warp(bar(IT_EMPTY + (made & 1)), ((made >> 1) & 1) ^ 1, abort_flag, p.status, kWaitNs);
      if (!ok) break;
      const int rows = it.last ? 0 : min(kRows, it.q_rows - it.first);
      if (lane == 0) {
        *item_at(made) = it;
        mbar_arrive_expect_tx(bar(IT_FULL + (made & 1)), rows * a.dim * 2);
      }
      __syncwarp();
      if (lane < rows) {
        const int t = (it.first + lane) / group, head = it.kv_head * group + it.first + lane - t * group;
        bulk_load(sm + Sh::kQ + (made & 1) * Sh::kQBytes + lane * Sh::kQPitch, a.q + (int64_t)(it.q_row + t) * a.q_token + (int64_t)head * a.q_head,
                  a.dim * 2, bar(IT_FULL + (made & 1)));
      }
      __syncwarp();
      ++made;
      if (it.last) break;
      for (int j = 0; j < it.steps; ++j, ++c) {
        const uint32_t s = c % Sh::kStages;
        ok = mbar_wait_warp(bar(ST_EMPTY + s), ((c / Sh::kStages) & 1) ^ 1, abort_flag, p.status, kWaitNs);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar(ST_FULL + s), Sh::kStageBytes);
          for (int h = 0; h < Sh::kHalves; ++h) {
            tma_load_3d(sm + s * Sh::kStageBytes + h * Sh::kHalfBytes, &map_k, h * 64, it.kv_head, it.k_row + j * kStep, bar(ST_FULL + s));
            tma_load_3d(sm + s * Sh::kStageBytes + Sh::kTensorBytes + h * Sh::kHalfBytes, &map_v, h * 64, it.kv_head, it.k_row + j * kStep, bar(ST_FULL + s));
          }
        }
        __syncwarp();
      }
    }
    if (*abort_flag) {                       // copies in flight land before the CTA leaves
      for (uint32_t i = made > 2 ? made - 2 : 0; i < made; ++i)
        for (int t = 0; t < 100000 && !mbar_try_wait(bar(IT_FULL + (i & 1)), (i >> 1) & 1); ++t) {}
      for (uint32_t i = c > Sh::kStages ? c - Sh::kStages : 0; i < c; ++i)
        for (int t = 0; t < 100000 && !mbar_try_wait(bar(ST_FULL + i % Sh::kStages), (i / Sh::kStages) & 1); ++t) {}
    }
    return;
  }

  // ---- a warp's 32 keys of each step and its half of the outputs.  This thread's part of a 16 x 16 tile: rows lane / 4 and 8 more,
  // columns 2 (lane % 4) and 8 more
  const int keys_from = (warp >> 1) * 32, out_half = warp & 1;
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  const float c2 = a.scale * kLog2e;
  // ldmatrix addresses.  K: keys lane % 8 and 8 more from lane 16 on; Q and V: rows lane % 16
  const int k_key = (lane & 7) + ((lane >> 4) << 3), k_chunk = (lane >> 3) & 1;
  const int v_key = lane & 15, v_chunk = lane >> 4;
  constexpr int kBlocks = DP / 16;           // blocks of 8 columns of a warp's outputs
  uint32_t c = 0, joins = 0;
  bool ok = true;
  auto meet = [&] {                          // of the four warps
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(JOIN));
    ok = mbar_wait_warp(bar(JOIN), joins & 1, abort_flag, p.status, kWaitNs) && ok;
    ++joins;
  };
  for (uint32_t i = 0; ok; ++i) {
    if (!mbar_wait_warp(bar(IT_FULL + (i & 1)), (i >> 1) & 1, abort_flag, p.status, kWaitNs)) break;
    const ShortItem it = *item_at(i);
    uint32_t q[DP / 16][4];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
      ldmatrix4(q[ks], sm + Sh::kQ + (i & 1) * Sh::kQBytes + v_key * Sh::kQPitch + (ks * 2 + v_chunk) * 16);
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(IT_EMPTY + (i & 1)));
    if (it.last) break;
    int token[2], head[2], mine[2];          // of this thread's two rows; keys they see
    bool valid[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = it.first + r0 + 8 * h;
      valid[h] = row < it.q_rows;
      const int t = valid[h] ? row / group : 0;
      token[h] = it.q_row + t;
      head[h] = it.kv_head * group + (valid[h] ? row - t * group : 0);
      mine[h] = !valid[h] ? 0 : causal ? max(0, min(it.keys, it.base + t + 1)) : it.keys;
    }
    const int least = __reduce_min_sync(0xffffffffu, min(valid[0] ? mine[0] : it.keys, valid[1] ? mine[1] : it.keys));
    const int most = __reduce_max_sync(0xffffffffu, max(mine[0], mine[1]));
    float o[kBlocks][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int j = 0; j < it.steps; ++j, ++c) {
      const uint32_t s = c % Sh::kStages;
      if (!mbar_wait_warp(bar(ST_FULL + s), (c / Sh::kStages) & 1, abort_flag, p.status, kWaitNs)) { ok = false; break; }
      const int key = j * kStep + keys_from;                 // first of this warp's
      if (key < most) {
        const uint32_t kt = sm + s * Sh::kStageBytes, vt = kt + Sh::kTensorBytes;
        if (key + 32 > it.keys) {                            // rows behind the last key: zeros, whatever lies there in memory
          constexpr int kPieces = kBlocks;                   // 16-byte pieces of this warp's half of a row
          for (int e = lane; e < (key + 32 - it.keys) * kPieces; e += 32) {
            const int row = keys_from + it.keys - key + e / kPieces, piece = out_half * kPieces + e % kPieces;
            *reinterpret_cast<uint4*>(smem + s * Sh::kStageBytes + Sh::kTensorBytes + (piece >> 3) * Sh::kHalfBytes + swizzled(row, piece & 7)) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
        float sc[4][4] = {};
#pragma unroll
        for (int part = 0; part < DP / 64; ++part) {         // operands of 64 columns are fetched together: each waits 30 clocks otherwise
          uint32_t b[4][2][4];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            ldmatrix4(b[e >> 1][e & 1], kt + part * Sh::kHalfBytes + swizzled(keys_from + (e & 1) * 16 + k_key, (e >> 1) * 2 + k_chunk));
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              mma_bf16(sc[2 * n], q[part * 4 + ks], b[ks][n][0], b[ks][n][1]);
              mma_bf16(sc[2 * n + 1], q[part * 4 + ks], b[ks][n][2], b[ks][n][3]);
            }
        }
        if (key + 32 > least) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key + n * 8 + c0 + (e & 1) >= mine[e >> 1]) sc[n][e] = -INFINITY;
        }
        float high[2], keep[2], base[2];
        bool rise = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          high[h] = m[h];
#pragma unroll
          for (int n = 0; n < 4; ++n) high[h] = fmaxf(high[h], fmaxf(sc[n][2 * h], sc[n][2 * h + 1]));
          high[h] = fmaxf(high[h], __shfl_xor_sync(0xffffffffu, high[h], 1));
          high[h] = fmaxf(high[h], __shfl_xor_sync(0xffffffffu, high[h], 2));
          rise = rise || high[h] > m[h];
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            keep[h] = m[h] == -INFINITY ? 0.f : exp2_fast((m[h] - high[h]) * c2);
            m[h] = high[h];
            l[h] *= keep[h];
          }
#pragma unroll
          for (int n = 0; n < kBlocks; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= keep[e >> 1];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) base[h] = m[h] == -INFINITY ? 0.f : m[h] * c2;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[n][e] = exp2_fast(fmaf(sc[n][e], c2, -base[e >> 1]));
            l[e >> 1] += sc[n][e];
          }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t w[4] = {bf16_pair(sc[2 * n][0], sc[2 * n][1]), bf16_pair(sc[2 * n][2], sc[2 * n][3]), bf16_pair(sc[2 * n + 1][0], sc[2 * n + 1][1]),
                                 bf16_pair(sc[2 * n + 1][2], sc[2 * n + 1][3])};
          uint32_t b[kBlocks / 2][4];
#pragma unroll
          for (int d = 0; d < kBlocks / 2; ++d) {
            const int chunk = out_half * kBlocks + 2 * d;    // of 8 columns, of the whole row
            ldmatrix4_trans(b[d], vt + (chunk >> 3) * Sh::kHalfBytes + swizzled(keys_from + n * 16 + v_key, (chunk & 7) + v_chunk));
          }
#pragma unroll
          for (int d = 0; d < kBlocks / 2; ++d) {
            mma_bf16(o[2 * d], w, b[d][0], b[d][1]);
            mma_bf16(o[2 * d + 1], w, b[d][2], b[d][3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(ST_EMPTY + s));
    }
    if (!ok) break;
    // the sums of a row: four lanes have its columns
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    if (most > 32) {                         // the second two warps have had keys
      float* const room = reinterpret_cast<float*>(smem + Sh::kJoin) + out_half * kRows * DP / 2;
      float2* const room_ml = reinterpret_cast<float2*>(smem + Sh::kMl);
      if (warp >= 2) {
        // elements where the lanes of a warp store and load 16 bytes next to one another
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) *reinterpret_cast<float4*>(room + (n * 32 + lane) * 4) = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
        if (out_half == 0 && (lane & 3) == 0) {
          room_ml[r0] = make_float2(m[0], l[0]);
          room_ml[r0 + 8] = make_float2(m[1], l[1]);
        }
      }
      meet();
      if (warp < 2) {
        float ka[2], kb[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 other = room_ml[r0 + 8 * h];
          const float high = fmaxf(m[h], other.x);
          ka[h] = m[h] == -INFINITY ? 0.f : exp2_fast((m[h] - high) * c2);
          kb[h] = other.x == -INFINITY ? 0.f : exp2_fast((other.x - high) * c2);
          l[h] = l[h] * ka[h] + other.y * kb[h];
          m[h] = high;
        }
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
          const float4 v = *reinterpret_cast<const float4*>(room + (n * 32 + lane) * 4);
          o[n][0] = fmaf(v.x, kb[0], o[n][0] * ka[0]);
          o[n][1] = fmaf(v.y, kb[0], o[n][1] * ka[0]);
          o[n][2] = fmaf(v.z, kb[1], o[n][2] * ka[1]);
          o[n][3] = fmaf(v.w, kb[1], o[n][3] * ka[1]);
        }
      }
      meet();
      if (!ok) break;
    }
    if (warp >= 2) continue;
    uint32_t odd = 0;                        // which of the two rows have a value that is not finite
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // a chunk whose keys all score -inf: its sums, zeros, as they are, since the chunks are joined with a weight of zero for it
      const float inv = mine[h] == 0 ? 0.f : it.part >= 0 && m[h] == -INFINITY ? 1.f : 1.0f / l[h];
      bool finite = true;
      const int64_t slot = ((int64_t)max(it.part, 0) * a.tokens_q + token[h]) * a.heads + head[h];
      uint16_t* const out = a.out + (int64_t)token[h] * a.out_token + (int64_t)head[h] * a.out_head;
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) {
        const float x = mine[h] > 0 ? o[n][2 * h] * inv : 0.f, y = mine[h] > 0 ? o[n][2 * h + 1] * inv : 0.f;
        finite = finite && fabsf(x) < INFINITY && fabsf(y) < INFINITY;
        const int d = out_half * DP / 2 + n * 8 + c0;
        if (valid[h] && d < a.dim) {
          if (it.part < 0) *reinterpret_cast<uint32_t*>(out + d) = bf16_pair(x, y);
          else *reinterpret_cast<float2*>(p.split.part_o + slot * a.dim + d) = make_float2(x, y);
        }
      }
      if (valid[h] && out_half == 0 && (lane & 3) == 0) {
        const float le = mine[h] > 0 ? fmaf(m[h], a.scale, logf(l[h])) : -INFINITY;
        if (it.part >= 0) p.split.part_lse[slot] = le;
        else if (a.lse != nullptr) a.lse[(int64_t)token[h] * a.heads + head[h]] = le;
      }
      if (valid[h] && !finite && mine[h] > 0) odd |= 1u << h;
    }
    __syncwarp();                            // the rows as they are lie in front of the ones made again
    // a warp multiplies 32 keys at a time, those of the last 32 that no row of the tile sees among them; the first lane of four stands for a row
    const int end = min((most + 31) & ~31, it.keys);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      const uint32_t bad = __ballot_sync(0xffffffffu, (odd >> h) & 1);
      if (bad != 0)
        redo_rows(a, p.split, it.k_row, it.kv_head, it.part, h ? token[1] : token[0], h ? head[1] : head[0], h ? mine[1] : mine[0],
                  (lane & 3) == 0 && (bad >> lane & 0xf) != 0, end, out_half * DP / 2, (out_half + 1) * DP / 2);
    }
  }
}

int64_t short_items(const AttnParams& a, int64_t* per_sequence) {
  const int64_t group = a.heads / a.kv_heads, rows = a.tokens_q * group;
  const int64_t tiles = rows / kRows + (a.tokens_q < a.sequences ? a.tokens_q : a.sequences);    // at most
  if (per_sequence != nullptr) *per_sequence = (rows / a.sequences + kRows - 1) / kRows * a.kv_heads;
  return tiles * a.kv_heads;
}

}  // namespace

// Only the sizes of a call are known here, not its offsets.  Into chunks of a third of a CTA's share, if the sequences are alike (16 tokens,
// pasts of 501 to 16,384: 12 tiles 110 us, 9 113, 6 118), of 4 tiles at least; and only where that pays.  A tile takes a CTA 1.2 us, all
// of them together what their bytes take; the second kernel and the parts 6 us more.  Measured, without and with chunks: 1 token on 16,000
// keys 130 and 22 us, on 1,300 15.3 and 12.7; 3 x 8 tokens on 600 11.9 and 16.5, 45 on 388 17.4 and 19.7.
AttnSplit attention_short_split(const AttnParams& a, void* workspace) {
  int64_t per_sequence = 0;
  const int64_t items = short_items(a, &per_sequence), slots = 2 * device_sms() * 3 / 4, tiles = (a.tokens_k + kKeyTile - 1) / kKeyTile;
  int64_t chunk = 0;
  if (items < 4 * slots) {
    const int64_t share = (tiles + a.sequences) * per_sequence / (3 * slots), average = (tiles + a.sequences - 1) / a.sequences;
    chunk = share < 4 ? 4 : share;
    const double longest = (double)(a.sequences == 1 || tiles < 2 * average ? tiles : 2 * average);
    const double all = (double)a.tokens_k * a.kv_heads * a.dim * 4 / 6e6;      // us
    const double parts = (double)a.tokens_q * a.heads * a.dim * 8 / 5e6 * (double)((average + chunk - 1) / chunk);
    if (fmax(1.2 * (double)chunk, all) + 6 + parts > 0.9 * fmax(1.2 * longest, all)) chunk = 0;
  }
  return attention_chunks(a, chunk, workspace);
}

int launch_attention_short(const AttnParams& a, const AttnSplit& split, cudaStream_t s) {
  ShortParams p = {};
  p.a = a;
  p.split = split;
  p.status = attention_status_word();
  if (p.status == nullptr) return set_error(SACQ_ERR_CUDA, "no status word on this device");
  CUtensorMap mk, mv;
  if (int rc = attention_tensor_maps(a, 0, 0, kStep, nullptr, &mk, &mv)) return rc;
  const bool wide = a.dim > 64;
  const void* fn = wide ? (const void*)attention_short_kernel<128> : (const void*)attention_short_kernel<64>;
  const size_t smem = wide ? ShortShape<128>::kTotal : ShortShape<64>::kTotal;
  static bool configured[2][64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[wide][dev]) {
    SACQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev >= 0 && dev < 64) configured[wide][dev] = true;
  }
  const int64_t most = short_items(a, nullptr) * split.chunks_most, slots = 2 * device_sms();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(most < slots ? most : slots));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&mk, &mv, &p};
  SACQ_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
  count_launch();
  return SACQ_OK;
}

}  // namespace sacq
