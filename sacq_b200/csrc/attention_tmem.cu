// Attention over packed sequences on the tensor cores (sm_100a), head dims up to 128, persistent CTAs.
//
// A tile is 128 rows of queries: 128 / pack tokens x `pack` heads of one key-value head (pack: the largest power of two
// that divides the group), so that single tokens share a tile with the other heads of their group and a causal tile's
// diagonal is 128 / pack keys wide.  Keys come 128 at a time:
//   S = Q K^T        tcgen05.mma, Q and K tiles in shared memory (TMA, SWIZZLE_128B), S in tensor memory, fp32
//   P = exp(S - m)   one thread per row: running maximum and sum, no shuffles; P goes back to tensor memory as bf16
//   O += P V         tcgen05.mma with P from tensor memory as A, the V tile as it lies (MN-major B), O in tensor memory
// P is rounded to bf16 because V is bf16 and one instruction's operands have one type; its sum is taken before that.
// O is rescaled only when a row's maximum has risen by more than 2^8 since the last time: until then exp(S - m) stays
// below 256, which bf16 and the fp32 sums hold as exactly as values below 1.
//
// An item of work is a pair of tiles of one sequence and head group, over its keys or a chunk of them.  Both tiles
// share the K and V tiles, each has its warpgroup, S and O: while the tensor cores work for one, the other's
// exponentials are taken.  Up to head dim 64 P has columns of its own, and S of the next keys is made as soon as the last one is in
// registers (8 causal prompts of 2048, 16 heads of 64: 130 against 143 us, 2 x 8192 to all keys: 684 against 791); wider, O leaves no
// room for that, and P lies over S.  Where the sequence has one tile's tokens only, the two warpgroups take its keys in turn and their
// results are joined.  Chunks (few items, many keys) leave fp32 results, joined by a second kernel in a fixed order.
//
// Roles: warps 0-3 and 4-7 softmax and epilogue of the two tiles, warp 8 MMA issuer and TMEM owner, warp 9 TMA and the
// list of items.  Every mbarrier wait is bounded (status word + CTA-wide abort flag).
#include <cuda.h>

#include "attention.cuh"
#include "encode.cuh"
#include "umma.cuh"

namespace sacq {

namespace {

using namespace umma;

constexpr int kTile = kKeyTile;
constexpr int kThreads = 320;
constexpr int kMmaWarp = 8, kLoadWarp = 9;
constexpr float kRescale = 8.0f;            // log2

struct TmemAttnParams {
  AttnParams a;
  int pack_log2;                            // heads of a tile
  int groups;                               // heads / pack
  AttnSplit split;
  int* status;
  int dynamic;                              // a CTA per item that there can be: running CTAs take over those that have not begun
};

struct alignas(16) Item {
  int last;                                 // no more items
  int q_row, q_left;                        // first query row; rows of the sequence from it on
  int head, kv_head;
  int k_row, keys;                          // first key row, keys of the chunk
  int base;                                 // causal: token t of the item sees min(keys, base + t + 1), else keys
  int n, n0;                                // key tiles of the item (dual: of the second tile), dual: of the first
  int dual;
  int part;                                 // chunk, or -1: the whole result
};

template <int DP>
struct Shape {
  static constexpr int kHalves = DP / 64;
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kHalfBytes = kTile * 128;          // 64 bf16 of every row
  static constexpr int kStages = DP == 128 ? 4 : 8;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kRing = 2 * kTileBytes;
  static constexpr uint32_t kJoin = kRing + kStages * kTileBytes;   // 128 rows x 64 fp32
  static constexpr uint32_t kJoinMl = kJoin + kTile * 256;          // 128 x (m, l)
  static constexpr uint32_t kBars = kJoinMl + kTile * 8;
  static constexpr uint32_t kItems = kBars + 8 * 64;
  static constexpr uint32_t kMisc = kItems + 2 * 64;
  static constexpr uint32_t kTotal = kMisc + 64;
  // tensor memory columns; the weights of a wide tile lie over the first half of its S
  static constexpr int kS = 0, kO = 256, kP = DP == 128 ? 0 : 384, kPStep = DP == 128 ? kTile : 64;
  static constexpr bool kWide = DP == 128;
};
// mbarriers
constexpr int Q_FULL = 0, Q_EMPTY = 1, S_FULL = 2, P_FULL = 4, O_FULL = 6, S_READ = 8, ITEM_FULL = 10, ITEM_EMPTY = 12,
              DRAIN = 14, TAKE = 15, KV_FULL = 16, KV_EMPTY = 32, JOIN_FULL = 48, JOIN_EMPTY = 52;

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
__device__ __forceinline__ void umma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_bf16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// fp32 accumulator, bf16 operands, A K-major, B K-major or (b_mn) MN-major, M = 128.
__device__ __forceinline__ uint32_t idesc_bf16(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// MN-major operand (a V tile): 64 columns x 8 rows to a swizzle atom, 1024 bytes from one group of 8 rows to the next, `half`
// bytes from 64 columns to the next 64.
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t addr, uint32_t half) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(half >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {      // without waiting
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Waits for the loads of this thread; the registers pass through, so that no use of them moves in front of it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {      // without waiting
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of three, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x of two values: on the special-function unit, or by a polynomial.  The unit takes 8 cycles for a warp, which would
// bound the kernel; of every 8 pairs kPolynomials go by x = n + f, f in [-1/2, 1/2], and a polynomial of degree 5 for 2^f (least
// largest relative error, 7.5e-8, fitted by iterated reweighted least squares), n added to its exponent.  From x = -127 down, -inf
// among them, that leaves 2^-149, which is zero in bf16: a weight of a column that is not seen has to be, whatever V holds there.
constexpr int kPolynomials = 2;
__device__ __forceinline__ uint64_t exp2_unit(uint64_t v) {
  float x, y;
  halves_of(v, x, y);
  return f32x2(exp2_fast(x), exp2_fast(y));
}
__device__ __forceinline__ uint64_t exp2_polynomial(uint64_t v) {
  float x, y;
  halves_of(v, x, y);
  v = f32x2(fmaxf(x, -127.f), fmaxf(y, -127.f));
  const uint64_t magic = f32x2(12582912.0f, 12582912.0f);            // 1.5 * 2^23: the sum holds the nearest integer in its low bits
  const uint64_t t = add2(v, magic);
  const uint64_t f = fma2(add2(t, f32x2(-12582912.0f, -12582912.0f)), f32x2(-1.f, -1.f), v);
  uint64_t r = fma2(f32x2(0.0013276472454890609f, 0.0013276472454890609f), f, f32x2(0.009675541892647743f, 0.009675541892647743f));
  r = fma2(r, f, f32x2(0.05550713092088699f, 0.05550713092088699f));
  r = fma2(r, f, f32x2(0.24022120237350464f, 0.24022120237350464f));
  r = fma2(r, f, f32x2(0.6931469440460205f, 0.6931469440460205f));
  r = fma2(r, f, f32x2(1.0000001192092896f, 1.0000001192092896f));
  float a, b, ta, tb;
  halves_of(r, a, b);
  halves_of(t, ta, tb);
  return f32x2(__uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23)), __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23)));
}
// Asks for a CTA of the grid that has not begun; it will not, and the answer (16 bytes) says which it was, or that there was none.
__device__ __forceinline__ void request_cta(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar) : "memory");
}
__device__ __forceinline__ bool answered_cta(uint32_t answer, uint32_t& cta) {
  uint32_t yes, x;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 a, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
      : "=r"(yes), "=r"(x) : "r"(answer) : "memory");
  cta = x;
  return yes != 0;
}
// An item's fields, the same in all lanes and known to be: what is computed from them may stay in uniform registers.
__device__ __forceinline__ Item uniform_item(const Item* at) {
  Item it;
#define SACQ_SAME(field) it.field = (int)warp_uniform((uint32_t)at->field)
  SACQ_SAME(last); SACQ_SAME(q_row); SACQ_SAME(q_left); SACQ_SAME(head); SACQ_SAME(kv_head); SACQ_SAME(k_row); SACQ_SAME(keys);
  SACQ_SAME(base); SACQ_SAME(n); SACQ_SAME(n0); SACQ_SAME(dual); SACQ_SAME(part);
#undef SACQ_SAME
  return it;
}
// Keys that token t of an item sees.
__device__ __forceinline__ int seen(const Item& it, bool causal, int t) { return causal ? max(0, min(it.keys, it.base + t + 1)) : it.keys; }
// Columns of key tile j that the tile's last token sees, in whole instructions of 16.
__device__ __forceinline__ int columns(int most, int j) { return (min(kTile, most - j * kTile) + 15) & ~15; }

// SPLIT: there may be chunks (their code costs the others registers: 44.6 us of the 64 x 256 tokens became 47.3).
template <int DP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
attention_tmem_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                      const __grid_constant__ TmemAttnParams p) {
  using Sh = Shape<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sm = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const sp = smem_raw + (sm - smem_u32(smem_raw));
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(sp + Sh::kMisc);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sp + Sh::kMisc + 8);
  Item* const items = reinterpret_cast<Item*>(sp + Sh::kItems);       // two of 64 bytes
  auto item_at = [&](uint32_t i) { return reinterpret_cast<Item*>(reinterpret_cast<uint8_t*>(items) + (i & 1) * 64); };
  auto bar = [&](int i) { return sm + Sh::kBars + 8u * i; };
  const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const AttnParams& a = p.a;
  const int tokens_log2 = 7 - p.pack_log2;                              // tokens of a tile
  const int tile_tokens = 1 << tokens_log2;
  const bool causal = a.causal != 0;
  static_assert(sizeof(Item) <= 64, "item slots");

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    mbar_init(bar(Q_FULL), 1);
    mbar_init(bar(Q_EMPTY), 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(bar(S_FULL + w), 1);
      mbar_init(bar(S_READ + w), 4);
      mbar_init(bar(P_FULL + w), 4);
      mbar_init(bar(O_FULL + w), 1);
      mbar_init(bar(ITEM_FULL + w), 1);
      mbar_init(bar(ITEM_EMPTY + w), 9);
    }
    mbar_init(bar(DRAIN), 1);
    mbar_init(bar(TAKE), 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(JOIN_FULL + i), 1);
      mbar_init(bar(JOIN_EMPTY + i), 1);
    }
    for (int s = 0; s < Sh::kStages; ++s) {
      mbar_init(bar(KV_FULL + s), 1);
      mbar_init(bar(KV_EMPTY + s), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == kMmaWarp) tmem_alloc(smem_u32(tmem_slot), 512);
  if (warp == kLoadWarp && lane == 0) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    prefetch_tensormap(&map_o);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_uniform(*tmem_slot);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == kLoadWarp) {
    // ---- the list of items, and the copies they need
    uint32_t c = 0, nq = 0, made = 0;        // key / value tiles, items with keys, items so far
    bool ok = true;
    auto take = [&](const CUtensorMap* map, const Item& it, int j) {
      const uint32_t s = c % Sh::kStages;
      ok = ok && mbar_wait_warp(bar(KV_EMPTY + s), ((c / Sh::kStages) & 1) ^ 1, abort_flag, p.status, kWaitNs);
      if (!ok) return;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar(KV_FULL + s), Sh::kTileBytes);
        for (int h = 0; h < Sh::kHalves; ++h)
          tma_load_3d(sm + Sh::kRing + s * Sh::kTileBytes + h * Sh::kHalfBytes, map, h * 64, it.kv_head, it.k_row + j * kTile, bar(KV_FULL + s));
      }
      __syncwarp();
      ++c;
    };
    const auto count = [&](int queries, int keys) -> int64_t {
      return (int64_t)((queries + 2 * tile_tokens - 1) >> (tokens_log2 + 1)) * chunks_of(p.split, keys) * p.groups;
    };
    ItemList<decltype(count)> list{a, count};
    list.look();
    // the next item: the CTA's stride further, or one that is taken over; asked for while this one's copies are issued
    const uint32_t answer = sm + Sh::kMisc + 16;
    uint32_t taken = 0;
    bool more = true;
    auto ask = [&] {
      if (p.dynamic && elect_one()) {
        fence_proxy_async();
        mbar_arrive_expect_tx(bar(TAKE), 16);
        request_cta(answer, bar(TAKE));
      }
      __syncwarp();
    };
    auto advance = [&](int64_t& index) {
      if (!p.dynamic) {
        index += gridDim.x;
        return;
      }
      ok = mbar_wait_warp(bar(TAKE), taken & 1, abort_flag, p.status, kWaitNs);
      ++taken;
      uint32_t cta = 0;
      more = ok && answered_cta(answer, cta);
      index = cta;
      __syncwarp();
    };
    for (int64_t index = blockIdx.x; ok; advance(index)) {
      Item it = {};
      Span sq, sk;
      int64_t r;
      it.last = !more || !list.find(index, sq, sk, r);
      if (p.dynamic && more && it.last) {                    // there can be more items than there are: their CTAs need not begin
        ask();
        continue;
      }
      if (!it.last) {
        // heads first, then chunks; the pairs of tiles from the last, longest one to the first
        const int lq = (int)sq.length, lk = (int)sk.length, chunks = SPLIT ? chunks_of(p.split, lk) : 1;
        const int pairs = (lq + 2 * tile_tokens - 1) >> (tokens_log2 + 1);
        const int group = digit_of(r, p.groups), part = digit_of(r, chunks);
        const int pair = pairs - 1 - (int)r;
        const int t0 = pair * 2 * tile_tokens;
        const int tiles = key_tiles(lk);
        const int first = chunks > 1 ? part * p.split.chunk : 0, n = chunks > 1 ? min(p.split.chunk, tiles - first) : tiles;
        it.q_row = (int)sq.begin + t0;
        it.q_left = lq - t0;
        it.head = group << p.pack_log2;
        it.kv_head = p.groups == a.kv_heads ? group : it.head / (a.heads / a.kv_heads);
        it.k_row = (int)sk.begin + first * kTile;
        it.keys = min(lk - first * kTile, n * kTile);
        it.base = lk - lq + t0 - first * kTile;
        it.dual = it.q_left > tile_tokens;
        const int most = seen(it, causal, min(it.q_left, it.dual ? 2 * tile_tokens : tile_tokens) - 1);
        it.n = key_tiles(most);
        it.n0 = it.dual ? key_tiles(seen(it, causal, tile_tokens - 1)) : 0;
        it.part = chunks > 1 ? part : -1;
      }
      ok = mbar_wait_warp(bar(ITEM_EMPTY + (made & 1)), ((made >> 1) & 1) ^ 1, abort_flag, p.status, kWaitNs);
      if (!ok) break;
      if (lane == 0) *item_at(made) = it;
      __syncwarp();
      it = uniform_item(item_at(made));
      if (lane == 0) mbar_arrive(bar(ITEM_FULL + (made & 1)));
      ++made;
      if (it.last) break;
      ask();
      if (it.n == 0) continue;
      ok = mbar_wait_warp(bar(Q_EMPTY), (nq & 1) ^ 1, abort_flag, p.status, kWaitNs);
      if (!ok) break;
      ++nq;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar(Q_FULL), (it.dual ? 2 : 1) * Sh::kTileBytes);
        for (int w = 0; w < (it.dual ? 2 : 1); ++w)
          for (int h = 0; h < Sh::kHalves; ++h)
            tma_load_3d(sm + Sh::kQ + w * Sh::kTileBytes + h * Sh::kHalfBytes, &map_q, h * 64, it.head, it.q_row + w * tile_tokens, bar(Q_FULL));
      }
      __syncwarp();
      // in the order of their use: K of the first two steps (both tiles of a wide one: of one), then V of a step and the next K
      const int ahead = it.dual && Sh::kWide ? 1 : 2;
      for (int j = 0; j < min(ahead, it.n); ++j) take(&map_k, it, j);
      for (int j = 0; j < it.n; ++j) {
        take(&map_v, it, j);
        if (j + ahead < it.n) take(&map_k, it, j + ahead);
      }
    }
    if (*abort_flag && p.dynamic)            // what is in flight lands before the CTA leaves
      for (int t = 0; t < 100000 && !mbar_try_wait(bar(TAKE), taken & 1); ++t) {}
    if (*abort_flag)
      for (uint32_t i = c > Sh::kStages ? c - Sh::kStages : 0; i < c; ++i)
        for (int t = 0; t < 100000 && !mbar_try_wait(bar(KV_FULL + i % Sh::kStages), (i / Sh::kStages) & 1); ++t) {}
  } else if (warp == kMmaWarp) {
    // ---- MMA issuer
    uint32_t c = 0, nq = 0, np0 = 0, np1 = 0;           // ring tiles, items with keys, products of each warpgroup
    const int k_steps = (a.dim + 15) / 16;
    const uint32_t idesc_pv = idesc_bf16(k_steps * 16, true);
    bool ok = true;
    auto next = [&]() -> uint32_t {          // the next tile of the ring
      const uint32_t s = c % Sh::kStages;
      ok = ok && mbar_wait_warp(bar(KV_FULL + s), (c / Sh::kStages) & 1, abort_flag, p.status, kWaitNs);
      ++c;
      return warp_uniform(s);
    };
    auto commit = [&](int b) {
      if (elect_one()) umma_commit(bar(b));
      __syncwarp();
    };
    auto qk = [&](int w, int tile, uint32_t s, int n) {       // S of warpgroup w from Q tile `tile`
      if (!ok) return;
      const uint32_t idesc = warp_uniform(idesc_bf16(n, false));
      const uint64_t qd = make_smem_desc(sm + Sh::kQ + tile * Sh::kTileBytes), kd = make_smem_desc(sm + Sh::kRing + s * Sh::kTileBytes);
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const uint64_t adv = (uint64_t)(((i >> 2) * Sh::kHalfBytes + (i & 3) * 32) >> 4);
        if (i < k_steps && elect_one()) umma_bf16_ss(tmem + Sh::kS + w * kTile, qd + adv, kd + adv, idesc, i > 0);
      }
      __syncwarp();
    };
    // O of warpgroup w += P V over the tile's first n keys.  (What the instructions are issued with has to be in uniform
    // registers, and the warp converged in front of and behind each group: 120 clocks each otherwise, 64 so.)
    auto pv = [&](int w, uint32_t s, int n, bool first) {
      if (!ok) return;
      n = (int)warp_uniform(n); w = (int)warp_uniform(w); s = warp_uniform(s);
      const uint64_t vd = make_mn_desc(sm + Sh::kRing + s * Sh::kTileBytes, Sh::kHalfBytes);
      const uint32_t more = warp_uniform(first ? 0u : 1u);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < kTile / 16; ++i)
        if (i * 16 < n && elect_one())
          umma_bf16_ts(tmem + Sh::kO + w * DP, tmem + Sh::kP + w * Sh::kPStep + i * 8, vd + (uint64_t)(i * 2048 >> 4), idesc_pv, i > 0 ? 1u : more);
      __syncwarp();
    };
    // rows of a V tile behind the last key, up to a whole instruction: zeros, whatever lies there in memory
    auto clear_tail = [&](uint32_t s, int keys) {
      if (!ok || keys >= kTile || (keys & 15) == 0) return;
      const int end = (keys + 15) & ~15;
      for (int i = lane; i < (end - keys) * 8 * Sh::kHalves; i += 32) {
        const int row = keys + (i >> 3) / Sh::kHalves, h = (i >> 3) % Sh::kHalves;
        *reinterpret_cast<uint4*>(sp + Sh::kRing + s * Sh::kTileBytes + h * Sh::kHalfBytes + row * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async();
      __syncwarp();
    };
    for (uint32_t i = 0; ok; ++i) {
      if (!mbar_wait_warp(bar(ITEM_FULL + (i & 1)), (i >> 1) & 1, abort_flag, p.status, kWaitNs)) break;
      const Item it = uniform_item(item_at(i));
      if (lane == 0) mbar_arrive(bar(ITEM_EMPTY + (i & 1)));
      if (it.last) break;
      if (it.n == 0) continue;
      if (!mbar_wait_warp(bar(Q_FULL), nq & 1, abort_flag, p.status, kWaitNs)) break;
      ++nq;
      const int most = seen(it, causal, min(it.q_left, it.dual ? 2 * tile_tokens : tile_tokens) - 1);
      if (it.dual) {
        const int most0 = seen(it, causal, tile_tokens - 1);
        auto scores = [&](int w, int j, uint32_t ks) {
          qk(w, w, ks, columns(w == 0 ? most0 : most, j));
          commit(S_FULL + w);
        };
        auto arrived = [&](int b, uint32_t phase) { ok = ok && mbar_wait_warp(bar(b), phase & 1, abort_flag, p.status, kWaitNs); };
        uint32_t ks = next();
        if (it.n0 > 0) scores(0, 0, ks);
        scores(1, 0, ks);
        commit(KV_EMPTY + ks);
        if (it.n == 1) commit(Q_EMPTY);
        for (int j = 0; j < it.n && ok; ++j) {
          if constexpr (!Sh::kWide) {        // S of the next keys as soon as the last one is in registers, beside the exponentials
            if (j + 1 < it.n) {
              ks = next();
              if (j + 1 < it.n0) {
                arrived(S_READ + 0, np0);
                tc_fence_after();
                scores(0, j + 1, ks);
              }
              arrived(S_READ + 1, np1);
              tc_fence_after();
              scores(1, j + 1, ks);
              commit(KV_EMPTY + ks);
              if (j + 2 == it.n) commit(Q_EMPTY);
            }
            const uint32_t vs = next();
            clear_tail(vs, it.keys - j * kTile);
            if (j < it.n0) {
              arrived(P_FULL + 0, np0++);
              pv(0, vs, columns(most0, j), j == 0);
              commit(O_FULL + 0);
            }
            arrived(P_FULL + 1, np1++);
            pv(1, vs, columns(most, j), j == 0);
            commit(O_FULL + 1);
            commit(KV_EMPTY + vs);
          } else {                           // the weights lie over S: it is made behind P V
            const uint32_t vs = next();
            clear_tail(vs, it.keys - j * kTile);
            if (j < it.n0) {
              arrived(P_FULL + 0, np0++);
              pv(0, vs, columns(most0, j), j == 0);
            }
            if (j + 1 < it.n) ks = next();
            if (j + 1 < it.n0) scores(0, j + 1, ks);
            else if (j + 1 == it.n0) commit(O_FULL + 0);
            arrived(P_FULL + 1, np1++);
            pv(1, vs, columns(most, j), j == 0);
            commit(KV_EMPTY + vs);
            if (j + 1 < it.n) {
              scores(1, j + 1, ks);
              commit(KV_EMPTY + ks);
              if (j + 2 == it.n) commit(Q_EMPTY);
            } else {
              commit(O_FULL + 1);
            }
          }
        }
      } else {
        auto scores = [&](int w, int j) {
          const uint32_t ks = next();
          qk(w, 0, ks, columns(most, j));
          commit(S_FULL + w);
          commit(KV_EMPTY + ks);
          if (j + 1 == it.n) commit(Q_EMPTY);
        };
        for (int j = 0; j < min(2, it.n); ++j) scores(j, j);
        for (int j = 0; j < it.n && ok; ++j) {
          const int w = j & 1;
          const uint32_t vs = next();
          clear_tail(vs, it.keys - j * kTile);
          ok = ok && mbar_wait_warp(bar(P_FULL + w), (w == 0 ? np0 : np1) & 1, abort_flag, p.status, kWaitNs);
          pv(w, vs, columns(most, j), j < 2);
          if (w == 0) ++np0; else ++np1;
          if (!Sh::kWide || j + 2 >= it.n) commit(O_FULL + w);
          commit(KV_EMPTY + vs);
          if (j + 2 < it.n) scores(w, j + 2);
        }
      }
    }
    commit(DRAIN);                           // nothing of this CTA is in flight when it gives its tensor memory back
    for (int t = 0; t < 1000000 && !mbar_try_wait(bar(DRAIN), 0); ++t) {}
  } else {
    // ---- softmax and epilogue: warpgroup w, one row per thread
    const int w = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_at = tmem + lanes + Sh::kS + w * kTile, p_at = tmem + lanes + Sh::kP + w * Sh::kPStep, o_at = tmem + lanes + Sh::kO + w * DP;
    const float c2 = a.scale * kLog2e;
    uint32_t ns = 0, no = 0, nj = 0;         // steps, items with keys, halves joined
    float* const join = reinterpret_cast<float*>(sp + Sh::kJoin) + row * 64;
    float* const join_ml = reinterpret_cast<float*>(sp + Sh::kJoinMl) + row * 2;
    bool ok = true;
    for (uint32_t i = 0; ok; ++i) {
      if (!mbar_wait_warp(bar(ITEM_FULL + (i & 1)), (i >> 1) & 1, abort_flag, p.status, kWaitNs)) break;
      Item it = *item_at(i);
      it.last = (int)warp_uniform(it.last); it.n = (int)warp_uniform(it.n); it.n0 = (int)warp_uniform(it.n0);
      it.dual = (int)warp_uniform(it.dual); it.part = (int)warp_uniform(it.part);
      if (lane == 0) mbar_arrive(bar(ITEM_EMPTY + (i & 1)));
      if (it.last) break;
      // this warp's copies out have read their room: where a lone tile's sums will be handed over
      if (!it.dual && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      const int t = (row >> p.pack_log2) + (it.dual ? w * tile_tokens : 0);      // token of the item
      const bool valid = t < it.q_left;
      const bool live = __any_sync(0xffffffffu, valid);
      const int mine = valid ? seen(it, causal, t) : it.keys;
      const int least = __reduce_min_sync(0xffffffffu, mine);
      const int tiles = it.dual && w == 0 ? it.n0 : it.n, step = it.dual ? 1 : 2;
      float m = -INFINITY, l = 0.f;          // m: the maximum that the weights are taken against
      bool first = true;
      for (int j = it.dual ? 0 : w; j < tiles; j += step) {
        if (!mbar_wait_warp(bar(S_FULL + w), ns & 1, abort_flag, p.status, kWaitNs)) { ok = false; break; }
        ++ns;
        if (live) {
          tc_fence_after();
          uint32_t s[4][32];
          const int end = mine - j * kTile;
          const bool masked = (j + 1) * kTile > least;
          float top[2] = {m, m};
#pragma unroll
          for (int h = 0; h < 2; ++h) {      // the second half is fetched while the first one's maximum is taken
            if (h == 0) {
              tmem_ld32(s_at, s[0]);
              tmem_ld32(s_at + 32, s[1]);
              tmem_wait_ld(s[0]);
              tmem_wait_ld(s[1]);
              tmem_ld32(s_at + 64, s[2]);
              tmem_ld32(s_at + 96, s[3]);
            } else {
              tmem_wait_ld(s[2]);
              tmem_wait_ld(s[3]);
              if (!Sh::kWide) {              // S may be made anew
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(S_READ + w));
              }
            }
            if (masked) {                    // columns that this row does not see
#pragma unroll
              for (int b = 2 * h; b < 2 * h + 2; ++b) {
                if (Sh::kWide && (b + 1) * 32 <= least - j * kTile) continue;      // (narrow: 131 us became 137)
                const int left = end - b * 32;
                const uint32_t visible = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if ((visible & (1u << e)) == 0) s[b][e] = 0xff800000u;
              }
            }
#pragma unroll
            for (int b = 2 * h; b < 2 * h + 2; ++b)
#pragma unroll
              for (int e = 0; e < 32; e += 2)
                top[b & 1] = max_nan(top[b & 1], __uint_as_float(s[b][e]), __uint_as_float(s[b][e + 1]));
          }
          const float high = max_nan(top[0], top[1], top[1]);
          if (!Sh::kWide && j >= step) {     // O and P of the step before are done with (wide: known from S)
            ok = mbar_wait_warp(bar(O_FULL + w), no & 1, abort_flag, p.status, kWaitNs);
            ++no;
            tc_fence_after();
          }
          // NaN: yes.  Rows behind the sequence are its neighbours' and have no say: a result's bits are its request's own
          if (__any_sync(0xffffffffu, valid && !((high - m) * c2 <= kRescale))) {
            const float keep = m == -INFINITY ? 0.f : exp2_fast((m - high) * c2);
            m = high;
            l *= keep;
            if (!first) {
#pragma unroll 1
              for (int b = 0; b < DP / 16; ++b) {
                uint32_t o[16];
                tmem_ld16(o_at + b * 16, o);
                tmem_wait_ld16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st16(o_at + b * 16, o);
              }
            }
          }
          // a row whose maximum is infinite or NaN is NaN: the weights of the special-function unit are
          const float base = m == -INFINITY ? 0.f : fabsf(m) < INFINITY ? -m * c2 : __uint_as_float(0x7fc00000u);
          const uint64_t scale2 = f32x2(c2, c2), base2 = f32x2(base, base);
          uint64_t sum[2] = {f32x2(0.f, 0.f), f32x2(0.f, 0.f)};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t weights[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const uint32_t* const pair = &s[2 * h + (e >> 4)][2 * (e & 15)];
              const uint64_t t = fma2(f32x2(__uint_as_float(pair[0]), __uint_as_float(pair[1])), scale2, base2);
              const uint64_t w2 = e % 8 < kPolynomials ? exp2_polynomial(t) : exp2_unit(t);
              float x, y;
              halves_of(w2, x, y);
              sum[e & 1] = add2(sum[e & 1], w2);
              weights[e] = bf16_pair(x, y);
            }
            tmem_st32(p_at + h * 32, weights);
          }
          float x, y;
          halves_of(add2(sum[0], sum[1]), x, y);
          l += x + y;
          tmem_wait_st();
          first = false;
        } else {
          if (!Sh::kWide && lane == 0) mbar_arrive(bar(S_READ + w));
          if (!Sh::kWide && j >= step) {
            ok = ok && mbar_wait_warp(bar(O_FULL + w), no & 1, abort_flag, p.status, kWaitNs);
            ++no;
          }
        }
        if (!ok) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL + w));
      }
      if (!ok) break;
      const bool any = (it.dual ? 0 : w) < tiles;
      if (any) {
        if (!mbar_wait_warp(bar(O_FULL + w), no & 1, abort_flag, p.status, kWaitNs)) break;
        ++no;
        tc_fence_after();
      }
      if (!live) continue;
      // one tile's keys were taken in turn: the second warpgroup hands over its sums, 64 columns at a time
      const bool joined = !it.dual && it.n > 1;
      if (!it.dual && w == 1) {
        if (!joined) continue;
#pragma unroll 1
        for (int h = 0; h < Sh::kHalves && ok; ++h) {
          uint32_t o[2][32];
          tmem_ld32(o_at + h * 64, o[0]);
          tmem_ld32(o_at + h * 64 + 32, o[1]);
          tmem_wait_ld(o[0]);
          tmem_wait_ld(o[1]);
          ok = mbar_wait_warp(bar(JOIN_EMPTY + quarter), (nj & 1) ^ 1, abort_flag, p.status, kWaitNs);
          if (!ok) break;
          ++nj;
          if (h == 0) *reinterpret_cast<float2*>(join_ml) = make_float2(m, l);
          // 16-byte pieces, shifted by the row so that the lanes of a warp fall on different banks
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint32_t* u = &o[e >> 3][4 * (e & 7)];
            *reinterpret_cast<uint4*>(join + ((e ^ (row & 15)) << 2)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(JOIN_FULL + quarter));
        }
        continue;
      }
      const int64_t token = (int64_t)it.q_row + t;
      const int head = it.head + (row & ((1 << p.pack_log2) - 1));
      const int64_t slot = ((int64_t)max(it.part, 0) * a.tokens_q + token) * a.heads + head;
      // rows leave through shared memory, 128 bytes of each at a time, so that a store covers 4 rows' lines and not 32
      uint8_t* const stage = sp + Sh::kJoin + quarter * 8192 + w * 4096;
      if (w == 1 && !mbar_wait_warp(bar(JOIN_EMPTY + quarter), (nj & 1) ^ 1, abort_flag, p.status, kWaitNs)) break;      // its own sums have been read
      // first token of the warp's rows; rows of 32 real queries go by one copy, others one by one
      const int slice = (quarter * 32 >> p.pack_log2) + (it.dual ? w * tile_tokens : 0);
      const bool whole = p.pack_log2 <= 5 && slice + (32 >> p.pack_log2) <= it.q_left;
      float inv = 0.f, scale0 = 1.f, scale1 = 0.f;
      bool finite = true;
#pragma unroll 1
      for (int h = 0; h < Sh::kHalves; ++h) {
        uint32_t o[2][32];
        if (any) {
          tmem_ld32(o_at + h * 64, o[0]);
          tmem_ld32(o_at + h * 64 + 32, o[1]);
          tmem_wait_ld(o[0]);
          tmem_wait_ld(o[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 64; ++e) o[e >> 5][e & 31] = 0u;
        }
        if (joined) {
          ok = mbar_wait_warp(bar(JOIN_FULL + quarter), nj & 1, abort_flag, p.status, kWaitNs);
          if (!ok) break;
          ++nj;
          if (h == 0) {
            const float2 ml = *reinterpret_cast<const float2*>(join_ml);
            const float high = fmaxf(m, ml.x);
            scale0 = m == -INFINITY ? 0.f : exp2_fast((m - high) * c2);
            scale1 = ml.x == -INFINITY ? 0.f : exp2_fast((ml.x - high) * c2);
            l = l * scale0 + ml.y * scale1;
            m = high;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint4 v = *reinterpret_cast<const uint4*>(join + ((e ^ (row & 15)) << 2));
            const uint32_t* const u = &v.x;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              uint32_t& x = o[e >> 3][4 * (e & 7) + f];
              x = __float_as_uint(fmaf(__uint_as_float(u[f]), scale1, __uint_as_float(x) * scale0));
            }
          }
          __syncwarp();
        }
        if (h * 64 + 64 > a.dim)             // columns of tensor memory that no product writes may hold anything
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (h * 64 + e >= a.dim) o[e >> 5][e & 31] = 0u;
        // a chunk whose keys all score -inf: its sums, zeros, as they are, since the chunks are joined with a weight of zero for it
        if (h == 0) inv = mine == 0 ? 0.f : SPLIT && it.part >= 0 && m == -INFINITY ? 1.f : 1.0f / l;
        const uint64_t inv2 = f32x2(inv, inv);
        uint64_t odd2 = f32x2(0.f, 0.f);     // NaN if a value is not finite
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          uint32_t* const u = &o[e >> 4][2 * (e & 15)];
          const uint64_t v = mul2(f32x2(__uint_as_float(u[0]), __uint_as_float(u[1])), inv2);
          odd2 = fma2(v, f32x2(0.f, 0.f), odd2);
          float x, y;
          halves_of(v, x, y);
          u[0] = __float_as_uint(x);
          u[1] = __float_as_uint(y);
        }
        float odd0, odd1;
        halves_of(odd2, odd0, odd1);
        if (mine > 0) {
          finite = finite && odd0 + odd1 == 0.f;
        } else {                             // a row that sees nothing: zeros, whatever was multiplied by none of its weights
#pragma unroll
          for (int e = 0; e < 64; ++e) o[e >> 5][e & 31] = 0u;
        }
        if (!SPLIT || it.part < 0) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");    // the last copy from here has read it
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float* const f = reinterpret_cast<const float*>(&o[e >> 2][8 * (e & 3)]);
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                make_uint4(bf16_pair(f[0], f[1]), bf16_pair(f[2], f[3]), bf16_pair(f[4], f[5]), bf16_pair(f[6], f[7]));
          }
          if (whole) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&map_o, h * 64, it.head, it.q_row + slice, sm + (uint32_t)(stage - sp));
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int r = e * 4 + (lane >> 3), piece = lane & 7, rr = quarter * 32 + r;
              const int tt = (rr >> p.pack_log2) + (it.dual ? w * tile_tokens : 0), d = h * 64 + piece * 8;
              const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
              if (tt < it.q_left && d < a.dim)
                *reinterpret_cast<uint4*>(a.out + ((int64_t)it.q_row + tt) * a.out_token + (int64_t)(it.head + (rr & ((1 << p.pack_log2) - 1))) * a.out_head + d) = v;
            }
          }
        } else if constexpr (SPLIT) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
#pragma unroll
          for (int g = 0; g < 2; ++g) {      // fp32: 32 columns of 32 rows at a time
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) = make_uint4(o[g][4 * e], o[g][4 * e + 1], o[g][4 * e + 2], o[g][4 * e + 3]);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int r = e * 4 + (lane >> 3), piece = lane & 7, rr = quarter * 32 + r;
              const int tt = (rr >> p.pack_log2) + (it.dual ? w * tile_tokens : 0), d = h * 64 + g * 32 + piece * 4;
              const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
              if (tt < it.q_left && d < a.dim)
                *reinterpret_cast<uint4*>(p.split.part_o + (((int64_t)it.part * a.tokens_q + it.q_row + tt) * a.heads + it.head + (rr & ((1 << p.pack_log2) - 1))) * a.dim + d) = v;
            }
          }
        }
        __syncwarp();
        if (joined && lane == 0) {           // the copy has read what the next half will overwrite
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          mbar_arrive(bar(JOIN_EMPTY + quarter));
        }
      }
      if (!ok) break;
      if (valid) {
        const float le = mine > 0 ? fmaf(m, a.scale, log2_fast(l) * 0.693147180559945f) : -INFINITY;
        if (SPLIT && it.part >= 0) p.split.part_lse[slot] = le;
        else if (a.lse != nullptr) a.lse[token * a.heads + head] = le;
      }
      // a value that is not finite may have come in with a weight of zero: from keys that other rows of the tile see, or
      // that share an instruction with them
      __syncwarp();                          // the rows as they are lie in front of the ones made again
      if (__any_sync(0xffffffffu, valid && !finite)) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
        const int most = seen(it, causal, min(it.q_left, (it.dual && w == 1 ? 2 : 1) * tile_tokens) - 1);
        redo_rows(a, p.split, it.k_row, it.kv_head, SPLIT ? it.part : -1, token, head, mine, valid && !finite, min((most + 15) & ~15, it.keys), 0, DP);
      }
    }
  }
  if (warp < kMmaWarp && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  // ---- common exit: every thread arrives here, also after an aborted wait
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

struct Tiles {
  int pack_log2, groups;
  int64_t items;
};
Tiles tiles_of(const AttnParams& a) {
  Tiles t = {};
  const int group = a.heads / a.kv_heads;
  while (t.pack_log2 < 7 && group % (2 << t.pack_log2) == 0) ++t.pack_log2;
  t.groups = a.heads >> t.pack_log2;
  const int64_t pair_tokens = 2 * (kTile >> t.pack_log2);
  const int64_t pairs = a.tokens_q / pair_tokens + (a.tokens_q < a.sequences ? a.tokens_q : a.sequences);   // at most
  t.items = pairs * t.groups;
  return t;
}

}  // namespace

// Cutting keys up costs a second kernel and fp32 parts that are written and read (the longest item of a call is shorter then, nothing
// else): 9 us and 8 bytes an element and part at 5 TB/s.  A step of 128 keys takes 0.9 us, of two tiles 2.  Measured, without and with
// chunks of 8 tiles: 1 x 64 queries to 16,384 keys, 16 / 8 heads, 118 and 27 us; 4 x 100 to 4,000, 8 heads, 37 and 24; 8 x 33 to
// 2,000, 16 / 8 heads, 23 and 24; prompts of 2,048, 16 / 8 heads, 37 and 64; 2,517, 12 heads, 45 and 82.
AttnSplit attention_tmem_split(const AttnParams& a, void* workspace) {
  const Tiles t = tiles_of(a);
  const double tiles = (double)((a.tokens_k + kKeyTile - 1) / kKeyTile), average = ceil(tiles / a.sequences);
  const double longest = a.sequences == 1 ? tiles : fmin(tiles, 2 * average);
  const bool pairs = a.tokens_q > (int64_t)a.sequences * (kTile >> t.pack_log2), half = a.causal && 2 * a.tokens_q > a.tokens_k;
  const double step = pairs ? 2.0 : 0.9, share = (double)t.items * average * (half ? 0.5 : 1.0) / device_sms();
  const double part = (double)a.tokens_q * a.heads * a.dim * 8 / 5e6;
  double best = 0.85 * step * fmax(longest, share);
  int64_t chunk = 0;
  for (int64_t c = 8; c < longest; c *= 2) {
    const double us = step * fmax((double)c, share) + 9 + part * ceil(average / (double)c);
    if (us < best) {
      best = us;
      chunk = c;
    }
  }
  return attention_chunks(a, chunk, workspace);
}

int launch_attention_tmem(const AttnParams& a, const AttnSplit& split, cudaStream_t s) {
  const Tiles t = tiles_of(a);
  TmemAttnParams p = {};
  p.a = a;
  p.pack_log2 = t.pack_log2;
  p.groups = t.groups;
  p.split = split;
  p.status = attention_status_word();
  if (p.status == nullptr) return set_error(SACQ_ERR_CUDA, "no status word on this device");
  const int64_t most = t.items * split.chunks_most;
  CUtensorMap mq, mk, mv, mo;
  const int pack = 1 << t.pack_log2;
  if (int rc = attention_tensor_maps(a, pack, kTile / pack, kTile, &mq, &mk, &mv)) return rc;
  if (int rc = attention_out_map(a, pack < 32 ? pack : 32, pack < 32 ? 32 / pack : 1, &mo)) return rc;
  const bool wide = a.dim > 64;
  const bool cut = split.chunks_most > 1;
  const void* fn = wide ? (cut ? (const void*)attention_tmem_kernel<128, true> : (const void*)attention_tmem_kernel<128, false>)
                        : (cut ? (const void*)attention_tmem_kernel<64, true> : (const void*)attention_tmem_kernel<64, false>);
  const size_t smem = (wide ? Shape<128>::kTotal : Shape<64>::kTotal) + 1024;
  static bool configured[2][2][64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[wide][cut][dev]) {
    SACQ_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev >= 0 && dev < 64) configured[wide][cut][dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  // Items differ in length (a causal prompt's last tile has all its keys): CTAs that take the next one when they are done
  // end together (two prompts of 8192 and 6001: 412 against 446 us).  Not with chunks, of which there can be many more than there are.
  p.dynamic = split.chunks_most == 1 && most > device_sms() && most <= 2147483647;
  cfg.gridDim = dim3((unsigned)(p.dynamic || most < device_sms() ? most : device_sms()));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&mq, &mk, &mv, &mo, &p};
  SACQ_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
  count_launch();
  return SACQ_OK;
}

}  // namespace sacq
