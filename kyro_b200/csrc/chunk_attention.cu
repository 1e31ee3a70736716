// chunk_attention.cu -- attention of a packed batch of prompt chunks over
// the paged cache (PagedAttention::forward, src/model/attention_kernel.rs:
// 22-136, for chunks of any length), on the sm_100 tensor cores.
//
// For row r = (token j, head h) of sequence b, over the slots t <= ctx + j:
//     s_t = scale q_r . k_t,  m = max s_t,  l = sum exp(s_t - m),
//     o_r = sum exp(s_t - m) v_t / l,  lse_r = m + log l,
// in one pass over the slots with a running m, l and o.
//
// The rows of a sequence that read one KV head are packed token-major (head
// in group fastest) into tiles of 128 rows, as many whole tokens as fit; an
// item is two such tiles against 128 slots at a time.  One CTA per SM walks
// its share of the items (chunk.cuh): the work is cut into equal stretches
// whatever the lengths are, and an item that crosses a border leaves partial
// sums that chunk_combine_kernel joins, in the order of the slots.  Warps:
//   0-3, 4-7  the softmax of tile 0 and of tile 1, one row per thread (its
//             TMEM lane): mask, running max and sum, P = exp2(s - m) over the
//             scores as bf16 in two halves of 64 slots, the rescale of O when
//             the max has grown by more than 2^8, the epilogue
//   8         walks the CTA's pieces, for all; K by TMA (128-byte swizzle), a
//             page and 64 dims at a time, into the ring that it shares with V.
//             A copy takes a warp about 75 cycles to issue, so V has a warp of
//             its own.
//   9, 10     the matrix instructions of tile 0 and of tile 1: S_h = Q_h K^T,
//             O_h += P_h V with P read from TMEM.  With two tiles of rows
//             they take turns, O_0 S_0' and then O_1 S_1', so that one tile's
//             softmax runs under the other's products (without turns both
//             tiles fall into step and compete for the same pipes: 4770 cycles
//             a step); while one issues, the other does its waiting (one
//             thread for both took 3870, now 3500 to 3700).  Warp 9 owns the
//             TMEM.
//   11        V by TMA, a whole page at a time, and the tiles of Q (a box of
//             64 dims x the group's heads x the tile's tokens; any row stride)
// In an item of one tile both softmax groups are at work too: they take the
// tiles of slots in turn, each with an m, l and O of its own, and group 0
// joins the two at the end (the rows of both lie in the same TMEM lanes).
// Without that a step would be one chain, S -> softmax -> O.
// Warps 8-11 hand most of their registers to the softmax warps.
// Slots past the item's last visible one are not loaded; their rows of V in
// shared memory are set to zero first, since 0 * NaN would reach O.
//
// What bounds it: a step's two tiles cost 2048 cycles of matrix instructions
// at D = 128 (1024 at D = 64) and 2048 of exponentials on the special-function
// unit, and it takes 3500 to 3700; an item costs 5400 beside its steps (2000
// of them the stores of its rows), a call 7 us beside its items.  4096 rows
// over 16384 slots, 64 heads of 128: 1.87 to 1.93 ms in calls one after the
// other, 1.00 to 1.03 PFLOP/s, as the clock goes under the power limit; 12
// prompts of up to 1500 tokens, 28 heads: 161 us; 16 sequences of up to 8 new
// tokens and 4096 slots, 32 heads: 37 us, 3.4 TB/s.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "chunk.cuh"
#include "f32x2.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace {

using namespace kyro::tc;
using kyro::chunk::PartDesc;
using kyro::chunk::Piece;
using kyro::chunk::Pieces;
using kyro::chunk::Seq;
using kyro::chunk::Shape;

constexpr int kBS = 16;                // tokens per KV block
constexpr int kTM = 128;               // rows per tile
constexpr int kItemRows = 2 * kTM;     // rows per item, padding rows among them
constexpr int kTN = 128;               // slots per tile
constexpr int kPages = kTN / kBS;      // 8
constexpr int kThreads = 384;
constexpr int kKWarp = 8, kMmaWarp = 9, kVWarp = 11;  // matrix warps 9 and 10
constexpr int kMaxCtas = kyro::chunk::kMaxCtas;
constexpr uint32_t kSlab = 128 * 128;  // 128 rows of 64 dims (Q, K)
constexpr uint32_t kPageSlab = kBS * 128;  // a page's 64 dims (V)
constexpr uint32_t kTmemCols = 512;    // S_h at h * 128, O_h at 256 + h * D
constexpr uint32_t kColO = 256;
// no CTA is given fewer steps than this.  Few or short chunks (the first 16
// attention batches of at most 512 rows that perf/operators.py's
// draw(random.Random(s)) gives for s = 0, 1, ..) take 15.4 us in the geometric
// mean, 17.1 with 2 and 19.2 with 4; nothing changes where there is work for
// all CTAs.
constexpr int kMinSteps = 1;
// what an item of two tiles, or one, costs beside its tiles of slots, in the
// eighths of a slot that AttnPolicy counts in
constexpr int kItemCost2 = 2560, kItemCost1 = 1600;

template <int D>
struct Geo {
  static constexpr int kSlabs = D / 64;
  static constexpr uint32_t kTile = kSlabs * kSlab;   // 128 rows x D
  static constexpr int kSlots = D == 128 ? 5 : 10;    // ring tiles (160 KB)
  static constexpr uint32_t kOffQ = kSlots * kTile;   // Q tile h at + h * kTile
  static constexpr uint32_t kTiles = kOffQ + 2 * kTile;
  static constexpr uint32_t kSmem = kTiles + 704 + 1024 + 1024;  // + barriers, group 1's m and l, alignment slack
};

struct ChunkAttnArgs {
  Shape sh;
  int hq, num_blocks;
  float scale_log2;
  int64_t os;
};

// Items of a KV head (two tiles of sh.tokens tokens), and the tiles of slots
// an item sees.  An item's cost is the slots it sees, in eighths: a tile of
// slots takes 3500 to 3700 cycles against two tiles of rows, and 2200 against
// one (the last item of a chunk may have one).
struct AttnPolicy {
  static __device__ __forceinline__ int prepare(const Seq&, const Shape&) { return 0; }
  static __device__ __forceinline__ int count(const Seq& s, const Shape& sh) {
    return (s.n + 2 * sh.tokens - 1) / (2 * sh.tokens);
  }
  static __device__ __forceinline__ int slots(const Seq& s, const Shape& sh, int t) {
    return s.ctx + min((t + 1) * 2 * sh.tokens, s.n);
  }
  static __device__ __forceinline__ int tiles(const Seq& s, const Shape& sh, int t) {
    return (slots(s, sh, t) + kTN - 1) / kTN;
  }
  static __device__ __forceinline__ int weight(const Seq& s, const Shape& sh, int t) {
    return s.n - t * 2 * sh.tokens > sh.tokens ? 8 : 5;
  }
  static __device__ __forceinline__ constexpr int kUnit(const Shape&) { return 8 * kTN; }
  static __device__ __forceinline__ int unit(const Seq& s, const Shape& sh, int t) {
    return weight(s, sh, t) * kTN;
  }
  static __device__ __forceinline__ int over(const Seq& s, const Shape& sh, int t) {
    return weight(s, sh, t) == 8 ? kItemCost2 : kItemCost1;
  }
  static __device__ __forceinline__ int cost(const Seq& s, const Shape& sh, int t) {
    return slots(s, sh, t) * weight(s, sh, t) + over(s, sh, t);
  }
  static __device__ __forceinline__ long long before(const Seq& s, const Shape& sh, int t) {
    // t items of ctx + step, ctx + 2 step, ..
    const int step = 2 * sh.tokens;
    const long long sum = (long long)t * (8ll * s.ctx + kItemCost2) +
                          8ll * step * ((long long)t * (t + 1) / 2);
    // but the chunk's last item ends at n, and may be of one tile
    if (t * step < s.n) return sum;
    return sum - (8ll * (s.ctx + t * step) + kItemCost2) + cost(s, sh, t - 1);
  }
};
using Walker = kyro::chunk::Walker<AttnPolicy>;

// workspace: descs [G][2], then (m, l) [G][2][2][256], then O [G][2][D/4][256] float4
constexpr size_t kDescBytes = (size_t)kMaxCtas * 2 * sizeof(PartDesc);
constexpr size_t kMlBytes = (size_t)kMaxCtas * 2 * 2 * kItemRows * 4;
constexpr size_t part_bytes(int d) { return (size_t)kMaxCtas * 2 * kItemRows * d * 4; }

// 64 scores of this thread's row; the ones from column `vis` on are masked.
__device__ __forceinline__ void load_scores(uint32_t addr, int vis, uint32_t (&x)[64]) {
  tmem_ld32(addr, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
  tmem_ld32(addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&x[32]));
  tmem_ld_wait();
  if (__any_sync(0xffffffffu, vis < 64)) {
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (i >= vis) x[i] = 0xff800000u;  // -inf
  }
}

// P = 2^(s * sl2 - m) for 64 scores (one half of a row's tile), written as
// bf16 pairs over 32 TMEM columns at pc; returns their sum.  (A share of the
// exponentials as polynomials on the FMA pipes gains nothing: a scheduler has
// two softmax warps, and what counts is the length of their chains.)
__device__ __forceinline__ float exp_half(const uint32_t (&x)[64], float sl2, float nref,
                                          uint32_t pc) {
  namespace fx = kyro::fx2;
  const fx::f2 sl = fx::pack(sl2, sl2), nr = fx::pack(nref, nref);
  fx::f2 sum[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      fx::f2 y = fx::fma(fx::pack(__uint_as_float(x[c * 32 + 2 * i]),
                                  __uint_as_float(x[c * 32 + 2 * i + 1])),
                         sl, nr);
      float lo, hi;
      fx::unpack(y, lo, hi);
      lo = kyro::ptx::fast_exp2(lo);
      hi = kyro::ptx::fast_exp2(hi);
      sum[i & 1] = fx::add(sum[i & 1], fx::pack(lo, hi));
      // P rounds to bf16 for the product with V; its sum does not
      pk[i] = kyro::ptx::pack_bf16x2(lo, hi);
    }
    tmem_st16(pc + c * 16, pk);
  }
  float lo, hi;
  fx::unpack(fx::add(sum[0], sum[1]), lo, hi);
  return lo + hi;
}

__device__ __forceinline__ float row_max64(const uint32_t (&x)[64]) {
  float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 64; i += 4)
#pragma unroll
    for (int v = 0; v < 2; ++v)
      m[v] = fmax3(m[v], __uint_as_float(x[i + 2 * v]), __uint_as_float(x[i + 2 * v + 1]));
  return fmaxf(m[0], m[1]);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_attention_kernel(const __grid_constant__ CUtensorMap tmQ,
                       const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const ChunkAttnArgs a,
                       const int32_t* __restrict__ starts,
                       const int64_t* __restrict__ block_table,
                       const int64_t* __restrict__ context_lens, __nv_bfloat16* __restrict__ out,
                       float* __restrict__ lse, PartDesc* __restrict__ descs,
                       float* __restrict__ part_ml, float4* __restrict__ part_o,
                       uint32_t* status) {
  using G = Geo<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = kyro::ptx::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + G::kTiles;
  auto slot_full = [&](int s) { return bar0 + 8u * s; };
  auto slot_empty = [&](int s) { return bar0 + 8u * (G::kSlots + s); };
  const uint32_t bar1 = bar0 + 16u * G::kSlots;
  auto q_full = [&](int h) { return bar1 + 8u * h; };
  auto q_empty = [&](int h) { return bar1 + 8u * (2 + h); };
  auto s_full = [&](int h) { return bar1 + 8u * (4 + h); };
  auto o_done = [&](int h) { return bar1 + 8u * (6 + h); };
  auto o_free = [&](int h) { return bar1 + 8u * (8 + h); };
  auto p_full = [&](int h, int half) { return bar1 + 8u * (10 + 2 * h + half); };
  const uint32_t mma_done = bar1 + 8u * 14;
  const uint32_t ml_full = bar1 + 8u * 15;  // group 1's m and l are in sh_ml
  auto turn = [&](int h) { return bar1 + 8u * (16 + h); };  // matrix warp h may go
  auto over = [&](int h) { return bar1 + 8u * (18 + h); };  // all that matrix warp h issued is done
  // ring item n (K tiles even, V tiles odd) lives in slot n % kSlots; its
  // fill is that slot's phase n / kSlots
  auto item_slot = [](int n) { return n % G::kSlots; };
  auto item_parity = [](int n) { return (uint32_t)((n / G::kSlots) & 1); };
  auto item_addr = [&](int n) { return base + (uint32_t)(n % G::kSlots) * G::kTile; };
  const uint32_t piece_bars = bar1 + 8u * 20;
  static_assert(16 * G::kSlots + 8 * 20 + 16 * kyro::chunk::kPieceSlots <= 400, "barriers");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + G::kTiles + 400);
  int* err = reinterpret_cast<int*>(gbase + G::kTiles + 404);
  Piece* piece_slots = reinterpret_cast<Piece*>(gbase + G::kTiles + 416);
  static_assert(416 + sizeof(Piece) * kyro::chunk::kPieceSlots <= 704, "pieces");
  float* sh_ml = reinterpret_cast<float*>(gbase + G::kTiles + 704);  // [2][128]
  // (before the first join, sh_ml is locate()'s)
  auto* scratch = reinterpret_cast<kyro::chunk::Scratch<kThreads>*>(sh_ml);
  static_assert(sizeof(*scratch) <= 1024, "scratch");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < G::kSlots; ++i) {
      kyro::ptx::mbar_init(slot_full(i), 1);
      kyro::ptx::mbar_init(slot_empty(i), 2);  // both matrix warps
    }
    for (int i = 0; i < 2; ++i) {
      kyro::ptx::mbar_init(q_full(i), 1);
      kyro::ptx::mbar_init(q_empty(i), 2);
      kyro::ptx::mbar_init(s_full(i), 1);
      kyro::ptx::mbar_init(o_done(i), 1);
      kyro::ptx::mbar_init(o_free(i), 4);
      kyro::ptx::mbar_init(p_full(i, 0), 4);
      kyro::ptx::mbar_init(p_full(i, 1), 4);
    }
    kyro::ptx::mbar_init(mma_done, 2);
    kyro::ptx::mbar_init(ml_full, 4);
    kyro::ptx::mbar_init(turn(0), 1);
    kyro::ptx::mbar_init(turn(1), 1);
    kyro::ptx::mbar_init(over(0), 1);
    kyro::ptx::mbar_init(over(1), 1);
    Pieces::init(piece_bars, kThreads / 32 - 1);
    *err = 0;
    kyro::ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc1(kyro::ptx::smem_addr(tmem_slot), kTmemCols);
    tmem_relinquish1();
  }
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  kyro::chunk::locate<AttnPolicy, kThreads>(a.sh, starts, context_lens, kMinSteps, status, scratch);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int group = a.sh.group, tokens = a.sh.tokens;
  Pieces pieces(piece_bars, piece_slots, err, status);
  Piece p;
  // the register split: 88 x 128 + 208 x 256 = the 168 x 384 of the launch
  if (warp >= kKWarp) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == kKWarp || warp == kVWarp) {
    // ------------------------------------------------ tiles of K, or of Q and V
    const bool is_v = warp == kVWarp;
    const CUtensorMap* map = is_v ? &tmV : &tmK;
    if (lane == 0) {
      kyro::ptx::prefetch_tensormap(map);
      if (is_v) kyro::ptx::prefetch_tensormap(&tmQ);
    }
    // this lane's part of a tile: a page (V), or 64 dims of one (K)
    const int pg = is_v ? lane : lane / G::kSlabs, slab = is_v ? 0 : lane % G::kSlabs;
    const uint32_t off = is_v ? (uint32_t)pg * kBS * D * 2 : slab * kSlab + (uint32_t)pg * kPageSlab;
    const uint32_t q_bytes = (uint32_t)(tokens * group) * D * 2;
    int q_uses[2] = {0, 0};  // fills of Q tile h
    int n = is_v;            // ring item
    bool ok = true;
    Walker walk(a.sh, starts, context_lens, scratch->start);
    auto next = [&](Piece& pc) {
      if (is_v) return pieces.get(pc);
      const bool any = walk.next(pc);
      return pieces.put(pc) && any;
    };
    // this lane's block of a tile of the piece
    auto fetch = [&](const Piece& pc, int j) -> int64_t {
      const int i = j * kPages + pg;
      return pg < kPages && i * kBS < AttnPolicy::slots(pc.s, a.sh, pc.t)
                 ? __ldg(&block_table[(int64_t)pc.b * a.sh.max_blocks + i])
                 : 0;
    };
    Piece pn;
    bool have = next(p);
    int64_t id = have ? fetch(p, p.tile0) : 0, id_n = 0;
    for (; ok && have; p = pn, id = id_n) {
      const int nblk = (AttnPolicy::slots(p.s, a.sh, p.t) + kBS - 1) / kBS;
      if (is_v) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tok0 = (p.t * 2 + h) * tokens;
          if (tok0 >= p.s.n || !ok) break;
          if (q_uses[h] > 0) ok = wait_bar_warp(q_empty(h), (q_uses[h] - 1) & 1, err, status);
          if (!ok) break;
          ++q_uses[h];
          if (lane == 0) {
            kyro::ptx::mbar_arrive_expect_tx(q_full(h), q_bytes);
            // tokens of the sequences behind this one, or zeros past the last
            // row, fill the tile: rows whose results go nowhere
            for (int s = 0; s < G::kSlabs; ++s)
              kyro::ptx::tma_load_3d(base + G::kOffQ + (uint32_t)h * G::kTile + s * kSlab, &tmQ,
                                     s * 64, p.kvh * group, p.s.start + tok0, q_full(h));
          }
        }
      }
      for (int j = p.tile0; ok && j < p.tile1; ++j, n += 2) {
        int64_t blk = id;
        if (j + 1 < p.tile1) id = fetch(p, j + 1);
        if (blk < 0 || blk >= a.num_blocks) {
          kyro::dev::flag(status, KYRO_DEV_BAD_BLOCK);
          blk = 0;
        }
        const int32_t z = (int32_t)(blk * a.sh.hkv + p.kvh);
        const int np = min(kPages, nblk - j * kPages);
        const int s = item_slot(n);
        if (n >= G::kSlots)
          ok = wait_bar_warp(slot_empty(s), item_parity(n - G::kSlots), err, status);
        ok = __all_sync(0xffffffffu, ok && !*(volatile int*)err);
        if (!ok) break;
        if (lane == 0)
          kyro::ptx::mbar_arrive_expect_tx(slot_full(s), (uint32_t)np * kBS * D * 2);
        __syncwarp();
        if (pg < np) {
          if (is_v)
            kyro::ptx::tma_load_4d(item_addr(n) + off, map, 0, 0, 0, z, slot_full(s));
          else
            kyro::ptx::tma_load_3d(item_addr(n) + off, map, slab * 64, 0, z, slot_full(s));
        }
        if (j == p.tile0) {
          // the next piece is known, and its first blocks, long before they are needed
          have = next(pn);
          if (have) id_n = fetch(pn, pn.tile0);
        }
      }
    }
    // no CTA leaves while a copy may still write its shared memory: after a
    // timeout the tiles in flight are waited for here
    __syncwarp();
    if (*(volatile int*)err && lane == 0) {
      for (int i = n - 2; i >= 0 && i >= n - G::kSlots - 1; i -= 2)
        kyro::ptx::mbar_wait_bounded(slot_full(item_slot(i)), item_parity(i), kWaitBudget);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (q_uses[h] > 0)
          kyro::ptx::mbar_wait_bounded(q_full(h), (q_uses[h] - 1) & 1, kWaitBudget);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ matrix instructions (one thread per warp)
    const int h = warp - kMmaWarp;
    if (lane == 0) {
      constexpr uint32_t idS = idesc_f16(kTM, kTN, false), idO = idesc_f16(kTM, D, true);
      constexpr uint32_t idS2 = idesc_f16(kTM, kTN / 2, false);
      int n = 0;               // ring items of the CTA
      int q_uses[2] = {0, 0};  // items that filled Q tile 0, tile 1
      int tiles[2] = {0, 0};   // tiles done by each softmax group
      int o_uses[2] = {0, 0};  // pieces that used O_0, O_1
      int turns = 0;
      bool next_in = false;    // the next K is in shared memory
      // S_1 and O_1 are warp 10's in items of two tiles and warp 9's in items
      // of one.  Products of different threads are in no order, so where the
      // kind of item changes, the new owner waits for the old one's.
      bool was_two = true;
      int overs[2] = {0, 0};
      auto hand_over = [&](bool two) {
        if (two == was_two) return true;
        was_two = two;
        const int from = two ? 0 : 1;
        const int k = overs[from]++;
        if (h == from) {
          umma1_commit(over(from));
          return true;
        }
        return wait_bar(over(from), k & 1, err, status);
      };
      bool ok = true;
      auto wait_slot = [&](int item) {
        return wait_bar(slot_full(item_slot(item)), item_parity(item), err, status);
      };
      // warp 0's k-th turn comes after warp 1's (k-1)-th, and warp 1's k-th
      // after warp 0's k-th
      auto my_turn = [&]() {
        const int k = turns++ - (h == 0);
        return k < 0 || wait_bar(turn(h), k & 1, err, status);
      };
      // S_g = Q_qg K^T of ring item `item`; half: of its first 64 slots
      auto s_mma = [&](int g, int qg, int item, bool half) {
        const uint32_t id = half ? idS2 : idS;
        tc_fence_after();
        const uint32_t kd = desc_lo(item_addr(item), 16);
        const uint32_t qd = desc_lo(base + G::kOffQ + (uint32_t)qg * G::kTile, 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((uint32_t)(k >> 2) * kSlab + (uint32_t)(k & 3) * 32) >> 4;
          umma1_ss(tmem + (uint32_t)g * 128, qd + off, kd + off, id, k > 0 ? 1u : 0u);
        }
      };
      // O_g (+)= P_g V of ring item `item`, as the halves of P come in; what
      // can be waited for before this warp's turn is
      auto o_mma = [&](int g, int item, int next, bool first, bool in_turn, bool half) -> bool {
        if (!wait_slot(item)) return false;
        // the last piece's O_g has been read
        if (first && o_uses[g] > 0 && !wait_bar(o_free(g), (o_uses[g] - 1) & 1, err, status))
          return false;
        if (!wait_bar(p_full(g, 0), tiles[g] & 1, err, status)) return false;
        // the rest is seen to be there already, or waited for in the turn
        const bool p1 = kyro::ptx::mbar_test_wait(p_full(g, 1), tiles[g] & 1);
        next_in =
            next >= 0 && kyro::ptx::mbar_test_wait(slot_full(item_slot(next)), item_parity(next));
        if (in_turn && !my_turn()) return false;
        tc_fence_after();
        const uint32_t vd = desc_lo(item_addr(item), kPageSlab);
        const uint32_t sd = tmem + (uint32_t)g * 128, od = tmem + kColO + (uint32_t)g * D;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma1_ts(od, sd + (uint32_t)k * 8, vd + (((uint32_t)k * kBS * D * 2) >> 4), idO,
                   (!first || k > 0) ? 1u : 0u);
        if (!p1) {
          if (!wait_bar(p_full(g, 1), tiles[g] & 1, err, status)) return false;
          tc_fence_after();
        }
        if (!half) {
#pragma unroll
          for (int k = 4; k < 8; ++k)
            umma1_ts(od, sd + (uint32_t)k * 8, vd + (((uint32_t)k * kBS * D * 2) >> 4), idO, 1u);
        }
        umma1_commit(o_done(g));
        ++tiles[g];
        return true;
      };
      while (ok && pieces.get_alone(p)) {
        const int J = p.tile1 - p.tile0;
        const int end = AttnPolicy::slots(p.s, a.sh, p.t) - p.tile0 * kTN;
        auto half = [&](int j) { return end - j * kTN <= kTN / 2; };
        // Both matrix warps wait for every fill and answer for it, of the ring
        // and of Q, whoever reads it: so neither can be a fill behind, where
        // a phase's parity would be taken for that of another.
        const bool two = p.s.n - p.t * 2 * tokens > tokens;
        ok = wait_bar(q_full(0), q_uses[0] & 1, err, status) && hand_over(two);
        if (!ok) break;
        if (two) {
          // two tiles of rows: this warp's against every tile of slots
          ok = wait_bar(q_full(1), q_uses[1] & 1, err, status) && wait_slot(n);
          if (!ok) break;
          kyro::ptx::mbar_arrive(q_empty(1 - h));
          s_mma(h, h, n, half(0));
          umma1_commit(s_full(h));
          umma1_commit(slot_empty(item_slot(n)));
          // with the last S of this piece issued, Q may be overwritten
          if (J == 1) umma1_commit(q_empty(h));
          for (int j = 0; j < J; ++j) {
            const int vi = n + 2 * j + 1, ki = vi + 1;
            ok = o_mma(h, vi, j + 1 < J ? ki : -1, j == 0, true, half(j));
            if (!ok) break;
            if (j + 1 < J) {
              if (!next_in && !(ok = wait_slot(ki))) break;
              s_mma(h, h, ki, half(j + 1));  // over P_h, which the O product above has read
              kyro::ptx::mbar_arrive(turn(1 - h));
              umma1_commit(s_full(h));
              umma1_commit(slot_empty(item_slot(vi)));
              umma1_commit(slot_empty(item_slot(ki)));
              if (j + 2 == J) umma1_commit(q_empty(h));
            } else {
              kyro::ptx::mbar_arrive(turn(1 - h));
              umma1_commit(slot_empty(item_slot(vi)));
            }
          }
          if (!ok) break;
          tiles[1 - h] += J;
          ++q_uses[0], ++q_uses[1], ++o_uses[0], ++o_uses[1];
        } else if (h == 0) {
          // one tile of rows: the groups take the tiles of slots in turn
          for (int j = 0; ok && j < min(J, 2); ++j) {
            ok = wait_slot(n + 2 * j);
            if (!ok) break;
            s_mma(j, 0, n + 2 * j, half(j));
            umma1_commit(s_full(j));
            umma1_commit(slot_empty(item_slot(n + 2 * j)));
          }
          if (ok && J <= 2) umma1_commit(q_empty(0));
          for (int j = 0; ok && j < J; ++j) {
            const int g = j & 1, vi = n + 2 * j + 1, ki = vi + 3;
            ok = o_mma(g, vi, j + 2 < J ? ki : -1, j < 2, false, half(j));
            if (!ok) break;
            umma1_commit(slot_empty(item_slot(vi)));
            if (j + 2 < J) {
              if (!next_in && !(ok = wait_slot(ki))) break;
              s_mma(g, 0, ki, half(j + 2));
              umma1_commit(s_full(g));
              umma1_commit(slot_empty(item_slot(ki)));
              if (j + 3 == J) umma1_commit(q_empty(0));
            }
          }
          ++q_uses[0], ++o_uses[0];
          if (J > 1) ++o_uses[1];
        } else {
          // warp 0 has them all; this one lets every fill pass
          kyro::ptx::mbar_arrive(q_empty(0));
          for (int i = n; ok && i < n + 2 * J; ++i) {
            ok = wait_slot(i);
            if (ok) kyro::ptx::mbar_arrive(slot_empty(item_slot(i)));
          }
          tiles[0] += (J + 1) / 2, tiles[1] += J / 2;
          ++q_uses[0], ++o_uses[0];
          if (J > 1) ++o_uses[1];
        }
        n += 2 * J;
      }
      // every product issued is done before the TMEM is freed
      umma1_commit(mma_done);
      wait_bar(mma_done, 0, err, status);
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------ softmax of tile h, one row per thread
    const int h = warp / 4;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int row_tok = row / group, row_head = row - row_tok * group;  // of the tile
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const float sl2 = a.scale_log2;
    const uint32_t sc = tmem + lane_base + (uint32_t)h * 128;
    const uint32_t oc = tmem + lane_base + kColO + (uint32_t)h * D;
    PartDesc* my_desc = descs + (size_t)blockIdx.x * 2;
    if (threadIdx.x == 0) my_desc[0].valid = my_desc[1].valid = 0;
    int tiles = 0, n = 0;  // tiles of this group, ring items of the CTA
    int joins = 0;
    bool ok = true;
    while (ok && pieces.get(p)) {
      // one tile of rows: the groups take the tiles of slots in turn
      const bool shared = p.s.n - p.t * 2 * tokens <= tokens;
      const int tok0 = (p.t * 2 + (shared ? 0 : h)) * tokens;  // the tile's first token
      const int J = p.tile1 - p.tile0;
      const int n0 = n;
      n += 2 * J;
      if (threadIdx.x == 0 && !(p.first() && p.last())) kyro::chunk::describe(my_desc, p);
      if (shared && h >= J) {
          continue;
      }
      const int ntok = min(tokens, p.s.n - tok0);
      const bool live = quarter * 32 < ntok * group;  // a warp of padding rows only keeps the step
      const bool real = row_tok < ntok;
      const int lim = p.s.ctx + tok0 + min(row_tok, ntok - 1) + 1;  // slots this row sees
      const int lim_tile = p.s.ctx + tok0 + 1;                      // slots every row sees
      const int end = AttnPolicy::slots(p.s, a.sh, p.t);  // slots the item sees
      float m_used = -INFINITY, l = 0.0f;
      const int j0 = shared ? h : 0, step = shared ? 2 : 1;
      for (int j = j0; j < J; j += step, ++tiles) {
        const int t0 = (p.tile0 + j) * kTN;
        const int vi = n0 + 2 * j + 1;  // V's ring item
        // an item's last tile may be of 64 slots
        const int halves = end - t0 > kTN / 2 ? 2 : 1;
        if (!wait_bar_warp(s_full(h), tiles & 1, err, status)) {
          ok = false;
          break;
        }
        if (t0 + kTN > end) {
          // rows of V that no row sees may not be in the tile: zero them.
          // Only now, with this tile's scores done: the slot's earlier fills
          // are over then, and its phase cannot be mistaken for an older one.
          if (!wait_bar_warp(slot_full(item_slot(vi)), item_parity(vi), err, status)) {
            ok = false;
            break;
          }
          if (t0 + row >= end && row < 64 * halves) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                               item_addr(vi) + (uint32_t)(row / kBS) * kBS * D * 2 +
                               (uint32_t)(c >> 3) * kPageSlab + (uint32_t)(row % kBS) * 128 +
                               (uint32_t)(c & 7) * 16),
                           "r"(0)
                           : "memory");
            fence_async_shared();
          }
        }
        tc_fence_after();
        if (!live) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            kyro::ptx::mbar_arrive(p_full(h, 0));
            kyro::ptx::mbar_arrive(p_full(h, 1));
          }
          continue;
        }
        const bool whole = t0 + kTN <= lim_tile;  // no masked score in the tile
        const int vis = lim - t0;
        // The scores are read from TMEM twice, 64 columns at a time, by two
        // short loops: holding all 128 in registers means unrolled code
        // several times as long, and its instruction misses were most of a
        // short call.
        float top = -INFINITY;
#pragma unroll 1
        for (int half = 0; half < halves; ++half) {
          uint32_t x[64];
          load_scores(sc + 64 * half, whole ? 64 : vis - 64 * half, x);
          top = fmaxf(top, row_max64(x));
        }
        // scores stay raw; the log2 scale enters the max and the exp2 argument
        const float m_new = fmaxf(m_used, top * sl2);
        bool need = false;
        if (j == j0)
          m_used = m_new;
        else
          need = m_new > m_used + 8.0f;
        if (__any_sync(0xffffffffu, need)) {
          // S_h of this tile was issued after O_h of the one before, so O_h
          // is final for that one by now; the wait only confirms it
          if (!wait_bar_warp(o_done(h), (tiles - 1) & 1, err, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float alpha = need ? kyro::ptx::fast_exp2(m_used - m_new) : 1.0f;
          if (need) {
            m_used = m_new;
            l *= alpha;
          }
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(oc + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(oc + c * 32, o);
          }
          tmem_st_wait();
        }
        const float nref = m_used == -INFINITY ? 0.0f : -m_used;
        // the first half's P goes to the matrix warp while the second half
        // is computed; P of slots 64 * half.. lands on score columns 32 *
        // half.., which have been read
#pragma unroll 1
        for (int half = 0; half < halves; ++half) {
          uint32_t x[64];
          load_scores(sc + 64 * half, whole ? 64 : vis - 64 * half, x);
          l += exp_half(x, sl2, nref, sc + 32 * half);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) kyro::ptx::mbar_arrive(p_full(h, half));
        }
        if (halves == 1 && lane == 0) kyro::ptx::mbar_arrive(p_full(h, 1));
      }
      if (!ok) break;
      if (!wait_bar_warp(o_done(h), (tiles - 1) & 1, err, status)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // the other group's sums: O = f0 O_0 + f1 O_1
      const bool join = shared && J > 1;
      float f0 = 1.0f, f1 = 0.0f;
      if (join) {
        if (h == 1) {
          sh_ml[row] = m_used;
          sh_ml[kTM + row] = l;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) kyro::ptx::mbar_arrive(ml_full);
          continue;  // group 0 reads O_1 and frees it
        }
        if (!wait_bar_warp(ml_full, joins & 1, err, status)) {
          ok = false;
          break;
        }
        ++joins;
        tc_fence_after();
        const float m1 = sh_ml[row], l1 = sh_ml[kTM + row];
        const float m = fmaxf(m_used, m1), mr = m == -INFINITY ? 0.0f : m;
        f0 = kyro::ptx::fast_exp2(m_used - mr);
        f1 = kyro::ptx::fast_exp2(m1 - mr);
        l = f0 * l + f1 * l1;
        m_used = m;
      }
      if (live) {
        // 32 dims of this row's sums
        auto load_o = [&](int c, uint32_t (&o)[32]) {
          tmem_ld32(oc + c * 32, o);
          if (join) {
            uint32_t o1[32];
            tmem_ld32(oc + D + c * 32, o1);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = __float_as_uint(f0 * __uint_as_float(o[i]) + f1 * __uint_as_float(o1[i]));
          } else {
            tmem_ld_wait();
          }
        };
        if (p.first() && p.last()) {
          const float inv = l > 0.0f ? 1.0f / l : 0.0f;
          const int64_t trow = p.s.start + tok0 + row_tok;
          const int head = p.kvh * group + row_head;
          __nv_bfloat16* orow = out + trow * a.os + (int64_t)head * D;
          const bool wide = (((uintptr_t)out | (uintptr_t)(a.os * 2)) & 31) == 0;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            load_o(c, o);
            if (real) {
              uint32_t pk[16];
#pragma unroll
              for (int i = 0; i < 16; ++i)
                pk[i] = kyro::ptx::pack_bf16x2(__uint_as_float(o[2 * i]) * inv,
                                               __uint_as_float(o[2 * i + 1]) * inv);
              // a lane's row is a line of its own: the widest stores there are
              if (wide) {
                kyro::ptx::st_global_32(orow + c * 32, pk);
                kyro::ptx::st_global_32(orow + c * 32 + 16, pk + 8);
              } else {
                uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
                for (int v = 0; v < 4; ++v)
                  dst[v] = make_uint4(pk[4 * v], pk[4 * v + 1], pk[4 * v + 2], pk[4 * v + 3]);
              }
            }
          }
          if (real && lse) lse[trow * a.hq + head] = (m_used + log2f(l)) * 0.6931471805599453f;
        } else {
          const size_t slot = (size_t)blockIdx.x * 2 + (p.first() ? 1 : 0);
          const int ir = h * kTM + row;
          part_ml[slot * 2 * kItemRows + ir] = m_used;
          part_ml[slot * 2 * kItemRows + kItemRows + ir] = l;
          float4* po = part_o + slot * (D / 4) * kItemRows + ir;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            load_o(c, o);
#pragma unroll
            for (int v = 0; v < 8; ++v)
              po[(c * 8 + v) * kItemRows] =
                  make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                              __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        kyro::ptx::mbar_arrive(o_free(h));
        if (join) kyro::ptx::mbar_arrive(o_free(1));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc1(tmem, kTmemCols);
}

// Joins the pieces of the item that CTA blockIdx.x of the attention began
// and did not end: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i, the pieces
// in the order of their slots.  A block takes kJoinRows of the item's rows.
// The pieces, their m and l, and their O are each loaded together, so that
// the join waits for memory three times and not once per piece.  (A block
// costs its launch even where there is nothing to join: the 16 batches above
// kMinSteps take 15.4 us with 32 rows and 512 threads a block, 15.9 with 16 and
// 256.)
constexpr int kJoinThreads = 512;
constexpr int kJoinRows = 32;

template <int D>
__global__ void __launch_bounds__(kJoinThreads, 2)
chunk_combine_kernel(const ChunkAttnArgs a, int ctas, const int32_t* __restrict__ starts,
                     const int64_t* __restrict__ context_lens, __nv_bfloat16* __restrict__ out,
                     float* __restrict__ lse, const PartDesc* __restrict__ descs,
                     const float* __restrict__ part_ml, const float4* __restrict__ part_o) {
  __shared__ int list[kMaxCtas], count;       // the pieces' slots
  __shared__ float sm[kMaxCtas][kJoinRows];   // m, then the piece's factor
  __shared__ float sl[kMaxCtas][kJoinRows];
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  const int c0 = blockIdx.x;
  const PartDesc d = descs[c0 * 2 + 1];
  if (!d.valid) return;
  const Seq s = kyro::chunk::seq_of(d.b, starts, context_lens, a.sh.T, a.sh.max_slots);
  const int row0 = blockIdx.y * kJoinRows;  // of the item
  {
    // rows past the tile's tokens, or the chunk's, are none
    const int h = row0 / kTM;
    const int rows = min(a.sh.tokens, s.n - (d.t * 2 + h) * a.sh.tokens) * a.sh.group;
    if (row0 - h * kTM >= rows) return;
  }
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int n = 0;
    for (int c = c0; c < ctas; c += 32) {
      const int slot = (c + lane) * 2 + (c + lane == c0);
      int valid = 0, last = 0;
      if (c + lane < ctas) {
        valid = descs[slot].valid;
        last = descs[slot].last;
      }
      uint32_t mv = __ballot_sync(0xffffffffu, valid);
      const uint32_t ml = __ballot_sync(0xffffffffu, valid && last);
      if (ml) mv &= (ml & -ml) | ((ml & -ml) - 1u);  // up to the item's last piece
      if ((mv >> lane) & 1u) list[n + __popc(mv & ((1u << lane) - 1u))] = slot;
      n += __popc(mv);
      if (ml) break;
    }
    if (lane == 0) count = n;
  }
  __syncthreads();
  const int np = count;
  for (int i = threadIdx.x; i < np * kJoinRows; i += kJoinThreads) {
    const int k = i / kJoinRows, r = i % kJoinRows;
    const float* ml = part_ml + (size_t)list[k] * 2 * kItemRows + row0 + r;
    sm[k][r] = ml[0];
    sl[k][r] = ml[kItemRows];
  }
  __syncthreads();
  constexpr int kPer = kJoinThreads / kJoinRows;  // threads per row
  constexpr int kVec = D / 4 / kPer;              // 4-dim pieces per thread
  // a warp's lanes lie along the rows, as the partial sums do
  const int rr = threadIdx.x % kJoinRows, part = threadIdx.x / kJoinRows;
  const int ir = row0 + rr, h = ir / kTM, row = ir % kTM;
  const int row_tok = row / a.sh.group, row_head = row - row_tok * a.sh.group;
  const int tok = (d.t * 2 + h) * a.sh.tokens + row_tok;
  float m = -INFINITY, l = 0.0f;
  for (int k = 0; k < np; ++k) m = fmaxf(m, sm[k][rr]);
  const float mr = m == -INFINITY ? 0.0f : m;
  float4 o[kVec];
#pragma unroll
  for (int v = 0; v < kVec; ++v) o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = 0; k < np; ++k) {
    const float f = kyro::ptx::fast_exp2(sm[k][rr] - mr);
    l += f * sl[k][rr];
    const float4* po = part_o + (size_t)list[k] * (D / 4) * kItemRows + ir;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const float4 x = po[(part * kVec + v) * kItemRows];
      o[v].x += f * x.x;
      o[v].y += f * x.y;
      o[v].z += f * x.z;
      o[v].w += f * x.w;
    }
  }
  if (row_tok >= a.sh.tokens || tok >= s.n) return;
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  const int head = d.kvh * a.sh.group + row_head;
  const int64_t trow = s.start + tok;
  uint2* orow = reinterpret_cast<uint2*>(out + trow * a.os + (int64_t)head * D) + part * kVec;
#pragma unroll
  for (int v = 0; v < kVec; ++v)
    orow[v] = make_uint2(kyro::ptx::pack_bf16x2(o[v].x * inv, o[v].y * inv),
                         kyro::ptx::pack_bf16x2(o[v].z * inv, o[v].w * inv));
  if (lse && part == 0) lse[trow * a.hq + head] = (m + log2f(l)) * 0.6931471805599453f;
}

int check(const kyro_chunk_params* p) {
  const char* fn = "kyro_chunk_attention";
  KY_TRY(kyro::chunk::check_params(p, fn));
  KY_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "%s: head_dim = %d (64 or 128 supported)",
             fn, p->head_dim);
  KY_REQUIRE(p->block_size == kBS, "%s: block_size = %d (only %d supported)", fn, p->block_size,
             kBS);
  // (an item's cost is counted in eighths of a slot, in 32 bits)
  KY_REQUIRE((int64_t)p->max_blocks_per_seq * kBS <= (1ll << 27),
             "%s: a sequence may hold at most 2^27 slots", fn);
  KY_REQUIRE((int64_t)p->num_blocks * p->num_kv_heads < (1ll << 31),
             "%s: num_blocks * num_kv_heads must fit in 31 bits", fn);
  KY_REQUIRE(p->num_heads / p->num_kv_heads <= kTM,
             "%s: %d query heads per KV head (at most %d)", fn, p->num_heads / p->num_kv_heads,
             kTM);
  KY_REQUIRE(p->scale >= 0.0f && std::isfinite(p->scale), "%s: scale = %g", fn, (double)p->scale);
  const int64_t dq = (int64_t)p->num_heads * p->head_dim;
  KY_REQUIRE(kyro::chunk::stride_ok(p->q_stride, dq) && kyro::chunk::stride_ok(p->out_stride, dq),
             "%s: a row stride is shorter than its row or not a multiple of 8", fn);
  return KYRO_OK;
}

template <int D>
int launch(kyro_ctx* ctx, const kyro_chunk_params* p, const ChunkAttnArgs& a, const void* q,
           const void* k_cache, const void* v_cache, const int32_t* starts,
           const int64_t* block_table, const int64_t* context_lens, void* out, float* lse,
           void* workspace) {
  // Q [T][Hq][D]: box (64 dims, a group's heads, a tile's tokens);
  // K [blocks * Hkv][16 tokens][D]: box (64 dims, 16 tokens, 1); V: a page
  CUtensorMap mq, mk, mv;
  const int64_t qs = kyro::chunk::stride_or(p->q_stride, (int64_t)p->num_heads * D);
  KY_TRY(make_map3(&mq, q, D, (uint64_t)p->num_heads, (uint64_t)p->num_tokens, (uint64_t)D * 2,
                   (uint64_t)qs * 2, (uint32_t)a.sh.group, (uint32_t)a.sh.tokens));
  const uint64_t rows = (uint64_t)p->num_blocks * p->num_kv_heads;
  KY_TRY(make_map3(&mk, k_cache, D, kBS, rows, (uint64_t)D * 2, (uint64_t)kBS * D * 2, kBS, 1));
  KY_TRY(make_page_map(&mv, v_cache, D, rows));
  PartDesc* descs = (PartDesc*)workspace;
  float* ml = (float*)((char*)workspace + kDescBytes);
  float4* po = (float4*)((char*)workspace + kDescBytes + kMlBytes);
  const int ctas = std::min(ctx->num_sms, kMaxCtas);
  KY_TRY(kyro::chunk::set_smem<chunk_attention_kernel<D>>(Geo<D>::kSmem, ctx->device));
  KY_TRY(kyro::launch_pdl(chunk_attention_kernel<D>, dim3((unsigned)ctas), dim3(kThreads),
                          Geo<D>::kSmem, ctx->stream, "chunk_attention_kernel", mq, mk, mv,
                          a, starts, block_table, context_lens,
                          (__nv_bfloat16*)out, lse, descs, ml, po, ctx->d_status));
  // no item has more rows than the call: tokens of one tile, or two tiles
  const int most = p->num_tokens > a.sh.tokens ? kItemRows : p->num_tokens * a.sh.group;
  return kyro::launch_pdl(chunk_combine_kernel<D>,
                          dim3((unsigned)ctas, (unsigned)((most + kJoinRows - 1) / kJoinRows)),
                          dim3(kJoinThreads), 0,
                          ctx->stream, "chunk_combine_kernel", a, ctas, starts, context_lens,
                          (__nv_bfloat16*)out, lse, (const PartDesc*)descs, (const float*)ml,
                          (const float4*)po);
}

}  // namespace

extern "C" {

size_t kyro_chunk_attention_workspace_size(const kyro_chunk_params* p) {
  if (check(p) != KYRO_OK) return 0;
  return kDescBytes + kMlBytes + part_bytes(p->head_dim);
}

int kyro_chunk_attention(kyro_ctx* ctx, const kyro_chunk_params* p, const void* q,
                         const void* k_cache, const void* v_cache, const int32_t* chunk_starts,
                         const int64_t* block_table, const int64_t* context_lens, void* out,
                         float* lse, void* workspace, size_t workspace_bytes) {
  const char* fn = "kyro_chunk_attention";
  KY_NVTX("kyro_chunk_attention");
  KY_TRY(kyro::enter(ctx));
  KY_TRY(check(p));
  if (p->batch == 0 || p->num_tokens == 0) return KYRO_OK;
  KY_REQUIRE(q && k_cache && v_cache && chunk_starts && block_table && context_lens && out,
             "%s: a required pointer is NULL", fn);
  KY_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k_cache % 16 == 0 &&
                 (uintptr_t)v_cache % 16 == 0 && (uintptr_t)out % 16 == 0,
             "%s: q, the caches and out must be 16-byte aligned", fn);
  const size_t need = kyro_chunk_attention_workspace_size(p);
  if (!workspace || workspace_bytes < need)
    return kyro::set_error(KYRO_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn,
                           workspace_bytes, need);
  KY_REQUIRE((uintptr_t)workspace % 256 == 0, "%s: workspace must be 256-byte aligned", fn);
  ChunkAttnArgs a;
  a.sh.B = p->batch;
  a.sh.T = p->num_tokens;
  a.sh.hkv = p->num_kv_heads;
  a.sh.group = p->num_heads / p->num_kv_heads;
  a.sh.tokens = kTM / a.sh.group;
  a.sh.max_blocks = p->max_blocks_per_seq;
  a.sh.max_slots = p->max_blocks_per_seq * kBS;
  a.hq = p->num_heads;
  a.num_blocks = p->num_blocks;
  const float scale = p->scale > 0.0f ? p->scale : 1.0f / sqrtf((float)p->head_dim);
  a.scale_log2 = scale * 1.4426950408889634f;
  const int64_t dq = (int64_t)p->num_heads * p->head_dim;
  a.os = kyro::chunk::stride_or(p->out_stride, dq);
  if (p->head_dim == 128)
    return launch<128>(ctx, p, a, q, k_cache, v_cache, chunk_starts, block_table, context_lens,
                       out, lse, workspace);
  return launch<64>(ctx, p, a, q, k_cache, v_cache, chunk_starts, block_table, context_lens, out,
                    lse, workspace);
}

}  // extern "C"
