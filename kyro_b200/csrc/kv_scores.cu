// kv_scores.cu -- the attention weight that every cached slot receives from
// a packed batch of prompt chunks, added to its score: what eviction from
// the cache goes by.  No counterpart in the reference.
//
// For slot t of sequence b and KV head h, over the rows r = (token j, head)
// of the chunk that see it (t <= ctx + j) and read that KV head:
//     m_t = sum_r exp(scale q_r . k_t - lse_r).
//
// The scores are formed transposed, S^T = K Q^T, with the slots as the rows
// of the matrix product: a slot is then one thread's TMEM lane, its sum
// stays in that thread's registers, and no sum crosses threads or needs an
// atomic.  An item is 256 slots of one KV head, as two tiles of 128 that
// stay in shared memory, against the rows of as many whole tokens as 128 rows
// hold (head in group fastest), from the first token that sees them.  One CTA
// per SM walks its share of the items (chunk.cuh); an item that crosses a
// border leaves its sums to kv_scores_join_kernel, which adds them in the order
// of the rows.  Warps:
//   0-7, 8-15  the sums of tile 0 and of tile 1: one slot per thread and two
//              threads per slot, which take half of a step's rows each and
//              join their sums through the TMEM (with one, two warps on a
//              scheduler left half of its issue slots empty: 335-350 us for
//              2401 rows of 64 heads over 20625 slots, now 320).  All
//              exponentials are the special-function unit's: a share of them
//              as polynomials on the FMA pipes cost more issue slots than it
//              saved (322-339 us)
//   16, 19     warp 16 walks the CTA's pieces, for all; K by TMA, a page and
//              64 dims at a time (128-byte swizzle), the item's first and
//              second tile.  A copy takes a warp about 75 cycles to issue, so
//              each tile has its own.
//   17         the matrix instructions, into two score buffers per tile;
//              also owns the TMEM
//   18         the tiles of Q by TMA (a box of 64 dims x the group's heads x
//              the step's tokens; any row stride), and their lse
// What bounds it: a step's two tiles cost 1024 cycles of matrix instructions
// and 2048 of exponentials at D = 128, and take 2540; without the exponentials
// they took 2250, so the loop's waits for TMEM and barriers count as much (two
// loads in flight, by 32 columns or by 16, were slower: 340 and 332 us).  32
// decode tokens over 130673 slots of 8 heads: 57 us, 4.7 TB/s of K.
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
namespace fx = kyro::fx2;

constexpr int kBS = 16;                // tokens per KV block
constexpr int kTM = 128;               // slots per tile
constexpr int kItemSlots = 2 * kTM;    // slots per item
constexpr int kTN = 128;               // rows per step
constexpr int kPages = kTM / kBS;      // 8
constexpr int kThreads = 640;
constexpr int kSumWarps = 16;
constexpr int kKWarp = 16, kMmaWarp = 17, kQWarp = 18, kKWarp2 = 19;
constexpr int kMaxCtas = kyro::chunk::kMaxCtas;
constexpr uint32_t kSlab = 128 * 128;  // 128 rows of 64 dims
constexpr uint32_t kTmemCols = 512;    // score buffer s of tile h at (2 * h + s) * 128
// no CTA is given fewer steps than this.  Few or short chunks (the first 16
// batches of scores of at most 512 rows that perf/operators.py's
// draw(random.Random(s)) gives for s = 0, 1, ..) take 12.2 us in the geometric
// mean, 12.3 with 1 and 13.4 with 4.
constexpr int kMinSteps = 2;

template <int D>
struct Geo {
  static constexpr int kSlabs = D / 64;
  static constexpr uint32_t kTile = kSlabs * kSlab;  // 128 rows x D
  static constexpr int kKSlots = D == 128 ? 4 : 8;   // tiles of K (128 KB)
  static constexpr int kQSlots = D == 128 ? 3 : 4;   // tiles of Q
  static constexpr uint32_t kOffQ = kKSlots * kTile;
  static constexpr uint32_t kOffLse = kOffQ + kQSlots * kTile;
  static constexpr uint32_t kOffBar = kOffLse + kQSlots * kTN * 4;
  // barriers (two per slot, 13 and the ring of pieces'), then the TMEM
  // address, the error flag, k_last and the pieces
  static constexpr uint32_t kBars =
      16 * (kKSlots + kQSlots) + 8 * 13 + 16 * kyro::chunk::kPieceSlots;
  static constexpr uint32_t kOffMisc = kOffBar + (kBars + 15) / 16 * 16;
  static constexpr uint32_t kOffPieces = kOffMisc + 16 + 32;
  static constexpr uint32_t kSmem =
      kOffPieces + sizeof(kyro::chunk::Piece) * kyro::chunk::kPieceSlots + 1024;  // + alignment
  static_assert(kKSlots * 4 <= 32 && kSmem <= 232448, "shared memory");
};

struct ScoreArgs {
  Shape sh;
  int hq, num_blocks;
  float scale_log2;
  int64_t slots;
};

// Items of a KV head (256 slots each), and the steps of sh.tokens tokens
// that see one.  An item's cost is the tokens that see it (a step's at
// least): a step costs sh.tokens.
struct ScorePolicy {
  static __device__ __forceinline__ int prepare(const Seq& s, const Shape& sh) {
    return (s.n + sh.tokens - 1) / sh.tokens;  // steps of the chunk
  }
  static __device__ __forceinline__ int count(const Seq& s, const Shape& sh) {
    return (s.ctx + s.n + kItemSlots - 1) / kItemSlots;
  }
  // the first step: tokens before the one at the item's first slot see none of it
  static __device__ __forceinline__ int step0(const Seq& s, const Shape& sh, int t) {
    return t * kItemSlots <= s.ctx ? 0 : (t * kItemSlots - s.ctx) / sh.tokens;
  }
  static __device__ __forceinline__ int tiles(const Seq& s, const Shape& sh, int t) {
    return s.aux - step0(s, sh, t);
  }
  static __device__ __forceinline__ int kUnit(const Shape& sh) { return sh.tokens; }
  static __device__ __forceinline__ int unit(const Seq&, const Shape& sh, int) { return sh.tokens; }
  static __device__ __forceinline__ int over(const Seq&, const Shape& sh, int) { return sh.tokens; }
  static __device__ __forceinline__ int cost(const Seq& s, const Shape& sh, int t) {
    return max(s.n, sh.tokens) + sh.tokens -
           max(0, t * kItemSlots - s.ctx);
  }
  static __device__ __forceinline__ long long before(const Seq& s, const Shape& sh, int t) {
    // items up to slot ctx are seen by all n tokens, later ones by 256 fewer each
    const int n = max(s.n, sh.tokens), t0 = s.ctx / kItemSlots + 1, late = max(0, t - t0);
    const long long skip = (long long)late * (t0 * kItemSlots - s.ctx) +
                           (long long)kItemSlots * ((long long)late * (late - 1) / 2);
    return (long long)t * (n + sh.tokens) - skip;
  }
};
using Walker = kyro::chunk::Walker<ScorePolicy>;

// workspace: descs [G][2], then the sums [G][2][256]
constexpr size_t kDescBytes = (size_t)kMaxCtas * 2 * sizeof(PartDesc);
constexpr size_t kPartBytes = (size_t)kMaxCtas * 2 * kItemSlots * 4;

// acc += exp2(x * scale + nl) over kCols columns; nl: minus the rows' lse
template <int kCols>
__device__ __forceinline__ void sum_cols(const uint32_t (&x)[kCols], const float4* nl, fx::f2 sl,
                                         fx::f2 (&acc)[2]) {
#pragma unroll
  for (int i = 0; i < kCols / 4; ++i) {
    const float4 e = nl[i];
    fx::f2 y[2] = {fx::fma(fx::pack(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1])), sl,
                           fx::pack(e.x, e.y)),
                   fx::fma(fx::pack(__uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3])),
                           sl, fx::pack(e.z, e.w))};
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float lo, hi;
      fx::unpack(y[v], lo, hi);
      acc[v] = fx::add(acc[v], fx::pack(kyro::ptx::fast_exp2(lo), kyro::ptx::fast_exp2(hi)));
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
kv_scores_kernel(const __grid_constant__ CUtensorMap tmQ,
                 const __grid_constant__ CUtensorMap tmK, const ScoreArgs a,
                 const float* __restrict__ lse,
                 const int32_t* __restrict__ starts, const int64_t* __restrict__ block_table,
                 const int64_t* __restrict__ context_lens, const float* scores, float* out,
                 PartDesc* __restrict__ descs, float* __restrict__ parts, uint32_t* status) {
  using G = Geo<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = kyro::ptx::smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + G::kOffBar;
  auto k_full = [&](int s) { return bar0 + 8u * s; };
  auto k_empty = [&](int s) { return bar0 + 8u * (G::kKSlots + s); };
  const uint32_t bar1 = bar0 + 16u * G::kKSlots;
  auto q_full = [&](int s) { return bar1 + 8u * s; };
  auto q_empty = [&](int s) { return bar1 + 8u * (G::kQSlots + s); };
  const uint32_t bar2 = bar1 + 16u * G::kQSlots;
  auto s_full = [&](int h, int buf) { return bar2 + 8u * (2 * h + buf); };
  auto s_empty = [&](int h, int buf) { return bar2 + 8u * (4 + 2 * h + buf); };
  const uint32_t mma_done = bar2 + 8u * 8;
  // the second halves' sums of tile h, of every other join: a second half can
  // be a join ahead (two short pieces are two score buffers), but not two
  auto m_full = [&](int h, int k) { return bar2 + 8u * (9 + 2 * h + (k & 1)); };
  const uint32_t piece_bars = bar2 + 8u * 13;
  auto k_addr = [&](int n) { return base + (uint32_t)(n % G::kKSlots) * G::kTile; };
  auto k_parity = [](int n) { return (uint32_t)((n / G::kKSlots) & 1); };
  auto q_addr = [&](int n) { return base + G::kOffQ + (uint32_t)(n % G::kQSlots) * G::kTile; };
  auto q_parity = [](int n) { return (uint32_t)((n / G::kQSlots) & 1); };
  float* sh_lse = reinterpret_cast<float*>(gbase + G::kOffLse);  // [kQSlots][kTN]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + G::kOffMisc);
  int* err = reinterpret_cast<int*>(gbase + G::kOffMisc + 4);
  int* k_last = reinterpret_cast<int*>(gbase + G::kOffMisc + 16);  // the last copy into a slot
  Piece* piece_slots = reinterpret_cast<Piece*>(gbase + G::kOffPieces);
  // (before the first step, sh_lse is locate()'s)
  auto* scratch = reinterpret_cast<kyro::chunk::Scratch<kThreads>*>(sh_lse);
  static_assert(sizeof(*scratch) <= kTN * 4 * G::kQSlots, "scratch");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < G::kKSlots; ++i) {
      kyro::ptx::mbar_init(k_full(i), 1);
      kyro::ptx::mbar_init(k_empty(i), 1);
      k_last[i] = -1;
    }
    for (int i = 0; i < G::kQSlots; ++i) {
      kyro::ptx::mbar_init(q_full(i), 1);
      kyro::ptx::mbar_init(q_empty(i), 1 + kSumWarps);  // the products, and every sum warp (its lse)
    }
    for (int h = 0; h < 2; ++h)
      for (int i = 0; i < 2; ++i) {
        kyro::ptx::mbar_init(s_full(h, i), 1);
        kyro::ptx::mbar_init(s_empty(h, i), kSumWarps / 2);
      }
    kyro::ptx::mbar_init(mma_done, 1);
    for (int h = 0; h < 2; ++h)
      for (int i = 0; i < 2; ++i) kyro::ptx::mbar_init(m_full(h, i), 4);
    Pieces::init(piece_bars, kThreads / 32 - 1);
    *err = 0;
    kyro::ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc1(kyro::ptx::smem_addr(tmem_slot), kTmemCols);
    tmem_relinquish1();
  }
  // rows that no token of a step fills stay zeros
  if (a.sh.tokens * a.sh.group < kTN) {
    for (uint32_t i = threadIdx.x * 16; i < G::kQSlots * G::kTile; i += kThreads * 16)
      *reinterpret_cast<uint4*>(gbase + G::kOffQ + i) = make_uint4(0, 0, 0, 0);
    fence_async_shared();
  }
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  kyro::chunk::locate<ScorePolicy, kThreads>(a.sh, starts, context_lens, kMinSteps, status,
                                             scratch);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int group = a.sh.group, tokens = a.sh.tokens;
  Pieces pieces(piece_bars, piece_slots, err, status);
  Piece p;
  // rows of a step, in whole 32s: the N of its matrix products
  auto cols_of = [&](const Piece& pc, int step) {
    return (min(tokens, pc.s.n - step * tokens) * group + 31) & ~31;
  };

  if (warp == kKWarp || warp == kKWarp2) {
    // ------------------------------------------------ tiles of K, tile h of each item
    const int h = warp == kKWarp2;
    if (lane == 0) kyro::ptx::prefetch_tensormap(&tmK);
    const int pg = lane / G::kSlabs, slab = lane % G::kSlabs;  // this lane's part of a tile
    // pages of the tile, and this lane's block
    auto look = [&](const Piece& pc, int64_t& blk) {
      const int L = pc.s.ctx + pc.s.n, i = (pc.t * 2 + h) * kPages;
      const int np = min(kPages, (L + kBS - 1) / kBS - i);
      blk = pg < np ? __ldg(&block_table[(int64_t)pc.b * a.sh.max_blocks + i + pg]) : 0;
      return np;
    };
    auto tiles_of = [&](const Piece& pc) {
      return pc.s.ctx + pc.s.n - pc.t * kItemSlots > kTM ? 2 : 1;
    };
    int n = 0;            // tiles of K so far, of both warps
    bool ok = true;
    int64_t blk;
    // the first of them walks, for all
    Walker walk(a.sh, starts, context_lens, scratch->start);
    auto next = [&](Piece& pc) {
      if (h) return pieces.get(pc);
      const bool any = walk.next(pc);
      return pieces.put(pc) && any;
    };
    bool have = next(p);
    int np = have ? look(p, blk) : 0;
    while (have) {
      // the next item's blocks are looked up while this one's copies wait
      Piece pn;
      int64_t blk_n = 0;
      const bool more = next(pn);
      const int np_n = more ? look(pn, blk_n) : 0;
      const int ntk = tiles_of(p);
      if (h < ntk) {
        if (blk < 0 || blk >= a.num_blocks) {
          kyro::dev::flag(status, KYRO_DEV_BAD_BLOCK);
          blk = 0;
        }
        const int i = n + h, s = i % G::kKSlots;
        if (i >= G::kKSlots) ok = wait_bar_warp(k_empty(s), k_parity(i - G::kKSlots), err, status);
        ok = __all_sync(0xffffffffu, ok && !*(volatile int*)err);
        if (!ok) break;
        if (lane == 0) kyro::ptx::mbar_arrive_expect_tx(k_full(s), (uint32_t)np * kBS * D * 2);
        __syncwarp();
        if (pg < np)
          kyro::ptx::tma_load_3d(k_addr(i) + slab * kSlab + (uint32_t)pg * kBS * 128, &tmK,
                                 slab * 64, 0, (int32_t)(blk * a.sh.hkv + p.kvh), k_full(s));
        if (lane == 0) k_last[s] = i;
      }
      n += ntk;
      p = pn;
      blk = blk_n;
      np = np_n;
      have = more;
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------ matrix instructions (one thread)
    if (lane == 0) {
      int nk = 0, nq = 0, steps[2] = {0, 0};
      bool ok = true;
      while (ok && pieces.get_alone(p)) {
        const int ntk = p.s.ctx + p.s.n - p.t * kItemSlots > kTM ? 2 : 1;
        const int st0 = ScorePolicy::step0(p.s, a.sh, p.t);
        for (int j = p.tile0; ok && j < p.tile1; ++j, ++nq) {
          ok = wait_bar(q_full(nq % G::kQSlots), q_parity(nq), err, status);
          const uint32_t id = idesc_f16(kTM, cols_of(p, st0 + j), false);
          for (int h = 0; ok && h < ntk; ++h) {
            if (j == p.tile0)
              ok = wait_bar(k_full((nk + h) % G::kKSlots), k_parity(nk + h), err, status);
            const int buf = steps[h] & 1;
            if (steps[h] >= 2)
              ok = ok && wait_bar(s_empty(h, buf), ((steps[h] >> 1) - 1) & 1, err, status);
            if (!ok) break;
            tc_fence_after();
            const uint32_t kd = desc_lo(k_addr(nk + h), 16), qd = desc_lo(q_addr(nq), 16);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t off = ((uint32_t)(k >> 2) * kSlab + (uint32_t)(k & 3) * 32) >> 4;
              umma1_ss(tmem + (uint32_t)(2 * h + buf) * 128, kd + off, qd + off, id,
                       k > 0 ? 1u : 0u);
            }
            umma1_commit(s_full(h, buf));
            if (j + 1 == p.tile1) umma1_commit(k_empty((nk + h) % G::kKSlots));
            ++steps[h];
          }
          if (ok) umma1_commit(q_empty(nq % G::kQSlots));
        }
        nk += ntk;
      }
      umma1_commit(mma_done);
      wait_bar(mma_done, 0, err, status);
    }
    __syncwarp();
  } else if (warp == kQWarp) {
    // ------------------------------------------------ tiles of Q and their lse
    if (lane == 0) kyro::ptx::prefetch_tensormap(&tmQ);
    const uint32_t bytes = (uint32_t)(tokens * group) * D * 2;
    int nq = 0;
    bool ok = true;
    // the four columns of a step that this lane has: their token and head
    int ctok[4], chead[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ctok[i] = (lane + 32 * i) / group;
      chead[i] = lane + 32 * i - ctok[i] * group;
    }
    while (ok && pieces.get(p)) {
      const int st0 = ScorePolicy::step0(p.s, a.sh, p.t);
      for (int j = p.tile0; j < p.tile1; ++j, ++nq) {
        const int tok0 = (st0 + j) * tokens;
        const int ntok = min(tokens, p.s.n - tok0);
        // in log2, negative; a column that is no row of the chunk weighs nothing
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = ctok[i] < ntok ? -1.4426950408889634f *
                                      lse[(int64_t)(p.s.start + tok0 + ctok[i]) * a.hq +
                                          p.kvh * group + chead[i]]
                                : -INFINITY;
        const int s = nq % G::kQSlots;
        if (nq >= G::kQSlots) ok = wait_bar_warp(q_empty(s), q_parity(nq - G::kQSlots), err, status);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) sh_lse[s * kTN + lane + 32 * i] = x[i];
        __syncwarp();
        if (lane == 0) {
          kyro::ptx::mbar_arrive_expect_tx(q_full(s), bytes);
          for (int sl = 0; sl < G::kSlabs; ++sl)
            kyro::ptx::tma_load_3d(q_addr(nq) + sl * kSlab, &tmQ, sl * 64, p.kvh * group,
                                   p.s.start + tok0, q_full(s));
        }
      }
    }
    __syncwarp();
    if (*(volatile int*)err && lane == 0) {
      for (int i = nq > G::kQSlots ? nq - G::kQSlots : 0; i < nq; ++i)
        kyro::ptx::mbar_wait_bounded(q_full(i % G::kQSlots), q_parity(i), kWaitBudget);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ sums of tile h, two threads per slot
    const int h = warp / 8;
    const int quarter = warp & 3;
    const int c0 = (warp & 4) ? kTN / 2 : 0;  // this thread's columns of a step: c0 .. c0 + 63
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const fx::f2 sl = fx::pack(a.scale_log2, a.scale_log2);
    PartDesc* my_desc = descs + (size_t)blockIdx.x * 2;
    if (threadIdx.x == 0) my_desc[0].valid = my_desc[1].valid = 0;
    int nq = 0, steps = 0, joins = 0;
    bool ok = true;
    // this thread's slot in an item, and its old score: loaded one item ahead
    auto slot_of = [&](const Piece& pc) { return pc.t * kItemSlots + h * kTM + row; };
    auto at_of = [&](const Piece& pc) {
      return ((int64_t)pc.b * a.sh.hkv + pc.kvh) * a.slots + slot_of(pc);
    };
    auto old_of = [&](const Piece& pc) {
      return c0 == 0 && pc.first() && pc.last() && slot_of(pc) < pc.s.ctx ? scores[at_of(pc)]
                                                                          : 0.0f;
    };
    Piece pn;
    bool have_piece = pieces.get(p);
    float old = have_piece ? old_of(p) : 0.0f;
    for (; have_piece; p = pn) {
      have_piece = pieces.get(pn);
      const float old_n = have_piece ? old_of(pn) : 0.0f;
      if (threadIdx.x == 0 && !(p.first() && p.last())) kyro::chunk::describe(my_desc, p);
      const int L = p.s.ctx + p.s.n;
      const int tile_slot = p.t * kItemSlots + h * kTM;
      const int t = slot_of(p);
      const bool have = tile_slot < L;
      const int st0 = ScorePolicy::step0(p.s, a.sh, p.t);
      // tokens before this one do not see the slot
      const int tok_min = t - p.s.ctx;
      const int warp_tok_min = tile_slot + quarter * 32 + 31 - p.s.ctx;
      // whether a step has rows in its second half at all
      const bool join = have && min(tokens, p.s.n) * group > kTN / 2;
      fx::f2 acc[2] = {0, 0};
      float m = 0.0f;
      for (int j = p.tile0; j < p.tile1; ++j, ++nq) {
        const int s = nq % G::kQSlots;
        if (!wait_bar_warp(q_full(s), q_parity(nq), err, status)) {
          ok = false;
          break;
        }
        if (have) {
          const int buf = steps & 1;
          if (!wait_bar_warp(s_full(h, buf), (steps >> 1) & 1, err, status)) {
            ok = false;
            break;
          }
          ++steps;
          tc_fence_after();
          const int tok0 = (st0 + j) * tokens;
          const int valid = min(tokens, p.s.n - tok0) * group;  // columns that are rows
          const uint32_t sc = tmem + lane_base + (uint32_t)(2 * h + buf) * 128 + c0;
          const float4* ls = reinterpret_cast<const float4*>(sh_lse + s * kTN + c0);
          if (tok0 + tokens <= p.s.n && warp_tok_min <= tok0) {
            // a whole step that every slot is seen by: no mask (the padding
            // rows are zeros and weigh nothing)
#pragma unroll 1
            for (int c = 0; c < kTN / 2 && c0 + c < valid; c += 32) {
              uint32_t x[32];
              tmem_ld32(sc + c, x);
              tmem_ld_wait();
              sum_cols<32>(x, ls + c / 4, sl, acc);
            }
          } else {
            const int cmin = kyro::chunk::hidden_cols(tok_min, tok0, group);
#pragma unroll 1
            for (int c = 0; c < kTN / 2 && c0 + c < valid; c += 8) {
              uint32_t x[8];
              tmem_ld8(sc + c, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (c0 + c + i < cmin || c0 + c + i >= valid) x[i] = 0xff800000u;  // weighs nothing
              sum_cols<8>(x, ls + c / 4, sl, acc);
            }
          }
          if (j + 1 == p.tile1) {
            float m0, m1;
            fx::unpack(fx::add(acc[0], acc[1]), m0, m1);
            m = m0 + m1;
            if (join) {
              // the second half's sum goes over a score that it has read; the
              // buffer is the first half's until it has taken it
              if (c0) {
                tmem_st1(sc, __float_as_uint(m));
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) kyro::ptx::mbar_arrive(m_full(h, joins));
              } else {
                if (!wait_bar_warp(m_full(h, joins), (joins >> 1) & 1, err, status)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                m += __uint_as_float(tmem_ld1(sc + kTN / 2));
              }
              ++joins;
            }
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          if (have) kyro::ptx::mbar_arrive(s_empty(h, (steps - 1) & 1));
          kyro::ptx::mbar_arrive(q_empty(s));
        }
      }
      if (!ok) break;
      if (c0 == 0) {
        if (p.first() && p.last()) {
          if (t < L) out[at_of(p)] = old + m;
        } else if (have) {
          parts[((size_t)blockIdx.x * 2 + (p.first() ? 1 : 0)) * kItemSlots + h * kTM + row] = m;
        }
      }
      old = old_n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // no CTA leaves while a copy may still write its shared memory: after a
  // timeout the tiles of K in flight are waited for here
  if (*(volatile int*)err && threadIdx.x == 0)
    for (int s = 0; s < G::kKSlots; ++s)
      if (k_last[s] >= 0)
        kyro::ptx::mbar_wait_bounded(k_full(s), k_parity(k_last[s]), kWaitBudget);
  if (warp == kMmaWarp) tmem_dealloc1(tmem, kTmemCols);
}

// Adds the pieces of the item that CTA blockIdx.x began and did not end, in
// the order of their rows.
__global__ void __launch_bounds__(kItemSlots)
kv_scores_join_kernel(const ScoreArgs a, int ctas, const int32_t* __restrict__ starts,
                      const int64_t* __restrict__ context_lens, const float* scores, float* out,
                      const PartDesc* __restrict__ descs, const float* __restrict__ parts) {
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  const int c0 = blockIdx.x;
  const PartDesc d = descs[c0 * 2 + 1];
  if (!d.valid) return;
  const Seq s = kyro::chunk::seq_of(d.b, starts, context_lens, a.sh.T, a.sh.max_slots);
  const int t = d.t * kItemSlots + threadIdx.x;
  if (t >= s.ctx + s.n) return;
  float m = 0.0f;
  for (int c = c0; c < ctas; ++c) {
    const size_t slot = (size_t)c * 2 + (c == c0);
    if (!descs[slot].valid) continue;
    m += parts[slot * kItemSlots + threadIdx.x];
    if (descs[slot].last) break;
  }
  const int64_t at = ((int64_t)d.b * a.sh.hkv + d.kvh) * a.slots + t;
  out[at] = (t < s.ctx ? scores[at] : 0.0f) + m;
}

int check(const kyro_chunk_params* p) {
  const char* fn = "kyro_kv_scores_add";
  KY_TRY(kyro::chunk::check_params(p, fn));
  KY_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "%s: head_dim = %d (64 or 128 supported)",
             fn, p->head_dim);
  KY_REQUIRE(p->block_size == kBS, "%s: block_size = %d (only %d supported)", fn, p->block_size,
             kBS);
  KY_REQUIRE((int64_t)p->num_blocks * p->num_kv_heads < (1ll << 31),
             "%s: num_blocks * num_kv_heads must fit in 31 bits", fn);
  KY_REQUIRE(p->num_heads / p->num_kv_heads <= kTN,
             "%s: %d query heads per KV head (at most %d)", fn, p->num_heads / p->num_kv_heads,
             kTN);
  KY_REQUIRE(p->scale >= 0.0f && std::isfinite(p->scale), "%s: scale = %g", fn, (double)p->scale);
  KY_REQUIRE(kyro::chunk::stride_ok(p->q_stride, (int64_t)p->num_heads * p->head_dim),
             "%s: a row stride is shorter than its row or not a multiple of 8", fn);
  return KYRO_OK;
}

template <int D>
int launch(kyro_ctx* ctx, const kyro_chunk_params* p, const ScoreArgs& a, const void* q,
           const void* k_cache, const float* lse, const int32_t* starts,
           const int64_t* block_table, const int64_t* context_lens, const float* scores,
           float* out, void* workspace) {
  // Q [T][Hq][D]: box (64 dims, a group's heads, a step's tokens);
  // K [blocks * Hkv][16 tokens][D]: box (64 dims, 16 tokens, 1)
  CUtensorMap mq, mk;
  const int64_t qs = kyro::chunk::stride_or(p->q_stride, (int64_t)p->num_heads * D);
  KY_TRY(make_map3(&mq, q, D, (uint64_t)p->num_heads, (uint64_t)p->num_tokens, (uint64_t)D * 2,
                   (uint64_t)qs * 2, (uint32_t)a.sh.group, (uint32_t)a.sh.tokens));
  const uint64_t rows = (uint64_t)p->num_blocks * p->num_kv_heads;
  KY_TRY(make_map3(&mk, k_cache, D, kBS, rows, (uint64_t)D * 2, (uint64_t)kBS * D * 2, kBS, 1));
  PartDesc* descs = (PartDesc*)workspace;
  float* parts = (float*)((char*)workspace + kDescBytes);
  const int ctas = std::min(ctx->num_sms, kMaxCtas);
  KY_TRY(kyro::chunk::set_smem<kv_scores_kernel<D>>(Geo<D>::kSmem, ctx->device));
  KY_TRY(kyro::launch_pdl(kv_scores_kernel<D>, dim3((unsigned)ctas), dim3(kThreads), Geo<D>::kSmem,
                          ctx->stream, "kv_scores_kernel", mq, mk, a, lse, starts,
                          block_table, context_lens, scores, out, descs, parts, ctx->d_status));
  return kyro::launch_pdl(kv_scores_join_kernel, dim3((unsigned)ctas), dim3(kItemSlots), 0,
                          ctx->stream, "kv_scores_join_kernel", a, ctas, starts, context_lens,
                          scores, out, (const PartDesc*)descs, (const float*)parts);
}

}  // namespace

extern "C" {

size_t kyro_kv_scores_add_workspace_size(const kyro_chunk_params* p) {
  if (check(p) != KYRO_OK) return 0;
  return kDescBytes + kPartBytes;
}

int kyro_kv_scores_add(kyro_ctx* ctx, const kyro_chunk_params* p, const void* q,
                       const void* k_cache, const float* lse, const int32_t* chunk_starts,
                       const int64_t* block_table, const int64_t* context_lens,
                       int64_t score_slots, const float* scores, float* scores_out,
                       void* workspace, size_t workspace_bytes) {
  const char* fn = "kyro_kv_scores_add";
  KY_NVTX("kyro_kv_scores_add");
  KY_TRY(kyro::enter(ctx));
  KY_TRY(check(p));
  KY_REQUIRE(score_slots >= 1, "%s: score_slots = %lld", fn, (long long)score_slots);
  if (p->batch == 0 || p->num_tokens == 0) return KYRO_OK;
  KY_REQUIRE(q && k_cache && lse && chunk_starts && block_table && context_lens && scores &&
                 scores_out,
             "%s: a required pointer is NULL", fn);
  KY_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k_cache % 16 == 0,
             "%s: q and the cache must be 16-byte aligned", fn);
  const size_t need = kyro_kv_scores_add_workspace_size(p);
  if (!workspace || workspace_bytes < need)
    return kyro::set_error(KYRO_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn,
                           workspace_bytes, need);
  KY_REQUIRE((uintptr_t)workspace % 256 == 0, "%s: workspace must be 256-byte aligned", fn);
  ScoreArgs a;
  a.sh.B = p->batch;
  a.sh.T = p->num_tokens;
  a.sh.hkv = p->num_kv_heads;
  a.sh.group = p->num_heads / p->num_kv_heads;
  a.sh.tokens = kTN / a.sh.group;
  a.sh.max_blocks = p->max_blocks_per_seq;
  a.sh.max_slots = (int)std::min<int64_t>(score_slots, (int64_t)p->max_blocks_per_seq * kBS);
  a.hq = p->num_heads;
  a.num_blocks = p->num_blocks;
  const float scale = p->scale > 0.0f ? p->scale : 1.0f / sqrtf((float)p->head_dim);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.slots = score_slots;
  if (p->head_dim == 128)
    return launch<128>(ctx, p, a, q, k_cache, lse, chunk_starts, block_table, context_lens, scores,
                       scores_out, workspace);
  return launch<64>(ctx, p, a, q, k_cache, lse, chunk_starts, block_table, context_lens, scores,
                    scores_out, workspace);
}

}  // extern "C"
