// chunk.cuh -- what the operators on packed prompt chunks share: the checks
// of kyro_chunk_params and the device-side view of one sequence's chunk.
#pragma once

#include <stdint.h>

#include <atomic>

#include "chunk_index.h"
#include "kyro_internal.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace kyro {
namespace chunk {

// Sequence b's new tokens: rows start .. start + n - 1, slots ctx .. ctx + n
// - 1.  n is 0 for an empty chunk and for one that cannot be taken (bad:
// its rows leave the packed tensors, or its slots the max_slots that the
// block table, and what else is kept per slot, has room for).
struct Seq {
  int start, n;
  int ctx;
  int aux;  // its Policy's
  int bad;
};

__device__ __forceinline__ Seq seq_from(int s0, int s1, int64_t ctx, int T, int max_slots) {
  Seq s;
  const int n = chunk_rows(s0, s1, ctx, T, max_slots);
  s.start = s0;
  s.bad = n < 0;
  s.n = n < 0 ? 0 : n;
  s.ctx = (int)ctx;
  return s;
}

__device__ __forceinline__ Seq seq_of(int b, const int32_t* __restrict__ starts,
                                      const int64_t* __restrict__ context_lens, int T,
                                      int max_slots) {
  return seq_from(__ldg(&starts[b]), __ldg(&starts[b + 1]), __ldg(&context_lens[b]), T,
                  max_slots);
}

// ---------------------------------------------------------------- the walk
// A persistent kernel's share of the work.  The batch is a line of items:
// sequence by sequence, KV head by KV head, `count` items of one head one
// after the other, each with a cost.  CTA c of G walks the stretch W c / G ..
// W (c + 1) / G of the line, whatever items it holds, so that every CTA has
// the same work for any mix of lengths; an item that crosses such a border
// is done in pieces.  Which items a CTA walks follows from the lengths alone.
//
// A Policy gives (Shape sh, Seq s):
//   prepare(s, sh)    what it keeps in s.aux
//   count(s, sh)      items of a head
//   tiles(s, sh, t)   tiles of slots or of rows that item t goes through
//   cost(s, sh, t)    of item t
//   before(s, sh, t)  the cost of the head's items before item t, in closed
//                     form (a sum over a long prompt's items would take the
//                     first microseconds of every call)
//   kUnit(sh)         the cost of a tile; unit(s, sh, t) that of item t's
//   over(s, sh, t)    what item t costs beside its tiles (its stationary
//                     operand, its epilogue); part of cost and before
struct Shape {
  int B, T, hkv, group, tokens, max_blocks, max_slots;  // tokens: of a tile of rows
};
struct WalkStart {
  long long rem;  // cost to walk
  int b, kvh, t, u;
  Seq s;
};
// A piece of an item: its tiles tile0 .. tile1 - 1 of `tiles`.
struct alignas(16) Piece {
  Seq s;
  int b, kvh, t, tile0, tile1, tiles;
  int end;  // no piece: the walk is over
  __device__ __forceinline__ bool first() const { return tile0 == 0; }
  __device__ __forceinline__ bool last() const { return tile1 == tiles; }
};

constexpr int kMaxCtas = 148;  // of a persistent kernel: one per SM

// The unfinished items of a CTA, in its workspace: slot 0 the piece that
// continues an item of an earlier CTA, slot 1 the piece that begins an item
// and does not end it.  A CTA has at most one of each.
struct PartDesc {
  int valid, last, b, kvh, t, pad[3];
};
__device__ __forceinline__ void describe(PartDesc* descs, const Piece& p) {
  PartDesc* d = descs + (p.first() ? 1 : 0);
  d->last = p.last();
  d->b = p.b;
  d->kvh = p.kvh;
  d->t = p.t;
  d->valid = 1;
}

template <class Policy>
__device__ __forceinline__ Seq load_seq(int b, const Shape& sh, const int32_t* __restrict__ starts,
                                        const int64_t* __restrict__ context_lens) {
  Seq s = seq_of(b, starts, context_lens, sh.T, sh.max_slots);
  s.aux = Policy::prepare(s, sh);
  return s;
}

// Shared memory of locate(); free again once the walker has its start.
template <int kThreads>
struct alignas(16) Scratch {
  WalkStart start;
  long long wsum[kThreads / 32];
};

// Where this CTA starts (all threads call it; kThreads a multiple of 32).  A
// sequence that cannot be taken is flagged, by CTA 0.  No more CTAs take
// part than leave min_tiles tiles for each.
template <class Policy, int kThreads>
__device__ void locate(const Shape& sh, const int32_t* __restrict__ starts,
                       const int64_t* __restrict__ context_lens, int min_tiles, uint32_t* status,
                       Scratch<kThreads>* scratch) {
  constexpr int kWarps = kThreads / 32;
  long long* wsum = scratch->wsum;
  WalkStart* out = &scratch->start;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto cost_of = [&](const Seq& s) -> long long {
    return s.n > 0 ? Policy::before(s, sh, Policy::count(s, sh)) * sh.hkv : 0;
  };
  long long mine = 0, kept = 0;  // kept: this thread's first sequence
  Seq first{};
  for (int b = tid; b < sh.B; b += kThreads) {
    const Seq s = load_seq<Policy>(b, sh, starts, context_lens);
    if (s.bad && blockIdx.x == 0) kyro::dev::flag(status, KYRO_DEV_BAD_LENGTH);
    const long long c = cost_of(s);
    if (b == tid) {
      kept = c;
      first = s;
    }
    mine += c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) wsum[warp] = mine;
  if (tid == 0) out->rem = 0;
  __syncthreads();
  long long W = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) W += wsum[i];
  // stretch c is W c / G .. W (c + 1) / G, in 32-bit divisions where W fits
  const long long parts = W / ((long long)min_tiles * Policy::kUnit(sh));
  const uint32_t G = parts < 1 ? 1u : parts < gridDim.x ? (uint32_t)parts : gridDim.x;
  const uint32_t c = blockIdx.x;
  if (c >= G || W == 0) return;
  const long long each = (W >> 32) ? W / G : (long long)((uint32_t)W / G);
  const uint32_t over = (uint32_t)(W - each * G);
  const long long lo = each * c + over * c / G;
  const long long hi = each * (c + 1) + over * (c + 1) / G;
  if (lo >= hi) return;
  long long base = 0;
  for (int b0 = 0; b0 < sh.B; b0 += kThreads) {
    const int b = b0 + tid;
    long long cost = kept;
    Seq s = first;
    if (b0 > 0) {
      cost = 0;
      if (b < sh.B) {
        s = load_seq<Policy>(b, sh, starts, context_lens);
        cost = cost_of(s);
      }
    }
    long long inc = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    long long before = base + inc - cost, sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += wsum[w];
      sum += wsum[w];
    }
    if (cost > 0 && lo >= before && lo < before + cost) {
      const long long head = cost / sh.hkv;
      long long r = lo - before;
      int kvh = 0;
      while (r >= head) {
        r -= head;
        ++kvh;
      }
      int l = 0, h = Policy::count(s, sh);  // before(l) <= r < before(h)
      while (h - l > 1) {
        const int m = (l + h) / 2;
        if (Policy::before(s, sh, m) <= r) l = m;
        else h = m;
      }
      out->b = b;
      out->s = s;
      out->kvh = kvh;
      out->t = l;
      out->u = (int)(r - Policy::before(s, sh, l));
      out->rem = hi - lo;
    }
    base += sum;
    if (base > lo) break;
  }
}

// The pieces of a stretch.  One warp of a CTA walks, and hands the pieces to
// the others through a ring in shared memory (Pieces): at short items the
// walk, done by every warp for itself, was half of all instructions.
template <class Policy>
struct Walker {
  Shape sh;
  const int32_t* starts;
  const int64_t* lens;
  long long rem;
  int b, kvh, t, u;
  bool loaded;
  Seq s;
  int count;

  __device__ __forceinline__ Walker(const Shape& shape, const int32_t* st, const int64_t* cl,
                                    const WalkStart& w)
      : sh(shape), starts(st), lens(cl), rem(w.rem), b(w.b), kvh(w.kvh), t(w.t), u(w.u),
        loaded(true), s(w.s) {
    count = rem > 0 ? Policy::count(s, sh) : 0;
  }

  __device__ __forceinline__ bool next(Piece& p) {
    while (rem > 0 && b < sh.B) {
      if (!loaded) {
        s = load_seq<Policy>(b, sh, starts, lens);
        count = s.n > 0 ? Policy::count(s, sh) : 0;
        loaded = true;
      }
      if (count == 0) {
        ++b;
        loaded = false;
        continue;
      }
      p.s = s;
      p.b = b;
      p.kvh = kvh;
      p.t = t;
      p.tiles = Policy::tiles(s, sh, t);
      const int cost = Policy::cost(s, sh, t);
      const int end = (long long)(cost - u) <= rem ? cost : u + (int)rem;
      const int unit = Policy::unit(s, sh, t);
      const int over = Policy::over(s, sh, t);
      p.tile0 = tile_at(u - over, cost - over, p.tiles, unit);
      p.tile1 = tile_at(end - over, cost - over, p.tiles, unit);
      rem -= end - u;
      u = end;
      if (u == cost) {
        u = 0;
        if (++t == count) {
          t = 0;
          if (++kvh == sh.hkv) {
            kvh = 0;
            ++b;
            loaded = false;
          }
        }
      }
      p.end = 0;
      if (p.tile1 > p.tile0) return true;
    }
    p.end = 1;
    return false;
  }

  // the tiles that the first `paid` of what an item's tiles cost pay for
  static __device__ __forceinline__ int tile_at(int paid, int all, int tiles, int unit) {
    return paid >= all ? tiles : paid <= 0 ? 0 : min(tiles, paid / unit);
  }
};

// The ring of pieces: barriers full(i) (one arrival: the walker's) and
// empty(i) (one of each reading warp).
constexpr int kPieceSlots = 3;
struct Pieces {
  uint32_t bars;  // 2 * kPieceSlots barriers
  Piece* slots;
  int* err;
  uint32_t* status;
  int n = 0;

  __device__ __forceinline__ Pieces(uint32_t b, Piece* s, int* e, uint32_t* st)
      : bars(b), slots(s), err(e), status(st) {}
  static __device__ __forceinline__ void init(uint32_t bars, int readers) {
    for (int i = 0; i < kPieceSlots; ++i) {
      kyro::ptx::mbar_init(bars + 16u * i, 1);
      kyro::ptx::mbar_init(bars + 16u * i + 8u, readers);
    }
  }
  __device__ __forceinline__ uint32_t full() const { return bars + 16u * (n % kPieceSlots); }
  __device__ __forceinline__ uint32_t phase() const { return (n / kPieceSlots) & 1; }

  // by the walking warp
  __device__ __forceinline__ bool put(const Piece& p) {
    if (n >= kPieceSlots && !kyro::tc::wait_bar_warp(full() + 8u, phase() ^ 1u, err, status))
      return false;
    if ((threadIdx.x & 31) == 0) {
      slots[n % kPieceSlots] = p;
      kyro::ptx::mbar_arrive(full());
    }
    __syncwarp();
    ++n;
    return true;
  }
  // by a whole warp; false at the end of the walk and after a timeout
  __device__ __forceinline__ bool get(Piece& p) {
    if (!kyro::tc::wait_bar_warp(full(), phase(), err, status)) return false;
    p = slots[n % kPieceSlots];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) kyro::ptx::mbar_arrive(full() + 8u);
    ++n;
    return !p.end;
  }
  // by one thread of a warp that reads alone
  __device__ __forceinline__ bool get_alone(Piece& p) {
    if (!kyro::tc::wait_bar(full(), phase(), err, status)) return false;
    p = slots[n % kPieceSlots];
    kyro::ptx::mbar_arrive(full() + 8u);
    ++n;
    return !p.end;
  }
};

// The checks every chunk operator makes of its sizes.
inline int check_params(const kyro_chunk_params* p, const char* fn) {
  KY_REQUIRE(p, "%s: params is NULL", fn);
  KY_REQUIRE(p->batch >= 0, "%s: batch = %d", fn, p->batch);
  KY_REQUIRE(p->num_tokens >= 0, "%s: num_tokens = %d", fn, p->num_tokens);
  KY_REQUIRE(p->num_heads > 0 && p->num_kv_heads > 0 && p->num_heads % p->num_kv_heads == 0,
             "%s: num_heads %d not a multiple of num_kv_heads %d", fn, p->num_heads,
             p->num_kv_heads);
  KY_REQUIRE(p->block_size > 0, "%s: block_size = %d", fn, p->block_size);
  KY_REQUIRE(p->max_blocks_per_seq > 0, "%s: max_blocks_per_seq = %d", fn,
             p->max_blocks_per_seq);
  KY_REQUIRE((int64_t)p->max_blocks_per_seq * p->block_size < (1ll << 30),
             "%s: max_blocks_per_seq * block_size must be below 2^30", fn);
  KY_REQUIRE(p->num_blocks > 0, "%s: num_blocks = %d", fn, p->num_blocks);
  return KYRO_OK;
}

// A row stride: `dense` where none is given; a row must hold its `dense`
// elements and start on 16 bytes.
inline int64_t stride_or(int64_t stride, int64_t dense) { return stride ? stride : dense; }
inline bool stride_ok(int64_t stride, int64_t dense) {
  return stride == 0 || (stride >= dense && stride % 8 == 0);
}

// Allow a kernel `bytes` of dynamic shared memory, once per kernel and device.
template <auto Kernel>
int set_smem(size_t bytes, int device) {
  static std::atomic<uint64_t> done{0};  // a bit per device
  const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
  if (done.load() & bit) return KYRO_OK;
  const cudaError_t err =
      cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (err != cudaSuccess) return kyro::cuda_error(err, "cudaFuncSetAttribute");
  done.fetch_or(bit);
  return KYRO_OK;
}

}  // namespace chunk
}  // namespace kyro
