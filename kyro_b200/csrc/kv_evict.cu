// kv_evict.cu -- eviction from the paged cache by accumulated attention
// weight: every sequence over the budget keeps, in each layer and KV head,
// its first and last slots and the highest scores between them.  Bounded
// caches have no counterpart in the reference, whose BlockManager
// (src/scheduler/block_manager.rs:15-153) only grows a sequence; the free
// list, ref counts and block table keep its semantics.
//
// Three kernels, chained by programmatic launches:
//   kv_evict_select_kernel  one CTA per (layer, sequence, KV head): the
//       threshold score by a radix select over the scores' order-preserving
//       32-bit keys (8 + 12 + 12 bits), then the kept slots in ascending
//       order, and the scores closed up in place.  One more CTA per sequence
//       looks up the blocks.
//   kv_evict_move_kernel    the kept K/V rows into the fresh blocks: bound
//       by memory, each row read and written once, 16 bytes at a time.
//   kv_evict_commit_kernel  pops and pushes on the free list, the new table
//       rows and lengths.
// Rows go to fresh blocks and not to the front of the old ones, so that any
// row can move at any time (no order between reads and writes), and a block
// that other sequences hold keeps its rows.
//
// Which sequences are served depends only on their lengths and the free
// list's size: all take the same number of blocks, in batch order, until the
// list is empty.  So a sequence's blocks follow from how many before it are
// over the budget, and every CTA works that out for itself.
#include <algorithm>

#include "chunk.cuh"

namespace {

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 256 * 32;           // counts of the radix select: 32 KB
constexpr int kMoveThreads = 256;
constexpr int kCommitThreads = 1024;
constexpr int kMaxLayers = 32;            // layers per launch
constexpr int kRowCache = 48 * 1024;      // scores of a row held in shared memory

struct EvictArgs {
  int B, bs, max_blocks, num_blocks, hkv, d, budget, sink, recent, reserved, held;
  int64_t score_slots;
};
struct LayerPtrs {
  float* scores[kMaxLayers];
  uint8_t* k[kMaxLayers];
  uint8_t* v[kMaxLayers];
};

// whether a sequence is to be cut: over the budget, and its slots (the
// reserved ones too) fit the table and the scores
__device__ __forceinline__ bool over(const EvictArgs& a, int64_t len) { return len > a.budget; }
__device__ __forceinline__ bool fits(const EvictArgs& a, int64_t len) {
  return kyro::chunk::evict_fits(len, a.reserved, (int64_t)a.max_blocks * a.bs, a.score_slots);
}
__device__ __forceinline__ int clamp_top(int t, int num_blocks) {
  return t < 0 ? 0 : t > num_blocks ? num_blocks : t;
}

__device__ __forceinline__ int64_t blocks_for(int64_t tokens, int bs) {
  return (tokens + bs - 1) / bs;
}

// The workspace: what the selection leaves for the other kernels.
struct Scratch {
  int32_t* top;    // the free list's size before the call
  int32_t* odd;    // [B] a cut sequence holds a shared or invalid block
  int32_t* fresh;  // [B][held] the fresh blocks of a cut sequence
};

// The order of scores as unsigned integers: -0 equals +0, every NaN is the
// highest.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float float_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// How many sequences before b are cut (all threads of the CTA call it).
__device__ int cut_before(const EvictArgs& a, const int64_t* __restrict__ context_lens, int b) {
  int total = 0;
  for (int i0 = 0; i0 < b; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    const int64_t len = i < b ? context_lens[i] : 0;
    total += __syncthreads_count(i < b && over(a, len) && fits(a, len));
  }
  return total;
}

// The radix select's first digit is the sign and seven bits of the exponent:
// scores share a handful of its values, and shared-memory atomics to one
// address go one at a time.  So each lane has its own count of each value
// (conflict-free, 32 KB); the other two digits (12 bits, mostly mantissa)
// spread by themselves.  The selection from 192 rows of up to 16384 slots
// takes 28 us, from 384 of up to 4096 19 us, from 32 of 1000 8.5 us (40, 30
// and 10.5 us with digits of 11, 11 and 10 bits, one count per value, one
// score at a time and one CTA of 1024 threads per SM): instructions, where the
// scores' bytes alone would take 2 us.  Three CTAs per SM where the rows are
// short: evictions (the first 14 that perf/operators.py's draw(random.Random(s))
// gives for s = 0, 1, ..; with the copy that puts their state back) take 16.6
// us in the geometric mean, 16.8 with two and 17.2 with four.
__global__ void __launch_bounds__(kSelThreads, 3)
kv_evict_select_kernel(const __grid_constant__ EvictArgs a, const __grid_constant__ LayerPtrs lp,
                       int layer0, int cached, const int64_t* __restrict__ context_lens,
                       const int32_t* __restrict__ free_stack,
                       const int32_t* __restrict__ free_top, int32_t* __restrict__ out_evicted,
                       int32_t* __restrict__ out_kept, const int64_t* __restrict__ block_table,
                       const int32_t* __restrict__ ref_counts, Scratch ws, uint32_t* status) {
  extern __shared__ __align__(16) float row_cache[];
  __shared__ __align__(16) int hist[kBins];
  __shared__ int warp_a[kSelWarps], warp_b[kSelWarps];
  __shared__ int sh_digit, sh_need;
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t len64 = context_lens[b];
  const bool is_over = over(a, len64), can = is_over && fits(a, len64);
  if (h == a.hkv) {  // reports for the sequence
    if (layer != 0) return;
    bool cut = false;
    if (can) {
      const int rank = cut_before(a, context_lens, b);
      const int top = clamp_top(*free_top, a.num_blocks);
      cut = ((int64_t)rank + 1) * a.held <= top;
      if (cut) {
        for (int i = tid; i < a.held; i += kSelThreads) {
          int32_t blk = free_stack[top - 1 - rank * a.held - i];
          if (blk < 0 || blk >= a.num_blocks) {
            kyro::dev::flag(status, KYRO_DEV_BAD_BLOCK);
            blk = -1;
          }
          ws.fresh[(int64_t)b * a.held + i] = blk;
        }
        // whether its release takes more than a push of every block
        int odd = 0;
        const int n = (int)blocks_for(len64 + a.reserved, a.bs);
        for (int i = tid; i < n; i += kSelThreads) {
          const int64_t blk = block_table[(int64_t)b * a.max_blocks + i];
          odd |= blk < 0 || blk >= a.num_blocks || ref_counts[blk] != 1;
        }
        odd = __syncthreads_or(odd);
        if (tid == 0) ws.odd[b] = odd;
      }
    }
    if (tid == 0) {
      out_evicted[b] = cut ? (int32_t)(len64 - a.budget) : is_over ? -1 : 0;
      if (is_over && !can) kyro::dev::flag(status, KYRO_DEV_BAD_LENGTH);
      if (b == 0) {
        const int top = *free_top;
        ws.top[0] = clamp_top(top, a.num_blocks);
        if (ws.top[0] != top) kyro::dev::flag(status, KYRO_DEV_STACK_OVERFLOW);
      }
    }
    return;
  }
  int32_t* kept = out_kept + (((int64_t)(layer0 + layer) * a.B + b) * a.hkv + h) * a.budget;
  float* row = lp.scores[layer] + ((int64_t)b * a.hkv + h) * a.score_slots;
  const int len = can ? (int)len64 : 0;
  const bool on_chip = len <= cached;
  if (can && on_chip) {
    // on its way while the sequence's turn at the free list is found
    const uint32_t dst = kyro::ptx::smem_addr(row_cache);
    int done = 0;
    if ((uintptr_t)row % 16 == 0) {
      done = len & ~3;
      for (int i = tid * 4; i < done; i += kSelThreads * 4)
        kyro::ptx::cp_async_16(dst + i * 4, row + i);
    }
    for (int i = done + tid; i < len; i += kSelThreads)
      kyro::ptx::cp_async_4(dst + i * 4, row + i);
  }
  bool cut = false;
  if (can) {
    const int top = clamp_top(*free_top, a.num_blocks);
    cut = ((int64_t)cut_before(a, context_lens, b) + 1) * a.held <= top;
  }
  kyro::ptx::cp_async_commit();
  kyro::ptx::cp_async_wait<0>();
  if (!cut) {
    for (int i = tid; i < a.budget; i += kSelThreads) kept[i] = -1;
    return;
  }
  // four scores at a time (i a multiple of 4; what lies past the row is anything)
  auto load4 = [&](int i, float (&x)[4]) {
    if (on_chip) {
      const float4 v = *reinterpret_cast<const float4*>(row_cache + i);
      x[0] = v.x;
      x[1] = v.y;
      x[2] = v.z;
      x[3] = v.w;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = i + c < len ? row[i + c] : 0.0f;
    }
  };
  const int lo = a.sink, hi = len - a.recent;  // the slots that compete
  int need = a.budget - a.sink - a.recent;     // how many of them stay (fewer than there are)
  uint32_t prefix = 0;                         // the threshold's digits so far
  // thr is the need-th highest key; `need` of the keys equal to it stay
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 24 : pass == 1 ? 12 : 0;
      const int bits = pass == 0 ? 8 : 12;
      const int n4 = pass == 0 ? 256 * 32 / 4 : 4096 / 4;
      for (int i = tid; i < n4; i += kSelThreads)
        reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
      __syncthreads();
      // (a NaN passes the comparison with the floats that the digits so far
      // stand for, and is then told by its key)
      const float least = pass == 0 ? 0.0f : float_of(prefix << (shift + 12));
      const float most = pass == 0 ? 0.0f : float_of(~(~prefix << (shift + 12)));
      auto count = [&](float x) {
        if (pass == 0) {
          atomicAdd(&hist[(key_of(x) >> 24) * 32 + lane], 1);
        } else if (!(x < least) && !(x > most)) {
          const uint32_t k = key_of(x);
          if ((k >> (shift + 12)) == prefix) atomicAdd(&hist[(k >> shift) & 4095u], 1);
        }
      };
      for (int i = (lo & ~3) + tid * 4; i < hi; i += kSelThreads * 4) {
        float x[4];
        load4(i, x);
        if (i >= lo && i + 3 < hi) {
#pragma unroll
          for (int c = 0; c < 4; ++c) count(x[c]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (i + c >= lo && i + c < hi) count(x[c]);
        }
      }
      __syncthreads();
      // from the highest bin down: two threads sum the lanes of one bin (the
      // first of them has it), or thread t takes the 8 bins below 4096 - 8t
      int mine = 0, bin0;
      int c8[8];
      if (pass == 0) {
        bin0 = 255 - (tid >> 1);
        const int* bin = hist + bin0 * 32 + (tid & 1) * 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) mine += bin[(i + (lane >> 1)) & 15];
        mine += __shfl_xor_sync(0xffffffffu, mine, 1);
        if (tid & 1) mine = 0;
      } else {
        bin0 = 4095 - 8 * tid;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int4 x = reinterpret_cast<const int4*>(hist + bin0 - 7)[1 - i];
          c8[4 * i] = x.w;
          c8[4 * i + 1] = x.z;
          c8[4 * i + 2] = x.y;
          c8[4 * i + 3] = x.x;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += c8[i];
      }
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += t;
      }
      if (lane == 31) warp_a[warp] = before;
      __syncthreads();
      before += __reduce_add_sync(0xffffffffu, lane < warp ? warp_a[lane] : 0) - mine;
      if (before < need && before + mine >= need) {
        int bin = bin0, c = before;
        if (pass != 0) {
          bool found = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            found = found || c + c8[i] >= need;
            if (!found) {
              c += c8[i];
              --bin;
            }
          }
        }
        sh_digit = bin;
        sh_need = need - c;
      }
      __syncthreads();
      prefix = (prefix << bits) | (uint32_t)sh_digit;
      need = sh_need;
    }
  } else {
    prefix = 0xffffffffu;
    need = 0;
    __syncthreads();
  }
  // the kept slots in order: the first ones are where they belong, the last
  // ones follow all others, and between them a warp walks its own stretch of
  // the row twice, counting, then placing, four slots a lane.  A slot's place
  // is the number of slots above the threshold before it and of the ties
  // before it, as far as they stay.
  for (int i = tid; i < lo; i += kSelThreads) kept[i] = i;
  for (int i = tid; i < a.recent; i += kSelThreads) {
    const int at = a.budget - a.recent + i;
    kept[at] = hi + i;
    if (on_chip) row[at] = row_cache[hi + i];
  }
  const bool thr_nan = prefix == 0xffffffffu;
  const float thr = float_of(prefix);
  const int seg = (hi - (lo & ~3) + kSelWarps * 128 - 1) / (kSelWarps * 128) * 128;
  const int s0 = (lo & ~3) + warp * seg, s1 = min(hi, s0 + seg);
  // above the threshold, equal to it: bits of the 4 slots at i
  auto classify = [&](int i, const float (&x)[4], uint32_t& gt, uint32_t& eq) {
    gt = eq = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (!(x[c] <= thr) && !thr_nan) gt |= 1u << c;  // a NaN is above every number
      if (x[c] == thr || (thr_nan && x[c] != x[c])) eq |= 1u << c;
    }
    if (i < lo || i + 3 >= s1) {
      uint32_t in = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (i + c >= lo && i + c < s1) in |= 1u << c;
      gt &= in;
      eq &= in;
    }
  };
  int ngt = 0, neq = 0;
  for (int i = s0 + lane * 4; i < s1; i += 128) {
    float x[4];
    uint32_t gt, eq;
    load4(i, x);
    classify(i, x, gt, eq);
    ngt += __popc(gt);
    neq += __popc(eq);
  }
  ngt = __reduce_add_sync(0xffffffffu, ngt);
  neq = __reduce_add_sync(0xffffffffu, neq);
  if (lane == 0) {
    warp_a[warp] = ngt;
    warp_b[warp] = neq;
  }
  __syncthreads();
  ngt = __reduce_add_sync(0xffffffffu, lane < warp ? warp_a[lane] : 0);
  neq = __reduce_add_sync(0xffffffffu, lane < warp ? warp_b[lane] : 0);
  const int end = a.budget - a.recent;
  for (int i0 = s0; i0 < s1; i0 += 128) {
    const int i = i0 + lane * 4;
    float x[4];
    uint32_t gt = 0, eq = 0;
    if (i < s1) {
      load4(i, x);
      classify(i, x, gt, eq);
    }
    // both counts up to this lane in one scan
    const uint32_t mine = __popc(gt) | (__popc(eq) << 16);
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t all = __shfl_sync(0xffffffffu, sum, 31);
    sum -= mine;
    const int ties = neq + (int)(sum >> 16);
    int at = lo + ngt + (int)(sum & 0xffffu) + min(ties, need);
    for (int more = __popc(eq) - max(0, need - ties); more > 0; --more)
      eq &= ~(0x80000000u >> __clz(eq));  // ties that do not stay
    const uint32_t take = gt | eq;
    if (take) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if ((take >> c & 1u) && at < end) {
          kept[at] = i + c;
          if (on_chip) row[at] = x[c];
          ++at;
        }
      }
    }
    ngt += (int)(all & 0xffffu);
    neq += (int)(all >> 16);
  }
  if (on_chip) return;
  __syncthreads();
  // a row that was not held on chip closes up here: a kept slot never moves
  // up, so a stretch is read before it or anything below it is overwritten
  for (int i0 = 0; i0 < a.budget; i0 += kSelThreads) {
    const int i = i0 + tid;
    float x = 0.0f;
    if (i < a.budget) x = row[kept[i]];
    __syncthreads();
    if (i < a.budget) row[i] = x;
  }
}

// Rows per CTA: their places are looked up once, a thread per row (kept
// list, block table, fresh blocks: three loads that wait for each other),
// and then the rows stream through with kUnroll pieces of 16 bytes of K and
// of V per thread in flight: 6.5 TB/s read and written at 823 MB, 56 us for
// 367 MB.
constexpr int kMoveRows = 256;  // at most
constexpr int kUnroll = 4;

__global__ void __launch_bounds__(kMoveThreads, 4)
kv_evict_move_kernel(const __grid_constant__ EvictArgs a, const __grid_constant__ LayerPtrs lp,
                     int layer0, int rows, int chunks, const int64_t* __restrict__ block_table,
                     const int32_t* __restrict__ evicted, const int32_t* __restrict__ kept,
                     const int32_t* __restrict__ fresh, uint32_t* status) {
  __shared__ int64_t from[kMoveRows], to[kMoveRows];  // rows of the cache, or -1
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  const int layer = blockIdx.y;
  const int chunk = blockIdx.x % chunks;
  const int bh = blockIdx.x / chunks, b = bh / a.hkv, h = bh - b * a.hkv;
  if (evicted[b] <= 0) return;
  const int r0 = chunk * rows, n = min(rows, a.budget - r0);
  const int p16 = a.d / 8;  // 16-byte pieces per row
  if (threadIdx.x < n) {
    const int i = r0 + threadIdx.x;
    const int s = kept[(((int64_t)(layer0 + layer) * a.B + b) * a.hkv + h) * a.budget + i];
    const int64_t to_blk = fresh[(int64_t)b * a.held + i / a.bs];
    const int64_t from_blk = block_table[(int64_t)b * a.max_blocks + s / a.bs];
    int64_t t = to_blk < 0 ? -1 : (to_blk * a.hkv + h) * a.bs + i % a.bs;
    if (from_blk < 0 || from_blk >= a.num_blocks) {
      kyro::dev::flag(status, KYRO_DEV_BAD_BLOCK);
      t = -1;
    }
    from[threadIdx.x] = (from_blk * a.hkv + h) * a.bs + s % a.bs;
    to[threadIdx.x] = t;
  }
  __syncthreads();
  const int total = n * p16;
  uint4* kc = reinterpret_cast<uint4*>(lp.k[layer]);
  uint4* vc = reinterpret_cast<uint4*>(lp.v[layer]);
  for (int base = 0; base < total; base += kUnroll * kMoveThreads) {
    uint4 x[kUnroll], y[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int it = base + u * kMoveThreads + threadIdx.x;
      const int r = it / p16, c = it - r * p16;
      if (it < total && to[r] >= 0) {
        x[u] = kc[from[r] * p16 + c];
        y[u] = vc[from[r] * p16 + c];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int it = base + u * kMoveThreads + threadIdx.x;
      const int r = it / p16, c = it - r * p16;
      if (it < total && to[r] >= 0) {
        kc[to[r] * p16 + c] = x[u];
        vc[to[r] * p16 + c] = y[u];
      }
    }
  }
}

// The pops, the releases, the table rows and the lengths, from what the
// selection left (this kernel changes the lengths and the free list, so its
// CTAs go by `evicted` and ws.top).  The old blocks of the cut sequences are
// numbered in batch and table order by a scan over tiles of one sequence per
// thread, and released by all CTAs' threads in turn.  If a sequence holds a
// shared (or invalid) block, one thread releases them all in order, so that
// holders of one block see each other's decrements: about 0.4 us a block.  24
// sequences x 2 layers of up to 4096 slots whose first 256 are shared by all
// take 1615 us that way, and 85 where nothing is.
//
// The move lets this kernel start once the selection is complete (each of its
// CTAs waits for that first), and reads nothing that is written here but the
// table: the releases run beside the move, and only the table's rows are
// written after it.
__global__ void __launch_bounds__(kCommitThreads)
kv_evict_commit_kernel(const __grid_constant__ EvictArgs a, int64_t* __restrict__ block_table,
                       int64_t* __restrict__ context_lens, int32_t* __restrict__ free_stack,
                       int32_t* __restrict__ free_top, int32_t* __restrict__ ref_counts,
                       const int32_t* __restrict__ evicted, Scratch ws, uint32_t* status) {
  __shared__ int offs[kCommitThreads + 1];
  __shared__ int wsum[32];
  kyro::dev::pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int served = 0, odd = 0;
  long long released = 0;
  for (int b0 = 0; b0 < a.B; b0 += kCommitThreads) {
    const int b = b0 + tid;
    const bool cut = b < a.B && evicted[b] > 0;
    served += __syncthreads_count(cut);
    odd |= __syncthreads_or(cut && ws.odd[b]);
  }
  int top = ws.top[0] - served * a.held;
  const int64_t gtid = (int64_t)blockIdx.x * kCommitThreads + tid;
  const int64_t gsize = (int64_t)gridDim.x * kCommitThreads;
  auto old_blocks = [&](int b) {
    return (int)blocks_for((int64_t)evicted[b] + a.budget + a.reserved, a.bs);
  };
  if (odd) {
    kyro::dev::pdl_wait();
    if (blockIdx.x != 0) return;
    // the fresh blocks of every sequence are popped before any is released
    for (int64_t i = tid; i < (int64_t)a.B * a.held; i += kCommitThreads)
      if (evicted[i / a.held] > 0 && ws.fresh[i] >= 0) ref_counts[ws.fresh[i]] = 1;
    __syncthreads();
    if (tid == 0) {
      for (int seq = 0; seq < a.B; ++seq) {
        if (evicted[seq] <= 0) continue;
        const int n = old_blocks(seq);
        for (int i = 0; i < n; ++i) {
          int64_t* slot = &block_table[(int64_t)seq * a.max_blocks + i];
          const int64_t blk = *slot;
          *slot = i < a.held ? ws.fresh[(int64_t)seq * a.held + i] : -1;
          if (blk < 0) continue;
          if (blk >= a.num_blocks) {
            kyro::dev::flag(status, KYRO_DEV_BAD_BLOCK);
            continue;
          }
          if (ref_counts[blk] > 0) ref_counts[blk] -= 1;
          if (ref_counts[blk] == 0) {
            if (top < a.num_blocks)
              free_stack[top++] = (int32_t)blk;
            else
              kyro::dev::flag(status, KYRO_DEV_STACK_OVERFLOW);
          }
        }
      }
      *free_top = top;
    }
    for (int b = tid; b < a.B; b += kCommitThreads)
      if (evicted[b] > 0) context_lens[b] = a.budget;
    return;
  }
  // the old blocks of sequences b0 .. b0 + kCommitThreads - 1, numbered
  auto scan = [&](int b0) {
    const int b = b0 + tid;
    int inc = b < a.B && evicted[b] > 0 ? old_blocks(b) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      int w = wsum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += t;
      }
      wsum[lane] = w;
    }
    __syncthreads();
    offs[tid + 1] = inc + (warp ? wsum[warp - 1] : 0);
    if (tid == 0) offs[0] = 0;
    __syncthreads();
    return offs[kCommitThreads];
  };
  auto seq_of = [&](int64_t e) {
    int l = 0, r = kCommitThreads;  // offs[l] <= e < offs[r]
    while (r - l > 1) {
      const int m = (l + r) / 2;
      if (offs[m] <= e) l = m;
      else r = m;
    }
    return l;
  };
  for (int b0 = 0; b0 < a.B; b0 += kCommitThreads) {
    const int total = scan(b0);
    for (int64_t e = gtid; e < total; e += gsize) {
      const int l = seq_of(e), i = (int)e - offs[l];
      const int64_t blk = block_table[(int64_t)(b0 + l) * a.max_blocks + i];
      if (i < a.held) {
        const int32_t f = ws.fresh[(int64_t)(b0 + l) * a.held + i];
        if (f >= 0) ref_counts[f] = 1;
      }
      ref_counts[blk] = 0;
      if (top + released + e < a.num_blocks)
        free_stack[top + released + e] = (int32_t)blk;
      else
        kyro::dev::flag(status, KYRO_DEV_STACK_OVERFLOW);
    }
    const int b = b0 + tid;
    if (blockIdx.x == 0 && b < a.B && evicted[b] > 0) context_lens[b] = a.budget;
    released += total;
  }
  kyro::dev::pdl_wait();
  for (int b0 = 0; b0 < a.B; b0 += kCommitThreads) {
    // (one tile's numbers are still there)
    const int total = a.B > kCommitThreads ? scan(b0) : offs[kCommitThreads];
    for (int64_t e = gtid; e < total; e += gsize) {
      const int l = seq_of(e), i = (int)e - offs[l];
      block_table[(int64_t)(b0 + l) * a.max_blocks + i] =
          i < a.held ? ws.fresh[(int64_t)(b0 + l) * a.held + i] : -1;
    }
  }
  if (blockIdx.x == 0 && tid == 0) *free_top = (int)min((long long)a.num_blocks, top + released);
}

int check_evict(const kyro_evict_params* p) {
  const char* fn = "kyro_kv_evict";
  KY_REQUIRE(p, "%s: params is NULL", fn);
  KY_REQUIRE(p->batch >= 0 && p->batch <= 65535, "%s: batch = %d (0..65535)", fn, p->batch);
  KY_REQUIRE(p->block_size > 0 && p->max_blocks_per_seq > 0 && p->num_blocks > 0,
             "%s: block_size %d max_blocks_per_seq %d num_blocks %d", fn, p->block_size,
             p->max_blocks_per_seq, p->num_blocks);
  KY_REQUIRE((int64_t)p->max_blocks_per_seq * p->block_size < (1ll << 30),
             "%s: max_blocks_per_seq * block_size must be below 2^30", fn);
  KY_REQUIRE(p->num_layers >= 1 && p->num_kv_heads >= 1, "%s: num_layers %d num_kv_heads %d", fn,
             p->num_layers, p->num_kv_heads);
  KY_REQUIRE(p->head_dim > 0 && p->head_dim % 8 == 0 && p->head_dim <= 1024,
             "%s: head_dim %d (a multiple of 8, at most 1024)", fn, p->head_dim);
  KY_REQUIRE(p->budget >= 1 && p->num_sink >= 0 && p->num_recent >= 0 && p->num_reserved >= 0,
             "%s: budget %d num_sink %d num_recent %d num_reserved %d", fn, p->budget,
             p->num_sink, p->num_recent, p->num_reserved);
  KY_REQUIRE((int64_t)p->num_sink + p->num_recent <= p->budget,
             "%s: num_sink %d + num_recent %d exceed the budget %d", fn, p->num_sink,
             p->num_recent, p->budget);
  KY_REQUIRE((int64_t)p->budget + p->num_reserved <= (int64_t)p->max_blocks_per_seq * p->block_size,
             "%s: budget %d + num_reserved %d exceed the block table", fn, p->budget,
             p->num_reserved);
  KY_REQUIRE(p->score_slots >= p->budget, "%s: score_slots %lld below the budget %d", fn,
             (long long)p->score_slots, p->budget);
  return KYRO_OK;
}

int held_blocks(const kyro_evict_params* p) {
  return (int)(((int64_t)p->budget + p->num_reserved + p->block_size - 1) / p->block_size);
}

size_t scratch_bytes(const kyro_evict_params* p) {
  return 16 + (size_t)p->batch * (1 + held_blocks(p)) * 4;
}

}  // namespace

extern "C" {

size_t kyro_kv_evict_workspace_size(const kyro_evict_params* p) {
  if (check_evict(p) != KYRO_OK) return 0;
  return scratch_bytes(p);
}

int kyro_kv_evict(kyro_ctx* ctx, const kyro_evict_params* p, float* const* scores,
                  void* const* k_caches, void* const* v_caches, int64_t* block_table,
                  int64_t* context_lens, int32_t* free_stack, int32_t* free_top,
                  int32_t* ref_counts, int32_t* out_evicted, int32_t* out_kept, void* workspace,
                  size_t workspace_bytes) {
  const char* fn = "kyro_kv_evict";
  KY_NVTX("kyro_kv_evict");
  KY_TRY(kyro::enter(ctx));
  KY_TRY(check_evict(p));
  if (p->batch == 0) return KYRO_OK;
  KY_REQUIRE(scores && k_caches && v_caches && block_table && context_lens && free_stack &&
                 free_top && ref_counts && out_evicted && out_kept,
             "%s: a required pointer is NULL", fn);
  for (int i = 0; i < p->num_layers; ++i) {
    KY_REQUIRE(scores[i] && (uintptr_t)scores[i] % 4 == 0 && k_caches[i] && v_caches[i] &&
                   (uintptr_t)k_caches[i] % 16 == 0 && (uintptr_t)v_caches[i] % 16 == 0,
               "%s: layer %d pointer NULL or a cache not 16-byte aligned", fn, i);
    for (int j = 0; j < i; ++j)
      KY_REQUIRE(scores[i] != scores[j] && k_caches[i] != k_caches[j] && v_caches[i] != v_caches[j],
                 "%s: layers %d and %d share a buffer", fn, j, i);
  }
  const size_t need = kyro_kv_evict_workspace_size(p);
  if (!workspace || workspace_bytes < need)
    return kyro::set_error(KYRO_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn,
                           workspace_bytes, need);
  KY_REQUIRE((uintptr_t)workspace % 4 == 0, "%s: workspace must be 4-byte aligned", fn);
  EvictArgs a;
  a.B = p->batch;
  a.bs = p->block_size;
  a.max_blocks = p->max_blocks_per_seq;
  a.num_blocks = p->num_blocks;
  a.hkv = p->num_kv_heads;
  a.d = p->head_dim;
  a.budget = p->budget;
  a.sink = p->num_sink;
  a.recent = p->num_recent;
  a.reserved = p->num_reserved;
  a.held = held_blocks(p);
  a.score_slots = p->score_slots;
  Scratch ws;
  ws.top = (int32_t*)workspace;
  ws.odd = ws.top + 4;
  ws.fresh = ws.odd + p->batch;
  // rows per CTA of the move: as many as leave two waves of CTAs
  auto ctas = [&](int rows) {
    return (int64_t)((p->budget + rows - 1) / rows) * p->batch * p->num_kv_heads * p->num_layers;
  };
  int rows = kMoveRows;
  while (rows > 32 && ctas(rows) < 8ll * ctx->num_sms) rows /= 2;
  const int chunks = (p->budget + rows - 1) / rows;
  const int64_t blocks = (int64_t)chunks * p->batch * p->num_kv_heads;
  KY_REQUIRE(blocks < (1ll << 31) && p->num_kv_heads <= 65535, "%s: batch too large", fn);
  // a row's scores are read five times: from shared memory when the longest
  // row that the table allows fits.  (What the table allows goes by its width:
  // 24 sequences x 2 layers of up to 4096 slots take 85 us with a table just
  // wide enough, 91 with one of 32768 slots, whose rows leave room for one CTA
  // per SM, and 85 with one of 131072, whose rows are read from memory.)
  const int64_t longest =
      std::min<int64_t>(p->score_slots, (int64_t)p->max_blocks_per_seq * p->block_size);
  const int cached = longest <= kRowCache ? ((int)longest + 3) / 4 * 4 : 0;
  KY_TRY(kyro::chunk::set_smem<kv_evict_select_kernel>(kRowCache * 4, ctx->device));
  for (int l0 = 0; l0 < p->num_layers; l0 += kMaxLayers) {
    const int nl = std::min(kMaxLayers, p->num_layers - l0);
    LayerPtrs lp = {};
    for (int i = 0; i < nl; ++i) lp.scores[i] = scores[l0 + i];
    KY_TRY(kyro::launch_pdl(kv_evict_select_kernel,
                            dim3((unsigned)a.hkv + (l0 == 0), (unsigned)a.B, (unsigned)nl),
                            dim3(kSelThreads),
                            (size_t)cached * 4, ctx->stream, "kv_evict_select_kernel", a, lp, l0,
                            cached, (const int64_t*)context_lens, (const int32_t*)free_stack,
                            (const int32_t*)free_top, out_evicted, out_kept,
                            (const int64_t*)block_table, (const int32_t*)ref_counts, ws,
                            ctx->d_status));
  }
  for (int l0 = 0; l0 < p->num_layers; l0 += kMaxLayers) {
    const int nl = std::min(kMaxLayers, p->num_layers - l0);
    LayerPtrs lp = {};
    for (int i = 0; i < nl; ++i) {
      lp.k[i] = (uint8_t*)k_caches[l0 + i];
      lp.v[i] = (uint8_t*)v_caches[l0 + i];
    }
    KY_TRY(kyro::launch_pdl(kv_evict_move_kernel, dim3((unsigned)blocks, (unsigned)nl),
                            dim3(kMoveThreads), 0, ctx->stream, "kv_evict_move_kernel", a, lp, l0,
                            rows, chunks, (const int64_t*)block_table,
                            (const int32_t*)out_evicted, (const int32_t*)out_kept,
                            (const int32_t*)ws.fresh, ctx->d_status));
  }
  // enough CTAs for one release per thread at the longest table
  const int64_t most = (int64_t)p->batch * p->max_blocks_per_seq;
  const int commit_ctas =
      (int)std::min<int64_t>(16, (most + kCommitThreads - 1) / kCommitThreads);
  return kyro::launch_pdl(kv_evict_commit_kernel, dim3((unsigned)commit_ctas),
                          dim3(kCommitThreads), 0, ctx->stream, "kv_evict_commit_kernel", a,
                          block_table, context_lens, free_stack, free_top, ref_counts,
                          (const int32_t*)out_evicted, ws, ctx->d_status);
}

}  // extern "C"
