// qk_norm_rope.cu -- per-head RMS norm of queries and keys, rotary position
// embedding and the paged K/V store of a packed batch of prompt chunks, in
// one pass (RmsNorm and RotaryEmbedding, src/model/layers.rs:4-61, and the
// append of src/model/llama.rs:81-102).
//
// For a head x of D elements at position t, with h = D / 2:
//     r = 1 / sqrt(sum(x^2) / D + eps),   y = x * r * w
//     z[i] = y[i] cos(a_i) - y[i+h] sin(a_i)
//     z[i+h] = y[i+h] cos(a_i) + y[i] sin(a_i),   a_i = t / theta^(2i/D)
// in fp32, rounded to bf16 once.  a_i is formed and reduced to [-pi, pi] in
// 64 bits: an fp32 product t * f_i is off by up to t * 2^-24, which at
// position 100000 is 0.006 rad, above the output's own rounding.
//
// Bound by memory: every row of q, k and v is read once and written once.
// An item is (token, head, c): 16 bytes of the head's first half and the 16
// of its second half they are rotated with, so a rotation stays in a thread
// and a norm is a shuffle over the head's D / 16 items.  A CTA takes a run of
// consecutive tokens: it looks up their sequences and forms their D / 2
// angles once, for all heads, and then streams their items, each thread with
// its next item's loads in flight while it works on one.  That takes 64
// registers, 4 CTAs per SM; two items ahead at 3 CTAs takes 129 us where this
// takes 123 (16384 rows of 64 + 16 heads of 128, no norm, 672 MB: 5.4 TB/s),
// two at a time 139.  A ragged 7721 rows of 28 + 8 heads of 64 with norms:
// 18 us, of which the instructions are about half; 64 decode tokens: 4.5 us
// (4.3 without the look at all sequences' starts).
#include <algorithm>
#include <cmath>

#include "chunk.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;   // head_dim / 2
constexpr int kMaxTokens = 48;  // tokens per CTA, as far as their angles fit
constexpr int kMaxAngles = 44 * 1024;  // bytes, of the 48 KB that every launch may have
constexpr int kCtasPerSm = 4;

struct NormRopeArgs {
  int B, T, hq, hkv, d, bs, max_blocks, num_blocks, tokens;
  uint32_t heads_magic;  // 2^32 / (hq + 2 hkv), rounded up
  float eps;
  int64_t qs, ks, vs, os;  // row strides, in elements
  double inv_freq[kMaxHalf];
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// G: lanes per head, the power of two that holds its D / 16 items.
template <int G>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a, const uint16_t* __restrict__ q_norm,
                    const uint16_t* __restrict__ k_norm, const int64_t* __restrict__ positions,
                    const uint16_t* q, const uint16_t* __restrict__ k_new,
                    const uint16_t* __restrict__ v_new, const int32_t* __restrict__ starts,
                    const int64_t* __restrict__ block_table,
                    const int64_t* __restrict__ context_lens, uint16_t* q_out,
                    uint16_t* __restrict__ k_cache, uint16_t* __restrict__ v_cache,
                    uint32_t* status) {
  extern __shared__ __align__(16) float cs[];  // [tokens][half] cosines, then the sines
  __shared__ int64_t sh_row[kMaxTokens];  // cache row of head 0: (blk * hkv) * bs + offset, or -1
  __shared__ int64_t sh_pos[kMaxTokens];
  __shared__ int sh_ok[kMaxTokens];
  kyro::dev::pdl_wait();
  kyro::dev::pdl_trigger();
  const int t0 = blockIdx.x * a.tokens;
  const int nt = min(a.tokens, a.T - t0);
  const int half = a.d / 2, hv = a.d / 16;
  const int heads = a.hq + 2 * a.hkv;
  const int items = nt * heads * G;
  float* sn = cs + a.tokens * half;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a thread's part of its heads is the same in all items; the token and head
  // of item `it` (exact: an item's number times the heads is below 2^32)
  const int c = threadIdx.x % G;
  auto place = [&](int it, int& tl, int& h) {
    const int hh = it / G;
    tl = (int)__umulhi((uint32_t)hh, a.heads_magic);
    h = hh - tl * heads;
  };

  struct Item {
    uint4 x1, x2;
  };
  auto load = [&](Item& r, int it) {
    int tl, h;
    place(it, tl, h);
    if (it < items && c < hv) {
      const int64_t t = t0 + tl;
      const uint16_t* src = h < a.hq ? q + t * a.qs + (int64_t)h * a.d
                            : h < a.hq + a.hkv
                                ? k_new + t * a.ks + (int64_t)(h - a.hq) * a.d
                                : v_new + t * a.vs + (int64_t)(h - a.hq - a.hkv) * a.d;
      r.x1 = reinterpret_cast<const uint4*>(src)[c];
      r.x2 = reinterpret_cast<const uint4*>(src)[hv + c];
    } else {
      r.x1 = r.x2 = make_uint4(0, 0, 0, 0);
    }
  };
  Item cur, nxt;
  load(cur, threadIdx.x);

  // The sequences that cannot be taken are flagged by one CTA; all see whether
  // the starts are in order, which the search goes by.  Loaded here and looked
  // at behind the search, from the last warp down, since a decode step's
  // tokens are the first warps'.
  const int b_first = kThreads - 1 - (int)threadIdx.x;
  int first0 = 0, first1 = 0;
  int64_t first_len = 0;
  if (b_first < a.B) {
    first0 = __ldg(&starts[b_first]);
    first1 = __ldg(&starts[b_first + 1]);
    if (blockIdx.x == 0) first_len = __ldg(&context_lens[b_first]);
  }
  // by one lane: where token t of sequence b goes (b -1 or a.B: it is padding)
  auto put = [&](int tl, int t, int b) {
    int64_t row = -1, pos = 0;
    int ok = 0;
    if (b >= 0 && b < a.B) {
      const kyro::chunk::Seq s =
          kyro::chunk::seq_of(b, starts, context_lens, a.T, a.max_blocks * a.bs);
      const int j = t - s.start;
      if (s.n > 0 && j >= 0 && j < s.n) {
        ok = 1;
        const int slot = s.ctx + j;
        pos = positions ? positions[t] : slot;
        const int64_t blk = block_table[(int64_t)b * a.max_blocks + slot / a.bs];
        if (blk < 0 || blk >= a.num_blocks)
          kyro::dev::flag(status, KYRO_DEV_BAD_BLOCK);
        else
          row = blk * a.hkv * a.bs + slot % a.bs;
      }
    }
    sh_row[tl] = row;
    sh_pos[tl] = pos;
    sh_ok[tl] = ok;
  };
  // the sequence of each token: the last b with starts[b] <= t, by two
  // rounds of 32 lanes (B <= 1023; more rounds beyond)
  for (int tl = warp; tl < nt; tl += kThreads / 32) {
    const int t = t0 + tl;
    int lo = 0, n = a.B + 1;  // starts[lo .. lo + n) holds the answer's upper neighbour
    while (n > 1) {
      const int step = (n + 31) / 32;
      const int i = lo + lane * step;
      const bool le = lane * step < n && __ldg(&starts[i]) <= t;
      const int cnt = __popc(__ballot_sync(0xffffffffu, le));
      if (cnt == 0) {
        lo = -1;
        break;
      }
      const int first = (cnt - 1) * step;
      lo += first;
      n = min(step, n - first);
    }
    if (lane == 0) put(tl, t, lo);
  }
  bool disorder = first0 > first1;
  bool bad = blockIdx.x == 0 &&
             kyro::chunk::seq_from(first0, first1, first_len, a.T, a.max_blocks * a.bs).bad;
  for (int b = b_first + kThreads; b < a.B; b += kThreads) {
    disorder |= __ldg(&starts[b]) > __ldg(&starts[b + 1]);
    bad |= blockIdx.x == 0 &&
           kyro::chunk::seq_of(b, starts, context_lens, a.T, a.max_blocks * a.bs).bad;
  }
  if (bad) kyro::dev::flag(status, KYRO_DEV_BAD_LENGTH);
  if (__syncthreads_or(disorder)) {
    // a start that decreases leads the search astray: the last of the
    // sequences that hold the token, among those that can be taken
    for (int tl = warp; tl < nt; tl += kThreads / 32) {
      const int t = t0 + tl;
      int last = -1;
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        bool holds = false;
        if (b0 + lane < a.B) {
          const kyro::chunk::Seq s =
              kyro::chunk::seq_of(b0 + lane, starts, context_lens, a.T, a.max_blocks * a.bs);
          // (a start may be any number where there are no rows)
          holds = s.n > 0 && t >= s.start && t - s.start < s.n;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, holds);
        if (m) last = b0 + 31 - __clz(m);
      }
      if (lane == 0) put(tl, t, last);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int tl = i / half, f = i - tl * half;
    // reduced by a multiple of 2 pi, whose two parts hold 106 bits
    const double ang = (double)sh_pos[tl] * a.inv_freq[f];
    const double k = rint(ang * 0.15915494309189535);
    const float r = (float)fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, ang));
    float s, c;
    sincosf(r, &s, &c);
    cs[tl * half + f] = c;
    sn[tl * half + f] = s;
  }
  __syncthreads();

  const float inv_d = 1.0f / (float)a.d;
  // (a warp's lanes all stay to the end: items are counted in whole warps)
  for (int base = 0; base + warp * 32 < items; base += kThreads, cur = nxt) {
    const int it = base + threadIdx.x;
    load(nxt, it + kThreads);
    int tl, h;
    place(it, tl, h);
    uint4 o1 = cur.x1, o2 = cur.x2;
    float f1[8], f2[8];
    unpack8(o1, f1);
    unpack8(o2, f2);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += f1[e] * f1[e] + f2[e] * f2[e];
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (it >= items || c >= hv || !sh_ok[tl]) continue;
    if (h < a.hq + a.hkv) {
      const uint16_t* w = h < a.hq ? q_norm : k_norm;
      if (w) {
        const float r = rsqrtf(ss * inv_d + a.eps);
        float w1[8], w2[8];
        unpack8(__ldg(reinterpret_cast<const uint4*>(w) + c), w1);
        unpack8(__ldg(reinterpret_cast<const uint4*>(w) + hv + c), w2);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f1[e] *= r * w1[e];
          f2[e] *= r * w2[e];
        }
      }
      const float4* cp = reinterpret_cast<const float4*>(cs + tl * half + c * 8);
      const float4* sp = reinterpret_cast<const float4*>(sn + tl * half + c * 8);
      float z1[8], z2[8];
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const float4 x = cp[v], y = sp[v];
        const float co[4] = {x.x, x.y, x.z, x.w}, si[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z1[4 * v + e] = f1[4 * v + e] * co[e] - f2[4 * v + e] * si[e];
          z2[4 * v + e] = f2[4 * v + e] * co[e] + f1[4 * v + e] * si[e];
        }
      }
      o1 = pack8(z1);
      o2 = pack8(z2);
    }
    uint4* dst;
    if (h < a.hq) {
      dst = reinterpret_cast<uint4*>(q_out + (int64_t)(t0 + tl) * a.os + (int64_t)h * a.d);
    } else {
      if (sh_row[tl] < 0) continue;
      const int kvh = h < a.hq + a.hkv ? h - a.hq : h - a.hq - a.hkv;
      uint16_t* cache = h < a.hq + a.hkv ? k_cache : v_cache;
      dst = reinterpret_cast<uint4*>(cache + (sh_row[tl] + (int64_t)kvh * a.bs) * a.d);
    }
    dst[c] = o1;
    dst[hv + c] = o2;
  }
}

}  // namespace

extern "C" int kyro_qk_norm_rope_kv_write(
    kyro_ctx* ctx, const kyro_chunk_params* p, float rope_theta, float eps, const void* q_norm,
    const void* k_norm, const int64_t* positions, const void* q, const void* k_new,
    const void* v_new, const int32_t* chunk_starts, const int64_t* block_table,
    const int64_t* context_lens, void* q_out, void* k_cache, void* v_cache) {
  const char* fn = "kyro_qk_norm_rope_kv_write";
  KY_NVTX("kyro_qk_norm_rope_kv_write");
  KY_TRY(kyro::enter(ctx));
  KY_TRY(kyro::chunk::check_params(p, fn));
  KY_REQUIRE(p->head_dim > 0 && p->head_dim % 16 == 0 && p->head_dim <= 2 * kMaxHalf,
             "%s: head_dim %d (a multiple of 16, at most %d)", fn, p->head_dim, 2 * kMaxHalf);
  KY_REQUIRE(rope_theta > 0.0f, "%s: rope_theta = %g", fn, (double)rope_theta);
  KY_REQUIRE(eps >= 0.0f, "%s: eps = %g", fn, (double)eps);
  const int d = p->head_dim;
  const int64_t dq = (int64_t)p->num_heads * d, dkv = (int64_t)p->num_kv_heads * d;
  KY_REQUIRE(kyro::chunk::stride_ok(p->q_stride, dq) && kyro::chunk::stride_ok(p->k_stride, dkv) &&
                 kyro::chunk::stride_ok(p->v_stride, dkv) &&
                 kyro::chunk::stride_ok(p->out_stride, dq),
             "%s: a row stride is shorter than its row or not a multiple of 8", fn);
  if (p->batch == 0 || p->num_tokens == 0) return KYRO_OK;
  KY_REQUIRE(q && k_new && v_new && chunk_starts && block_table && context_lens && q_out &&
                 k_cache && v_cache,
             "%s: a required pointer is NULL", fn);
  for (const void* x : {q_norm, k_norm, q, k_new, v_new, (const void*)q_out,
                        (const void*)k_cache, (const void*)v_cache})
    KY_REQUIRE((uintptr_t)x % 16 == 0, "%s: tensors must be 16-byte aligned", fn);
  const int hv = d / 16;
  const int g = hv <= 1 ? 1 : hv <= 2 ? 2 : hv <= 4 ? 4 : hv <= 8 ? 8 : 16;
  const int64_t heads = (int64_t)p->num_heads + 2ll * p->num_kv_heads;
  KY_REQUIRE(heads <= 8192, "%s: %lld heads of q, k and v (at most 8192)", fn, (long long)heads);
  NormRopeArgs a;
  a.B = p->batch;
  a.T = p->num_tokens;
  a.hq = p->num_heads;
  a.hkv = p->num_kv_heads;
  a.d = d;
  a.bs = p->block_size;
  a.max_blocks = p->max_blocks_per_seq;
  a.num_blocks = p->num_blocks;
  a.heads_magic = (uint32_t)(((1ull << 32) + heads - 1) / heads);
  // one wave of CTAs, each with its run of tokens
  const int wave = kCtasPerSm * ctx->num_sms;
  a.tokens = std::min({kMaxTokens, kMaxAngles / (4 * d), (p->num_tokens + wave - 1) / wave});
  a.eps = eps;
  a.qs = kyro::chunk::stride_or(p->q_stride, dq);
  a.ks = kyro::chunk::stride_or(p->k_stride, dkv);
  a.vs = kyro::chunk::stride_or(p->v_stride, dkv);
  a.os = kyro::chunk::stride_or(p->out_stride, dq);
  // theta^(-2i/d) one from the last: at most 127 products in 64 bits of a ratio
  // that is a rounding off itself, in all 254 half steps of 2^-53: off by 2^-45
  const double ratio = std::pow((double)rope_theta, -2.0 / d);
  double f = 1.0;
  for (int i = 0; i < d / 2; ++i, f *= ratio) a.inv_freq[i] = f;
  const dim3 grid((unsigned)((p->num_tokens + a.tokens - 1) / a.tokens));
  auto run = [&](auto kernel) {
    return kyro::launch_pdl(kernel, grid, dim3(kThreads), (size_t)a.tokens * d * 4, ctx->stream, "qk_norm_rope_kernel", a,
                            (const uint16_t*)q_norm, (const uint16_t*)k_norm, positions,
                            (const uint16_t*)q, (const uint16_t*)k_new, (const uint16_t*)v_new,
                            chunk_starts, block_table, context_lens, (uint16_t*)q_out,
                            (uint16_t*)k_cache, (uint16_t*)v_cache, ctx->d_status);
  };
  switch (g) {
    case 1: return run(qk_norm_rope_kernel<1>);
    case 2: return run(qk_norm_rope_kernel<2>);
    case 4: return run(qk_norm_rope_kernel<4>);
    case 8: return run(qk_norm_rope_kernel<8>);
    default: return run(qk_norm_rope_kernel<16>);
  }
}
