// Attention of many rows (prompts, chunks of them, several new tokens of many heads) over a paged key-value cache, on the tensor cores.
//
// A tile is up to 128 rows: all query heads of a key head for as many tokens as fit, so every key and value that is fetched serves the
// whole group.  One CTA per SM works on a pair of neighbouring tiles with the same ring of key and value blocks (128 tokens each): while the
// tensor cores multiply for one tile, the other's scores go through the softmax.
//     S = Q K^T   tcgen05.mma, both operands in shared memory, 128 x 128 fp32 in tensor memory
//     P           a thread has a row: maximum, 2^(s - m), sum, rounded to the cache's type, stored over S as the next operand
//     O += P V    tcgen05.mma, P in tensor memory, V [token][dim] in shared memory (rows along N); the first 64 keys' products run
//                 beside the weights of the others
// O stays in tensor memory; it is multiplied only when a row's maximum has grown by more than 2^8 since it was last set, by the softmax
// warps themselves: S of a block complete means that O of the block before is, since the MMAs of a CTA complete in order.
//
// Warps: 0 TMA (the pages of a block: one load per page and 64 dims; a page behind the last token lies outside the tensor map, which
// gives zeros), 1 MMA, 2 zeroes the values of a block that nobody sees, 3 hands out the work (Plan), 4..7 and 8..11 the rows of the two tiles.
//
// What bounds it: a prompt of 8192 tokens of 32 heads over 8 key heads takes 460 us (1200 TFLOP/s, 0.73 of cuBLAS' burst), 537 in a long
// row of calls, where the power cap lowers the clock (1030, 0.74 of cuBLAS' rate there).  The same
// launches without the softmax take 342 us: S reads 8 KB of shared memory for every 64 clocks of the tensor core and V and the ring's
// filling the rest of its 128 bytes a clock.  A block takes 3500 clocks: the
// softmax of a tile 2100 (of which the special-function unit has 770) and its products 1300 behind it; the other tile's fill the gaps of
// both.  Short prompts (2048 x 32 heads 50.5 us, 0.42): 12000 clocks until the first scores, 9000 between two items of a CTA.  A cap adds
// six packed operations for two scores as long as all of a block are below 0.4 of it: 512 tokens of 28 heads on 30000 take 331 us (670
// TFLOP/s), without a cap 254.  Larger ones go through tensor memory with two special functions each: 570 with queries eight times as
// large, and 85 instead of 64 for a prompt of 2048 with a cap of 30.  120 CTAs have half of a pair's keys each in that chunk; sevenths on
// all of them took 4 % less with the cap and 4 % more without.
// Partial results lie with the rows side by side, so that a row's thread adds up its own and reads 8 x 16 bytes of two parts at a time; with
// the dims side by side and a part after the other that took 41 us for two parts, and 100 tokens on 5000 (32 heads, ten parts) 174 instead
// of 38.
// Measured and not kept, us for 8192 tokens where the present form took 485: all 128 scores of a row in registers 494 (and 70 instead of 50
// for 2048: the longer code waits for its instructions), 64 at a time 551, 32 at a time 529, two threads a row 535..596, scores in two
// halves of N = 64 with a buffer each 523 (412 instead of 342 without the softmax).
// Pages of 8 bits (kBytes; a translation unit of its own, paged_attn_prompt8.cu): TMA brings the codes of a block into a ring of their own, and
// four more warps (12..15) make fp16 tiles of them, code times the scale of its 16 tokens, in the ring from which the products are made as always.
// Of scales below 2^-15 that product is no number of fp16: the tile holds more, by a power of two for 16 tokens, and their scores or weights less.
// That is 64 KB more through shared memory for a block, beside products that read 128 bytes a clock of it: 2048 tokens of 32 heads 58 us, 512 on
// 30000 416 with the cap, 292 without (16 bits 51, 334, 223 in the same row of calls).  With one warp for the tiles 75 and 573: 512 conversions a
// block and lane, one after the other.
#include <atomic>
#include <type_traits>

#include "paged_common.cuh"
#include "tmap.h"

namespace b200 {

namespace {

using namespace ptx;

#ifdef B200_PAGED_BYTES
constexpr bool kBytes = true;                  // pages of 8 bits
#else
constexpr bool kBytes = false;
#endif
constexpr int kRows = 128;                     // of a tile
constexpr int kBlock = 128;                    // tokens of a block of keys
constexpr int kThreads = kBytes ? 512 : 384;
constexpr int kTurners = 4;                    // 8 bits: warps that make fp16 tiles of codes
constexpr int kHalfBytes = kBlock * 128;       // 64 dims of a block
constexpr int kReady = 4;                      // value blocks between the zeroing warp and the MMA warp
constexpr int kWorks = 2;                      // work descriptors in flight
constexpr int kKept = 64;                      // sequences whose sizes the scheduling warp keeps
constexpr uint64_t kWaitNs = 4000000000ull;
constexpr int kRaw = 2;                        // blocks of codes in flight
constexpr int kLacks = 8;                      // blocks whose small scales are kept: the converting warps are at most five ahead of the rows
// 128 x 72 + 256 x 216 = 384 x 168; 256 x 40 + 256 x 216 = 512 x 128
constexpr int kAuxRegs = kBytes ? 40 : 72, kRowRegs = 216, kLaunchRegs = kBytes ? 128 : 168;
__device__ int g_prompt_error = 0;

struct PromptParams {
  CUtensorMap tm_q;                            // {D, heads, tokens}, box {64, group, tokens of a tile}, SWIZZLE_128B
  CUtensorMap tm_k, tm_v;                      // {D, page, kv_heads, pages}, box {64, page, 1, 1}, SWIZZLE_128B; 8 bits: box {D, page, 1, 1}
  PagedAttnParams a;
  int tile_tokens;
  int wide_out;                                // out is 32-byte aligned
  unsigned long long per_pair;                 // 2^40 / (tokens of a pair), rounded up: exact below 2^24 pairs
  unsigned long long* counters;                // [cut tile]
  PromptWords* words;
};

struct Work {
  int b, h;                                    // b < 0: no more
  int first, rows, base, length;               // of the sequence: first row, rows, position of the first, tokens in the cache
  int token;                                   // the pair's first
  int u0, u1;                                  // its chunk of blocks
  Range<kBlock> range;
  int first_u[2], last[2];                     // of each tile: its first block (u) behind the prefix, its last one or -1
  int chunk, chunks, cut_tile, part, part_step;
};
// The work of a launch, the same for every CTA: pairs of tiles in the order of the blocks they see, most first, each with all its key
// heads; a sequence of many blocks may have its pairs cut into chunks.  CTAs take the next one from a counter.
struct Plan {
  int c;                                       // a sequence of more blocks than this is cut
  int level, behind;                           // the blocks of the last item's pair (at first the most there are), and how many chunks have more
  struct Seq {
    int base, rows, most, first;               // position of the first row, rows, blocks of the last pair; first row
  };
  Seq* kept;                                   // of the first kKept sequences: a load from global memory is a trip to L2 here
  __device__ __forceinline__ static int blocks(int tokens) { return max((tokens + kBlock - 1) / kBlock, 1); }
  __device__ __forceinline__ static Seq load(const PromptParams& p, int b) {
    const PagedAttnParams& a = p.a;
    const Sequence s = sequence_of(a.c, b);
    Seq q = {s.length - s.rows, s.rows, blocks(s.length), s.first};
    if (a.causal && a.window) q.most = min(q.most, (a.window + 2 * p.tile_tokens) / kBlock + 2 + (a.prefix ? max(a.prefix[b], 0) / kBlock : 0));
    return q;
  }
  __device__ __forceinline__ Seq sequence(const PromptParams& p, int b) const { return b < kKept ? kept[b] : load(p, b); }
  __device__ __forceinline__ int chunks(const Seq& q) const { return q.most > c ? (q.most + c - 1) / c : 1; }
  // Pairs of tiles that hold so many tokens.  (A division by a variable takes this warp longer than the rest of its search.)
  __device__ __forceinline__ static int pairs_of(const PromptParams& p, int tokens) {
    return (int)((unsigned long long)(unsigned)(tokens + 2 * p.tile_tokens - 1) * p.per_pair >> 40);
  }
  __device__ __forceinline__ static int pairs(const PromptParams& p, const Seq& q) { return pairs_of(p, q.rows); }
  // Pairs of a sequence with x blocks or more (the number of blocks grows with the pair's place).
  __device__ __forceinline__ static int at_least(const PromptParams& p, const Seq& q, int x) {
    const int all = pairs(p, q), need = (x - 1) * kBlock + 1 - q.base;
    if (x > q.most) return 0;
    if (x <= 1 || !p.a.causal || need <= 0) return all;
    return max(all - (pairs_of(p, need) - 1), 0);
  }
  // Several ways to cut, one a lane: the longest pairs into 1, 2, ... chunks, all others into chunks no longer.  What a way costs: its
  // rounds of items over the CTAs times an item's average length, 3 blocks of time for its beginning and end and 6 more for partial
  // results; or the longest item.
  __device__ __forceinline__ Plan(const PromptParams& p, int lane, Seq* memory) : c(0x3fffffff), kept(memory) {
    const PagedAttnParams& a = p.a;
    int64_t total = 0;
    int longest = 1;
#pragma unroll 1
    for (int b = lane; b < a.c.batch; b += 32) {
      const Seq q = load(p, b);
      if (b < kKept) kept[b] = q;
      const int first = a.causal ? min(blocks(q.base + 2 * p.tile_tokens), q.most) : q.most, n = pairs(p, q);
      total += (int64_t)n * (first + q.most);
      if (n) longest = max(longest, q.most);
    }
    __syncwarp();
    total = warp_sum64(total) * a.c.kv_heads / 2;
    longest = __reduce_max_sync(0xffffffffu, longest);
    level = longest;
    behind = 0;
    if (a.c.batch > kKept) {                   // (looking at all ways would take longer than it saves)
      const int share = (int)((total + a.slots - 1) / a.slots);
      if (longest > 2 * share) c = max(share, 8);
      return;
    }
    const int mine = max((longest + lane) / (lane + 1), 4);
    int items = 0, parts = 0, cut = 0;
#pragma unroll 1
    for (int b = 0; b < a.c.batch; ++b) {
      const Seq q = kept[b];
      const int tiles = pairs(p, q) * a.c.kv_heads, n = q.most > mine ? (q.most + mine - 1) / mine : 1;
      items += tiles * n;
      if (n > 1) {
        parts += tiles * n;
        cut += tiles;
      }
    }
    int cost = 0x7fffffff;
    if (items > 0 && parts <= kPartsOfSlots * a.slots && cut * 2 <= kCutTiles) {
      const float rounds = (float)((items + a.slots - 1) / a.slots);
      cost = (int)fmaxf(fminf(rounds * ((float)total * 4.f / (float)items + (parts ? 36.f : 12.f)), 1e9f), (float)(min(mine, longest) * 4 + 12));
    }
    const int best = __reduce_min_sync(0xffffffffu, cost);
    c = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, cost == best)) - 1);
  }
  // Item `index`, which is larger than the one before, into w; w.b stays -1 where there is none.
  __device__ __forceinline__ void find(const PromptParams& p, int index, int lane, Work& w) {
    const PagedAttnParams& a = p.a;
    const int h = index % a.c.kv_heads, rank = index / a.c.kv_heads;
    int tile, n, in, cut = 0, parts = 0;
    if (a.c.batch == 1) {                      // the order is the pairs' own, the last one first
      n = chunks(kept[0]);
      if (rank >= pairs(p, kept[0]) * n) return;
      w.b = 0;
      tile = pairs(p, kept[0]) - 1 - (n > 1 ? rank / n : rank);
      in = n > 1 ? rank % n : 0;
    } else {
      // the largest x such that more than `rank` chunks belong to pairs with x blocks or more; ranks only grow, so it only falls: from the last
      // one downwards in growing steps, then between
      auto count = [&](int at) {
        int n = 0;
#pragma unroll 1
        for (int b = lane; b < a.c.batch; b += 32) {
          const Seq q = sequence(p, b);
          n += at_least(p, q, at) * chunks(q);
        }
        return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
      };
      int x = 0, above = level + 1, step = 1;
#pragma unroll 1
      while (above - x > 1) {
        const int mid = x > 0 || step > above ? (x + above) >> 1 : max(above - step, 1);
        const int n = count(mid);
        step *= 2;
        if (n > rank) {
          x = mid;
        } else {
          above = mid;
          behind = n;
        }
      }
      if (x == 0) return;
      level = x;
      in = rank - behind;
#pragma unroll 1
      for (int b0 = 0;; b0 += 32) {              // (ends: there are more than `in` of them)
        Seq q = {};
        int here = 0;
        if (b0 + lane < a.c.batch) {
          q = sequence(p, b0 + lane);
          here = (at_least(p, q, x) - at_least(p, q, x + 1)) * chunks(q);
        }
        const int upto = warp_scan(here, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, upto > in);
        if (hit) {
          const int l = __ffs(hit) - 1;
          in -= __shfl_sync(0xffffffffu, upto - here, l);
          w.b = b0 + l;
          break;
        }
        in -= __shfl_sync(0xffffffffu, upto, 31);
        if (b0 + 32 >= a.c.batch) return;
      }
      const Seq q = sequence(p, w.b);
      n = chunks(q);
      tile = pairs(p, q) - at_least(p, q, x + 1) - 1 - (n > 1 ? in / n : in);
      in = n > 1 ? in % n : 0;
      // place in scratch memory: behind the cut pairs of the sequences in front
      if (n > 1)
#pragma unroll 1
        for (int b = lane; b < w.b; b += 32) {
          const Seq o = sequence(p, b);
          if (chunks(o) > 1) {
            cut += pairs(p, o);
            parts += pairs(p, o) * chunks(o);
          }
        }
      cut = (int)__reduce_add_sync(0xffffffffu, (unsigned)cut);
      parts = (int)__reduce_add_sync(0xffffffffu, (unsigned)parts);
    }
    const Seq q = sequence(p, w.b);
    const Sequence s = {q.first, q.rows, q.base + q.rows};
    w.h = h;
    w.first = s.first;
    w.rows = s.rows;
    w.base = q.base;
    w.length = s.length;
    w.token = tile * 2 * p.tile_tokens;
    w.chunks = n;
    w.chunk = in;
    w.cut_tile = ((cut + tile) * a.c.kv_heads + h) * 2;
    w.part = (parts + tile * n + w.chunk) * a.c.kv_heads + h;
    w.part_step = a.c.kv_heads;
    w.range.set(a, s, w.b, w.token, min(w.token + 2 * p.tile_tokens, s.rows) - 1);
    w.u0 = 0;
    w.u1 = w.range.units;
    if (n > 1) {
      w.u0 = (int)((int64_t)w.range.units * w.chunk / n);
      w.u1 = (int)((int64_t)w.range.units * (w.chunk + 1) / n);
    }
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const int from = w.token + t * p.tile_tokens;
      Range<kBlock> r;
      r.set(a, s, w.b, from, min(from + p.tile_tokens, s.rows) - 1);
      // its own blocks begin where the pair's do, or later, and end where the pair's do, or earlier
      const int end = w.range.pre_units + (r.high + kBlock - 1) / kBlock - w.range.second;
      w.first_u[t] = w.range.pre_units + max(r.low / kBlock - w.range.second, 0);
      w.last[t] = min(max(end, w.range.pre_units), w.u1) - 1;
      if (w.last[t] < w.first_u[t]) w.last[t] = min(w.range.pre_units, w.u1) - 1;       // (none of its own: the prefix's)
      if (from >= s.rows || r.high == 0 || w.last[t] < w.u0) w.last[t] = -1;
    }
  }
};

// Whether a tile sees anything of block u.
struct Sight {
  int pre, first, last;
  __device__ __forceinline__ Sight(const Work& w, int t) : pre(w.range.pre_units), first(w.first_u[t]), last(w.last[t]) {}
  __device__ __forceinline__ bool operator()(int u) const { return u <= last && (u >= first || u < pre); }
};

template <int D>
struct Smem {
  static constexpr int kStages = D == 64 ? 8 : kBytes ? 4 : 5;
  static constexpr int kBlockBytes = kHalfBytes * (D / 64);
  unsigned char q[2][kBlockBytes];
  unsigned char ring[kStages][kBlockBytes];
  unsigned char raw[kBytes ? kRaw : 1][kBytes ? kBlock * D : 16];
  uint64_t raw_full[kRaw], raw_empty[kRaw], q_ready;
  uint2 lacks[kBytes ? kLacks : 1];            // 8 bits: of keys and of values, four bits for 16 tokens (see lacking_power)
  uint64_t q_full, q_empty;
  uint64_t full[kStages], empty[kStages], ready[kReady];
  uint64_t s_full[2], p_ready[2][2], o_full[2], o_empty[2];       // [tile][half of a block]
  uint64_t work_full[kWorks], work_empty[kWorks], issued, joined[2];
  Work work[kWorks];
  uint32_t tmem_base;
  int abort_flag;
  int last_here[2];
  unsigned epoch;
  Plan::Seq kept[kKept];
};

// Four MMAs along K under one election; the descriptors advance by 32 bytes (operands with rows along K), the address of an A in tensor
// memory by 8 columns and a B with rows along N by 2048 bytes (16 rows).
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, t, e;\n"
      ".reg .b64 a1, a2, a3, b1, b2, b3;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.eq.b32 t, 0, 0;\n"
      "add.s64 a1, %1, 2;\n"
      "add.s64 b1, %2, 2;\n"
      "add.s64 a2, %1, 4;\n"
      "add.s64 b2, %2, 4;\n"
      "add.s64 a3, %1, 6;\n"
      "add.s64 b3, %2, 6;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, t, e;\n"
      ".reg .b32 a1, a2, a3;\n"
      ".reg .b64 b1, b2, b3;\n"
      "elect.sync _|e, 0xffffffff;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.eq.b32 t, 0, 0;\n"
      "add.s32 a1, %1, 8;\n"
      "add.s64 b1, %2, 128;\n"
      "add.s32 a2, %1, 16;\n"
      "add.s64 b2, %2, 256;\n"
      "add.s32 a3, %1, 24;\n"
      "add.s64 b3, %2, 384;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n"
      "}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Bounded wait of a whole warp; false: it ran out, here or in another warp, and the kernel ends.  The lanes vote on every outcome: tensor
// memory is read and written by whole warps, so one lane must not go on where another has given up.  (A barrier that is complete stays so
// until this warp has gone on: lanes can only see it late.)
template <bool kRelaxed>
__device__ __forceinline__ bool wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 1; i < 0x7fffffffu; ++i) {
    if (kRelaxed) __nanosleep(100);
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
    if ((i & 127u) == 0 && __any_sync(0xffffffffu, globaltimer_ns() - t0 > kWaitNs)) break;
  }
  *abort_flag = 1;
  atomicExch(&g_prompt_error, code);
  return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return wait_long<false>(bar, parity, abort_flag, code);
}
// The same with a pause between two looks, for warps that have time.
__device__ __forceinline__ bool wait_relaxed(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return wait_long<true>(bar, parity, abort_flag, code);
}

// 2^x of two values without the special-function unit: x = n + f with n the nearest whole number (by adding 1.5 * 2^23, whose sum has n
// in its low bits), a polynomial of degree 4 for 2^f on [-1/2, 1/2] (least largest relative error, found by the exchange
// algorithm: 2.7e-6; a weight is rounded to 2^-12 or worse right after), n added to the exponent.
// x from -126 on, below that 2^-126.
__device__ __forceinline__ void exp2_poly(float& x, float& y) {
  constexpr float c[5] = {0.9999993f, 0.6931218f, 0.24024744f, 0.05591786f, 0.009570102f};
  constexpr float kMagic = 12582912.f;
  const float u = fmaxf(x, -126.f), v = fmaxf(y, -126.f);
  float tu = u, tv = v, nu, nv, fu, fv, pu = c[4], pv = pu;
  add2(tu, tv, kMagic, kMagic);
  nu = tu;
  nv = tv;
  add2(nu, nv, -kMagic, -kMagic);
  fma2(fu, fv, nu, nv, -1.f, -1.f, u, v);
#pragma unroll
  for (int i = 3; i >= 0; --i) fma2(pu, pv, pu, pv, fu, fv, c[i], c[i]);
  x = __uint_as_float(__float_as_uint(pu) + (__float_as_uint(tu) << 23));
  y = __uint_as_float(__float_as_uint(pv) + (__float_as_uint(tv) << 23));
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {        // (NaN where one of them is)
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// What happens to a score before the softmax: a scale > 0; that and a cap; that and a bias by distance; anything.
constexpr int kPlain = 0, kCapped = 1, kSloped = 2, kGeneral = 3;     // (and kWide: with a cap for which Cap::any will not do)
// Pairs of weights of eight that go that way: 8192 tokens 0 487, 2 479, 3 495, 4 596 us.
constexpr int kPolyOfEight = 2;

// Pairs of 16-bit values to fp16; a bf16 value beyond fp16's range becomes an infinity.
[[maybe_unused]] __device__ __forceinline__ uint32_t to_half2(__half, uint32_t v) { return v; }
[[maybe_unused]] __device__ __forceinline__ uint32_t to_half2(__nv_bfloat16, uint32_t v) {
  const float2 f = unpack2(__nv_bfloat16(), v);
  return pack2(__half(), f.x, f.y);
}

// 8 bits: the power of two by which a scale below 2^-15 (0 otherwise; 9 at most) is made 2^-15 to 2^-14, so that code times scale is a number of
// fp16 for all codes.  Scores of its keys are made smaller by it, and so are the weights of its values.
[[maybe_unused]] __device__ __forceinline__ int lacking_power(uint32_t half_bits) { return half_bits - 1u < 0x1ffu ? __clz(half_bits) - 22 : 0; }

// A row's 128 scores, and 64 of its weights in pairs, by those powers; not in line, where they would slow the loop down that hardly ever wants them.
[[maybe_unused]] __device__ __noinline__ void smaller_scores(uint32_t at, uint32_t lacks) {
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    uint32_t x[16];
    tmem_ld_32x32b_x16(at + 16 * i, x);
    tmem_ld_wait();
    const float f = power_of_two(-(int)(lacks >> 4 * i & 15u));
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
    tmem_st_32x32b_x16(at + 16 * i, x);
  }
  tmem_st_wait();
}
[[maybe_unused]] __device__ __noinline__ void smaller_weights(uint32_t at, uint32_t lacks) {
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    uint32_t x[16];
    tmem_ld_32x32b_x16(at + 16 * i, x);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const __half2 f = __float2half2_rn(power_of_two(-(int)(lacks >> (8 * i + 4 * (j / 8)) & 15u)));
      const __half2 w = __hmul2(*reinterpret_cast<const __half2*>(&x[j]), f);
      x[j] = *reinterpret_cast<const uint32_t*>(&w);
    }
    tmem_st_32x32b_x16(at + 16 * i, x);
  }
}

template <typename T, int D, int kForm, bool kWide>
__global__ void __launch_bounds__(kThreads, 1)
paged_prompt_kernel(const __grid_constant__ PromptParams p) {
  using Shared = Smem<D>;
  constexpr int kStages = Shared::kStages, kBlockBytes = Shared::kBlockBytes, kHalves = D / 64;
  using M = typename std::conditional<kBytes, __half, T>::type;          // what is multiplied
  constexpr bool kTurnQ = !std::is_same<T, M>::value;
  constexpr uint32_t kIdescS = umma_idesc_16bit_f32(kRows, kBlock, std::is_same<M, __nv_bfloat16>::value, false);
  constexpr uint32_t kIdescO = umma_idesc_16bit_f32(kRows, D, std::is_same<M, __nv_bfloat16>::value, true);
  extern __shared__ unsigned char smem_unaligned[];
  Shared& sm = *reinterpret_cast<Shared*>(smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u));
  volatile int* abort_flag = &sm.abort_flag;
  const PagedAttnParams& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int i = 0; i < kStages; ++i) { mbar_init(&sm.full[i], kBytes ? kTurners : 1); mbar_init(&sm.empty[i], 1); }
    for (int i = 0; i < kReady; ++i) mbar_init(&sm.ready[i], kBytes ? kTurners : 1);
    for (int i = 0; i < kRaw; ++i) { mbar_init(&sm.raw_full[i], 1); mbar_init(&sm.raw_empty[i], kTurners); }
    mbar_init(&sm.q_ready, kTurners);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.p_ready[t][0], 4);
      mbar_init(&sm.p_ready[t][1], 4);
      mbar_init(&sm.o_full[t], 1);
      mbar_init(&sm.o_empty[t], 4);
      mbar_init(&sm.joined[t], 4);
    }
    mbar_init(&sm.issued, 1);
    for (int i = 0; i < kWorks; ++i) { mbar_init(&sm.work_full[i], 1); mbar_init(&sm.work_empty[i], kBytes ? 10 + kTurners : 11); }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  pdl_wait();
  pdl_launch_dependents();

  // the next work descriptor; null: there is none, or a wait ran out.  It stays until it is handed back.
  uint32_t works = 0;
  auto next_work = [&]() -> const Work* {
    if (!wait(&sm.work_full[works % kWorks], (works / kWorks) & 1, abort_flag, 1)) return nullptr;
    const Work* w = &sm.work[works % kWorks];
    return w->b >= 0 ? w : nullptr;
  };
  auto work_done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.work_empty[works % kWorks]);
    ++works;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAuxRegs));
    if (warp == 0) {
      // ---------------------------------------------------------------------- TMA
      const int per_page = 7 - a.c.page_log2, pages = 1 << per_page;       // of a block
      uint32_t pos = 0, items = 0;
      auto issued = [&]() {
        if (lane == 0) mbar_arrive(&sm.issued);
        work_done();
      };
      for (const Work* wp; (wp = next_work()) != nullptr; issued()) {
        const Work& w = *wp;
        if (w.u1 == w.u0) continue;
        if (items > 0 && !wait_relaxed(&sm.q_empty, (items - 1) & 1, abort_flag, 2)) break;
        ++items;
        const int tiles = w.token + p.tile_tokens < w.rows ? 2 : 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sm.q_full, (uint32_t)(tiles * kHalves * p.tile_tokens * a.group * 128));
          for (int t = 0; t < tiles; ++t)
            for (int i = 0; i < kHalves; ++i)
              tma_load_3d(sm.q[t] + i * kHalfBytes, &p.tm_q, i * 64, w.h * a.group, w.first + w.token + t * p.tile_tokens, &sm.q_full);
        }
        // lane: page lane % pages of the block, dims 64 * (lane / pages); the page numbers a block ahead
        const int in_block = lane & (pages - 1), half = lane >> per_page;
        const int used = (w.length + (1 << a.c.page_log2) - 1) >> a.c.page_log2;
        const Range<kBlock> range = w.range;
        const int b = w.b, h = w.h, u1 = w.u1;
        auto page_at = [&](int u) {
          const int i = range.unit(u) * pages + in_block;
          return i < used ? page_of(a.c, b, i) : a.c.pages;                 // (behind the last page: outside the map)
        };
        int id = page_at(w.u0);
        bool ok = true;
        for (int u = w.u0; ok && u < u1; ++u) {
          const int id_next = u + 1 < u1 ? page_at(u + 1) : 0;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if constexpr (kBytes) {
              const uint32_t slot = pos % kRaw, round = pos / kRaw;
              if (round > 0 && !wait_relaxed(&sm.raw_empty[slot], (round - 1) & 1, abort_flag, 3)) { ok = false; break; }
              if (lane == 0) mbar_arrive_expect_tx(&sm.raw_full[slot], kBlock * D);
              __syncwarp();
              if (half == 0)
                tma_load_4d(sm.raw[slot] + (in_block << a.c.page_log2) * D, kv ? &p.tm_v : &p.tm_k, 0, 0, h, id, &sm.raw_full[slot]);
              ++pos;
              continue;
            }
            const uint32_t slot = pos % kStages, round = pos / kStages;
            if (round > 0 && !wait_relaxed(&sm.empty[slot], (round - 1) & 1, abort_flag, 3)) { ok = false; break; }
            if (lane == 0) mbar_arrive_expect_tx(&sm.full[slot], kBlockBytes);
            __syncwarp();
            if (half < kHalves)
              tma_load_4d(sm.ring[slot] + half * kHalfBytes + (in_block << (a.c.page_log2 + 7)), kv ? &p.tm_v : &p.tm_k, half * 64, 0, h, id,
                          &sm.full[slot]);
            ++pos;
          }
          id = id_next;
        }
        if (!ok) break;
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------------- MMA
      const uint64_t dq = umma_desc_k128(smem_u32(sm.q[0]));
      const uint64_t dk = umma_desc_k128(smem_u32(sm.ring[0]));
      const uint64_t dv = umma_desc_mn128(smem_u32(sm.ring[0]), kHalfBytes);
      constexpr uint32_t kStep = kBlockBytes >> 4, kHalfStep = kHalfBytes >> 4;
      uint32_t pos = 0, vblocks = 0, items = 0, n_p[2] = {0, 0}, n_o[2] = {0, 0};
      auto scores = [&](int t, uint32_t slot) {
#pragma unroll
        for (int i = 0; i < kHalves; ++i)
          mma4_ss(tmem + t * 128, dq + t * kStep + i * kHalfStep, dk + (uint64_t)(slot * kStep) + i * kHalfStep, kIdescS, i > 0);
        umma_commit(&sm.s_full[t]);
      };
      bool ok = true;
      for (const Work* wp; ok && (wp = next_work()) != nullptr; work_done()) {
        const int u0 = wp->u0, u1 = wp->u1, last[2] = {wp->last[0], wp->last[1]};
        const Sight sees[2] = {Sight(*wp, 0), Sight(*wp, 1)};
        if (u1 == u0) continue;
        if (!wait(kTurnQ ? &sm.q_ready : &sm.q_full, items & 1, abort_flag, 4)) break;
        ++items;
        bool begun[2] = {false, false};
        uint32_t slot = pos % kStages;
        if (!wait(&sm.full[slot], (pos / kStages) & 1, abort_flag, 5)) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (sees[t](u0)) scores(t, slot);
        umma_commit(&sm.empty[slot]);
        if (u1 - u0 == 1) umma_commit(&sm.q_empty);
        ++pos;
        for (int u = u0; ok && u < u1; ++u) {
          const uint32_t vslot = pos % kStages;
          ++pos;
          const bool more = u + 1 < u1;
          const uint32_t kslot = pos % kStages, kround = pos / kStages;
          bool keys = false;
          ok = wait(&sm.ready[vblocks % kReady], (vblocks / kReady) & 1, abort_flag, 6);
          ++vblocks;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && sees[t](u)) {
              if (!begun[t] && n_o[t] > 0) ok = wait(&sm.o_empty[t], (n_o[t] - 1) & 1, abort_flag, 7);
#pragma unroll
              for (int h = 0; h < 2; ++h) {         // (the first half's products run beside the second half's weights)
                ok = ok && wait(&sm.p_ready[t][h], n_p[t] & 1, abort_flag, 8);
                if (!ok) break;
                tc_fence_after_sync();
                mma4_ts(tmem + 256 + t * D, tmem + t * 128 + 32 * h, dv + (uint64_t)(vslot * kStep) + h * 512, kIdescO, begun[t] || h > 0);
              }
              begun[t] = true;
              ++n_p[t];
              if (ok && u == last[t]) {
                umma_commit(&sm.o_full[t]);
                ++n_o[t];
              }
            }
            if (ok && more && sees[t](u + 1)) {
              if (!keys) ok = wait(&sm.full[kslot], kround & 1, abort_flag, 9);
              keys = true;
              if (ok) scores(t, kslot);
            }
          }
          if (ok && more && !keys) ok = wait(&sm.full[kslot], kround & 1, abort_flag, 9);
          if (!ok) break;
          umma_commit(&sm.empty[vslot]);
          if (more) {
            umma_commit(&sm.empty[kslot]);
            if (u + 2 == u1) umma_commit(&sm.q_empty);
            ++pos;
          }
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------------- values that nobody sees: 0 * NaN is NaN
      uint32_t pos = 0, vblocks = 0;
      bool ok = true;
      for (const Work* wp; !kBytes && ok && (wp = next_work()) != nullptr; work_done()) {
        const Range<kBlock> range = wp->range;
        const int u1 = wp->u1;
        for (int u = wp->u0; u < u1; ++u, pos += 2) {
          const uint32_t slot = (pos + 1) % kStages, round = (pos + 1) / kStages;
          if (!wait_relaxed(&sm.full[slot], round & 1, abort_flag, 10)) { ok = false; break; }
          const int from = range.unit(u) * kBlock;
          const bool whole = from + kBlock <= range.pre || (from >= range.low && from + kBlock <= range.high);
          if (!whole) {
            for (int i = lane; i < kBlock * 8 * kHalves; i += 32) {
              const int token = from + ((i >> 3) & (kBlock - 1));
              if (!(token < range.pre || (token >= range.low && token < range.high)))
                reinterpret_cast<uint4*>(sm.ring[slot])[i] = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&sm.ready[vblocks % kReady]);
          ++vblocks;
        }
      }
    } else {
      // ---------------------------------------------------------------------- the work, longest tiles first
      if (lane == 0) sm.epoch = __ldcg(&p.words->epoch);   // (handed over with the first descriptor)
      Plan plan(p, lane, sm.kept);
      for (uint32_t i = 0;; ++i) {
        const uint32_t slot = i % kWorks, round = i / kWorks;
        if (round > 0 && !wait_relaxed(&sm.work_empty[slot], (round - 1) & 1, abort_flag, 11)) break;
        // the next item is taken when this one's loads are all on their way, two or three blocks before its end: taken earlier, the CTA with
        // the longest item would get one of the second longest too
        if (i > 0 && !wait_relaxed(&sm.issued, (i - 1) & 1, abort_flag, 15)) break;
        int index = blockIdx.x;
        if (i > 0) {
          if (lane == 0) index = gridDim.x + atomicAdd(&p.words->next, 1);
          index = __shfl_sync(0xffffffffu, index, 0);
        }
        Work w;
        w.b = -1;
        plan.find(p, index, lane, w);
        if (lane == 0) {
          sm.work[slot] = w;
          mbar_arrive(&sm.work_full[slot]);
        }
        if (w.b < 0) break;
      }
      // the CTA that comes last leaves the words as the next launch expects them (a CTA that has given up comes here too)
      if (lane == 0 && atomicAdd(&p.words->through, 1) == (int)gridDim.x - 1) {
        p.words->next = 0;
        p.words->through = 0;
        p.words->epoch = sm.epoch + 1;
      }
    }
  } else if (kBytes && warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAuxRegs));
    // ---------------------------------------------------------------------- 8 bits: tiles of fp16, in the layout in which TMA would put them
    if constexpr (kBytes) {
      const int turner = warp - 12;
      uint32_t pos = 0, vblocks = 0, items = 0;
      bool ok = true;
      for (const Work* wp; ok && (wp = next_work()) != nullptr; work_done()) {
        const Work& w = *wp;
        const Range<kBlock> range = w.range;
        const int u1 = w.u1;
        if (w.u1 == w.u0) continue;
        if (kTurnQ) {                                          // the queries, where they lie
          if (!wait(&sm.q_full, items & 1, abort_flag, 16)) break;
          const int tiles = w.token + p.tile_tokens < w.rows ? 2 : 1;
          uint4* at = reinterpret_cast<uint4*>(sm.q[0]);
#pragma unroll 4
          for (int i = turner * 32 + lane; i < tiles * (kBlockBytes / 16); i += kTurners * 32) {
            const uint4 v = at[i];
            at[i] = make_uint4(to_half2(T(), v.x), to_half2(T(), v.y), to_half2(T(), v.z), to_half2(T(), v.w));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.q_ready);
        }
        ++items;
        const int used = (w.length + (1 << a.c.page_log2) - 1) >> a.c.page_log2;
        // lane 0..7: the scale of 16 keys, 8..15: of 16 values; a block ahead
        auto scale_at = [&](int u) {
          const int token = range.unit(u) * kBlock + 16 * (lane & 7), page = token >> a.c.page_log2;
          if (lane >= 16 || page >= used) return __float2half(0.f);
          const int64_t id = page_of(a.c, w.b, page);
          const int in_page = (token & ((1 << a.c.page_log2) - 1)) >> 4;
          return __ldg((lane < 8 ? a.k_scales : a.v_scales) + ((id * a.c.kv_heads + w.h) << (a.c.page_log2 - 4)) + in_page);
        };
        __half next = scale_at(w.u0);
        for (int u = w.u0; ok && u < u1; ++u) {
          const uint32_t stored = __half_as_ushort(next);
          const int lacks = lacking_power(stored);
          const __half scale = __ushort_as_half((unsigned short)(stored << lacks));        // (of subnormal numbers the bits are the value)
          if (turner == 0) {                                   // (seen by the rows behind the scores, which wait for these keys)
            uint2 all = {0u, 0u};
            if (__builtin_expect(__any_sync(0xffffffffu, lacks), 0)) {
              const uint32_t bits = (uint32_t)lacks << 4 * (lane & 7);
              all = {__reduce_or_sync(0xffffffffu, lane < 8 ? bits : 0u), __reduce_or_sync(0xffffffffu, lane >= 8 ? bits : 0u)};
            }
            if (lane == 0) sm.lacks[vblocks % kLacks] = all;
          }
          if (u + 1 < u1) next = scale_at(u + 1);
          const int from = range.unit(u) * kBlock;
          const bool whole = from + kBlock <= range.pre || (from >= range.low && from + kBlock <= range.high);
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv, ++pos) {
            const uint32_t raw = pos % kRaw, slot = pos % kStages, round = pos / kStages;
            if (!wait(&sm.raw_full[raw], (pos / kRaw) & 1, abort_flag, 10) ||
                (round > 0 && !wait(&sm.empty[slot], (round - 1) & 1, abort_flag, 17))) {
              ok = false;
              break;
            }
            // 16 codes a lane and step, 16 tokens D / 32 steps.  Lanes of four have 64 codes of a token; where a token has two such halves, neighbours
            // of eight lanes have one half of a token and the other half of the next: the banks of all eight are different as they read and as
            // they write (chunks of 16 bytes, 2 c and 2 c + 1, swizzled by the token).
            const int half = D == 128 ? (lane >> 2 ^ lane >> 3) & 1 : 0;
            const int token0 = D == 128 ? (lane >> 2 & 1) + 2 * (lane >> 4) : lane >> 2, chunk = 2 * (lane & 3);
            const unsigned char* codes = sm.raw[raw] + token0 * D + half * 64 + (lane & 3) * 16;
            unsigned char* to = sm.ring[slot] + half * kHalfBytes + token0 * 128;
            constexpr int kStep = 512 / D;                     // tokens of a step
#pragma unroll
            for (int g = 0; g < kBlock / 16 / kTurners; ++g) {
              const int group = turner * (kBlock / 16 / kTurners) + g;
              const __half2 by = __half2half2(__shfl_sync(0xffffffffu, scale, 8 * kv + group));
              uint4 c[D / 32];
#pragma unroll
              for (int i = 0; i < D / 32; ++i) c[i] = *reinterpret_cast<const uint4*>(codes + (group * 16 + i * kStep) * D);
#pragma unroll
              for (int i = 0; i < D / 32; ++i) {
                const int token = group * 16 + i * kStep;      // (and token0)
                const uint32_t words[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
                uint32_t v[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  e4m3_to_half4(words[k], v[2 * k], v[2 * k + 1]);
#pragma unroll
                  for (int o = 0; o < 2; ++o) {
                    const __half2 value = __hmul2(*reinterpret_cast<const __half2*>(&v[2 * k + o]), by);
                    v[2 * k + o] = *reinterpret_cast<const uint32_t*>(&value);
                  }
                }
                if (kv && !whole) {
                  const int at = from + token + token0;
                  if (!(at < range.pre || (at >= range.low && at < range.high)))
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = 0;
                }
                unsigned char* row = to + token * 128;
                const int flip = (token + token0) & 7;
                *reinterpret_cast<uint4*>(row + ((chunk ^ flip) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ flip) << 4)) = make_uint4(v[4], v[5], v[6], v[7]);
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&sm.raw_empty[raw]);
              mbar_arrive(&sm.full[slot]);
              if (kv) mbar_arrive(&sm.ready[vblocks % kReady]);
            }
          }
          ++vblocks;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
    // ---------------------------------------------------------------------- the rows
    const int t = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t s_at = tmem + t * 128 + ((uint32_t)((warp & 3) * 32) << 16), o_at = s_at - t * 128 + 256 + t * D;
    uint32_t phases = 0;                         // parities: bit 0 of s_full, 1 of o_full, 2 of joined
    uint32_t blocks = 0;                         // 8 bits: of earlier items
    bool ok = true;
    // The four warps of the tile meet; false: one of them has given up (a barrier without a limit would wait for it for ever).
    auto tile_barrier = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.joined[t]);
      phases ^= 4;
      return wait(&sm.joined[t], phases >> 2 & 1 ^ 1, abort_flag, 14);
    };
    const int token_in_tile = r / a.group, head_in_group = r - token_in_tile * a.group;
    const float to_log2 = a.scale * kLog2e;
    const Cap cap(a.scale, a.cap);
    for (const Work* wp; ok && (wp = next_work()) != nullptr; work_done()) {
      const Work& w = *wp;
      const Sight sees(w, t);
      const Range<kBlock> range = w.range;
      const int u0 = w.u0, u1 = w.u1;
      const int token = w.token + t * p.tile_tokens + token_in_tile;
      const bool mine = token_in_tile < p.tile_tokens && token < w.rows;
      const int at = mine ? w.base + token : -1;
      const int head = w.h * a.group + head_in_group;
      const int tile_first = w.base + w.token + t * p.tile_tokens;
      const int tile_last = w.base + min(w.token + (t + 1) * p.tile_tokens, w.rows) - 1;
      const int window = a.window ? a.window : 0x7fffffff;
      const float slope = (kForm == kSloped || kForm == kGeneral) && a.slopes && mine ? a.slopes[head] * kLog2e : 0.f;
      float m = -INFINITY, l[4] = {0.f, 0.f, 0.f, 0.f};
      bool begun = false;
      for (int u = u0; u < u1; ++u) {
        if (!sees(u)) continue;
        if (!wait(&sm.s_full[t], phases & 1, abort_flag, 12)) { ok = false; break; }
        phases ^= 1;
        tc_fence_after_sync();
        uint2 lacks = {0u, 0u};
        if constexpr (kBytes) lacks = sm.lacks[(blocks + (u - u0)) % kLacks];
        // First pass: the maximum, 32 columns at a time, the next ones on their way; scores that a mask changes, or a cap or a bias where
        // its short form does not hold, go back to tensor memory.  Second pass: the weights.  (What does not fit in registers comes from
        // L2 with this much shared memory, and so do the instructions of long code.)
        const int from = range.unit(u) * kBlock;
        // (a row without a position sees nothing, the prefix neither)
        const bool whole = tile_first >= 0 && (from + kBlock <= range.pre || (from + kBlock - 1 <= tile_first && tile_last - from < window));
        uint32_t raw[2][32];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // (four chains: one would be 64 dependent steps)
        float top;
        auto highest = [&](const uint32_t(&x)[32]) {
#pragma unroll
          for (int j = 0; j < 16; ++j) tops[j & 3] = max3(tops[j & 3], __uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
        };
        auto all_tops = [&]() { return max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]); };
        const float bias = kForm == kSloped ? -slope * (float)(at - from) : 0.f;       // of the block's first key, which lies before the row
        bool direct = whole && kForm != kGeneral && (kForm != kSloped || from + kBlock - 1 <= tile_first);
        if (direct) tmem_ld_32x32b_x32(s_at, raw[0]);
        if constexpr (kBytes) {
          if (__builtin_expect(lacks.x != 0, 0)) {       // keys whose tile holds more
            if (direct) tmem_ld_wait();
            smaller_scores(s_at, lacks.x);
            if (direct) tmem_ld_32x32b_x32(s_at, raw[0]);
          }
        }
        if (direct) {
          float lows[2] = {INFINITY, INFINITY};
#pragma unroll 1
          for (int i = 0; i < 4; i += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t(&x)[32] = raw[h];
              tmem_ld_wait();
              if (i + h < 3) tmem_ld_32x32b_x32(s_at + 32 * (i + h + 1), raw[h ^ 1]);
              if (kForm == kSloped) {
                const float at_i = fmaf(slope, (float)(32 * (i + h)), bias);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  float v, w, bv, bw;
                  fma2(bv, bw, (float)(2 * j), (float)(2 * j + 1), slope, slope, at_i, at_i);
                  fma2(v, w, __uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]), to_log2, to_log2, bv, bw);
                  tops[j & 3] = max3(tops[j & 3], v, w);
                }
              } else {
                highest(x);
              }
              if (kForm == kCapped)
#pragma unroll
                for (int j = 0; j < 16; ++j) lows[j & 1] = min3(lows[j & 1], __uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
            }
          }
          top = all_tops();
          if (kForm == kCapped) {
            direct = __all_sync(0xffffffffu, !mine || fmaxf(fabsf(top), fabsf(fminf(lows[0], lows[1]))) * cap.per_cap <= 0.4f);
            top = cap.small(top);
          } else if (kForm == kPlain) {
            top *= to_log2;
          }
        }
        if (!direct) {
          // Scores that a cap, a bias or a mask changes go back to tensor memory.  Columns [0, prefix) and [first, end) are seen.
          int prefix = at >= 0 ? range.pre - from : 0, end = at >= 0 ? at - from + 1 : 0;
          int first = at - from >= window ? at - from - window + 1 : 0;
          float distance = (float)(at - from);
#pragma unroll
          for (int i = 0; i < 4; ++i) tops[i] = -INFINITY;
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            uint32_t(&x)[32] = raw[0];
            tmem_ld_32x32b_x32(s_at + 32 * i, x);
            tmem_ld_wait();
            if (kForm == kCapped || (kForm == kGeneral && a.cap > 0.f)) {
              if (!kWide) {
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(cap.any(__uint_as_float(x[j])));
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(a.capped.of(__uint_as_float(x[j])));
              }
            } else if (kForm != kPlain) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * to_log2);
            }
            if (kForm == kSloped || (kForm == kGeneral && a.slopes)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(fmaf(-slope, fabsf(distance - (float)j), __uint_as_float(x[j])));
              distance -= 32.f;
            }
            if (!whole) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(j < prefix || (j >= first && j < end))) x[j] = 0xff800000u;
            }
            prefix -= 32;
            first -= 32;
            end -= 32;
            tmem_st_32x32b_x32(s_at + 32 * i, x);
            highest(x);
          }
          tmem_st_wait();
          top = all_tops() * (kForm == kPlain ? to_log2 : 1.f);
        }
        tmem_ld_32x32b_x32(s_at, raw[0]);
        // A score that is no number, or infinite, makes the row NaN.  (Not by itself: the polynomial takes it for a small one.)
        if (!(top < INFINITY)) {
          m = INFINITY;
          l[0] = NAN;
        }
        // (A row of the tile that is nobody's holds whatever the shared memory held: it must not send the others through the longer ways.)
        const bool above = mine && top > m + kSlack;
        if (__any_sync(0xffffffffu, above)) {
          const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : exp2_approx(m - to);
          m = to;
#pragma unroll
          for (int i = 0; i < 4; ++i) l[i] *= f;
          if (begun) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(o_at + 16 * i, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_32x32b_x16(o_at + 16 * i, o);
            }
          }
        }
        begun = true;
        const float minus = m == -INFINITY ? 0.f : -m;
        // (weights 32 i .. go over scores 16 i .., which have been read; unrolled further, the sums wait for the end in registers)
        auto weights = [&](auto changed) {
          const float scale_log2 = kForm == kPlain || (kForm == kSloped && !changed) ? to_log2 : 1.f;
#pragma unroll 1
          for (int i = 0; i < 4; i += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t(&x)[32] = raw[h];
              tmem_ld_wait();
              if (i + h < 3) tmem_ld_32x32b_x32(s_at + 32 * (i + h + 1), raw[h ^ 1]);
              const float at_i = fmaf(slope, (float)(32 * (i + h)), bias + minus);
              uint32_t packed[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float v = __uint_as_float(x[2 * j]), w = __uint_as_float(x[2 * j + 1]);
                if (kForm == kSloped && !changed) {
                  float bv, bw;
                  fma2(bv, bw, (float)(2 * j), (float)(2 * j + 1), slope, slope, at_i, at_i);
                  fma2(v, w, v, w, scale_log2, scale_log2, bv, bw);
                } else if (kForm == kCapped && !changed) {
                  cap.small(v, w, minus);
                } else if (kForm == kPlain) {
                  fma2(v, w, v, w, scale_log2, scale_log2, minus, minus);
                } else {
                  add2(v, w, minus, minus);
                }
                if ((j & 7) < kPolyOfEight) {
                  exp2_poly(v, w);
                } else {
                  v = exp2_approx(v);
                  w = exp2_approx(w);
                }
                add2(l[2 * (j & 1)], l[2 * (j & 1) + 1], v, w);
                packed[j] = pack2(M(), v, w);
              }
              tmem_st_32x32b_x16(s_at + 16 * (i + h), packed);
            }
            if constexpr (kBytes) {
              if (__builtin_expect(lacks.y != 0, 0)) {   // weights of values whose tile holds more
                tmem_st_wait();
                smaller_weights(s_at + 16 * i, lacks.y >> 8 * i);
              }
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_ready[t][i >> 1]);
          }
        };
        if (kForm == kPlain || direct) weights(std::false_type());
        else weights(std::true_type());
      }
      if (!ok) break;
      blocks += u1 - u0;
      // ---- the tile's result -------------------------------------------------------------------------------------------------
      const float sum = m == -INFINITY ? 0.f : (l[0] + l[1]) + (l[2] + l[3]);   // (a row that saw nothing: 2^-126 of every key)
      const bool any = w.last[t] >= 0;
      if (any) {
        if (!wait(&sm.o_full[t], phases >> 1 & 1, abort_flag, 13)) break;
        phases ^= 2;
        tc_fence_after_sync();
      }
      if (w.chunks == 1) {
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        T* out = static_cast<T*>(a.out) + ((int64_t)(w.first + token) * a.heads + head) * D;
        const bool some = any && sum != 0.f;
        uint32_t o[2][16];
        if (any) tmem_ld_32x32b_x16(o_at, o[0]);
#pragma unroll 1
        for (int i = 0; i < D / 16; i += 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (any) {
              tmem_ld_wait();
              if (i + h + 1 < D / 16) tmem_ld_32x32b_x16(o_at + 16 * (i + h + 1), o[h ^ 1]);
            }
            if (mine) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                o[h][j] = some ? pack2(T(), __uint_as_float(o[h][2 * j]) * inv, __uint_as_float(o[h][2 * j + 1]) * inv) : 0u;
              uint4* to = reinterpret_cast<uint4*>(out) + 2 * (i + h);
              if (p.wide_out) {                  // (whole sectors: every lane has another row)
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(o[h][0]), "r"(o[h][1]), "r"(o[h][2]), "r"(o[h][3]),
                             "r"(o[h][4]), "r"(o[h][5]), "r"(o[h][6]), "r"(o[h][7])
                             : "memory");
              } else {
                to[0] = make_uint4(o[h][0], o[h][1], o[h][2], o[h][3]);
                to[1] = make_uint4(o[h][4], o[h][5], o[h][6], o[h][7]);
              }
            }
          }
        }
      } else {
        // 16 bytes of all rows lie together, so a warp's store and load is one piece
        const int64_t tile = ((int64_t)w.part * 2 + t) * kRows;
        reinterpret_cast<float2*>(a.partial_ml)[tile + r] = make_float2(m, sum);
        uint4* to = reinterpret_cast<uint4*>(a.partial + tile * D) + r;
#pragma unroll 1
        for (int i = 0; i < D / 16; ++i) {
          uint32_t o[16];
          if (any) {
            tmem_ld_32x32b_x16(o_at + 16 * i, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            to[(4 * i + j) * kRows] = any && sum != 0.f ? make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]) : make_uint4(0, 0, 0, 0);
        }
      }
      if (any) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty[t]);
      }
      if (w.chunks == 1) continue;
      // ---- a tile that was cut: the CTA that comes last adds up, in the order of the chunks -------------------------------------
      __threadfence();
      if (!tile_barrier()) break;
      if (r == 0) {
        // A counter holds a launch's number above its parts that have arrived: what an earlier launch left, whole or half counted because a
        // wait ran out, gives way.  (The first one's result is not waited for.)
        unsigned long long* counter = p.counters + w.cut_tile + t;
        const unsigned long long none = (unsigned long long)sm.epoch << 32;
        atomicMax(counter, none);
        sm.last_here[t] = atomicAdd(counter, 1ull) - none == (unsigned long long)(w.chunks - 1);
      }
      if (!tile_barrier()) break;
      const bool last = sm.last_here[t] != 0;
      if (!tile_barrier()) break;
      if (!last) continue;
      __threadfence();
      if (!mine) continue;                       // (work_done brings the warp together again)
      const int64_t tile = (((int64_t)w.part - (int64_t)w.chunk * w.part_step) * 2 + t) * kRows, step = (int64_t)w.part_step * 2 * kRows;
      float2* ml = reinterpret_cast<float2*>(a.partial_ml) + tile + r;
      float M = -INFINITY, L = 0.f;
#pragma unroll 4
      for (int k = 0; k < w.chunks; ++k) M = fmaxf(M, __ldcg(&ml[k * step].x));
#pragma unroll 4
      for (int k = 0; k < w.chunks; ++k) {         // the maximum's place takes the part's weight
        const float2 of = __ldcg(&ml[k * step]);
        const float f = of.x == -INFINITY ? 0.f : exp2_approx(of.x - M);
        L += of.y * f;
        __stcg(&ml[k * step].x, f);
      }
      const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
      T* out = static_cast<T*>(a.out) + ((int64_t)(w.first + token) * a.heads + head) * D;
      const float4* from = reinterpret_cast<const float4*>(a.partial + tile * D) + r;
      constexpr int kAtOnce = 8;
#pragma unroll 1
      for (int q = 0; q < D / 4; q += kAtOnce) {
        float v[4 * kAtOnce];
#pragma unroll
        for (int j = 0; j < 4 * kAtOnce; ++j) v[j] = 0.f;
#pragma unroll 2
        for (int k = 0; k < w.chunks; ++k) {
          const float f = __ldcg(&ml[k * step].x);
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) {
            const float4 o = __ldcg(from + k * step * (D / 4) + (q + j) * kRows);
            v[4 * j] += o.x * f; v[4 * j + 1] += o.y * f; v[4 * j + 2] += o.z * f; v[4 * j + 3] += o.w * f;
          }
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; j += 2) {
          uint32_t x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = pack2(T(), v[4 * j + 2 * i] * inv, v[4 * j + 2 * i + 1] * inv);
          reinterpret_cast<uint4*>(out)[(q + j) / 2] = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
    }
  }

  if (*abort_flag) {
    // loads and products may still be under way into this CTA's memory: let them land before it is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

#ifdef B200_PAGED_BYTES
int launch_paged8_prompt(const char* who, const B200PagedCache* c, PagedAttnParams a, cudaStream_t stream) {
#else
int launch_paged_prompt(const char* who, const B200PagedCache* c, PagedAttnParams a, cudaStream_t stream) {
#endif
  PromptParams p;
  p.tile_tokens = kRows / a.group;
  const uint32_t page = (uint32_t)c->page_size, group = (uint32_t)a.group;
  const CUtensorMapDataType type = c->dtype == B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t D = (uint64_t)c->head_dim;
  int rc;
  {
    const uint64_t d[3] = {D, (uint64_t)a.heads, (uint64_t)c->tokens};
    const uint64_t s[2] = {D * 2, (uint64_t)a.q_stride * 2};
    const uint32_t b[3] = {64, group, (uint32_t)p.tile_tokens};
    if ((rc = make_tmap(&p.tm_q, type, 3, a.q, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
  }
  for (int v = 0; v < 2; ++v) {
    const uint64_t d[4] = {D, page, (uint64_t)c->kv_heads, (uint64_t)c->pages};
    constexpr uint64_t kSize = kBytes ? 1 : 2;
    const uint64_t s[3] = {D * kSize, (uint64_t)page * D * kSize, (uint64_t)(v ? c->v_page_stride : c->k_page_stride) * kSize};
    const uint32_t b[4] = {kBytes ? (uint32_t)D : 64u, page, 1, 1};
    if ((rc = make_tmap(v ? &p.tm_v : &p.tm_k, kBytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type, 4, v ? c->v_pages : c->k_pages, d, s, b,
                        kBytes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
  }
  a.slots = sm_count();
  p.wide_out = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0;
  p.per_pair = ((1ull << 40) + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
  p.counters = reinterpret_cast<unsigned long long*>(a.arrived + kFewCounters);
  p.words = reinterpret_cast<PromptWords*>(p.counters + kCutTiles);
  p.a = a;
  // pairs of tiles of all sequences, at most, and their chunks
  const int64_t pairs = (c->tokens + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens) + c->batch;
  const int64_t most = pairs * c->kv_heads + (int64_t)kPartsOfSlots * a.slots;
  if (kPartsOfSlots * a.slots > kCutTiles) return fail(B200_EINVAL, "%s: more than %d multiprocessors", who, kCutTiles / kPartsOfSlots);
  if (most > 0x3fffffffLL || pairs >= 1 << 24) return fail(B200_EINVAL, "%s: too many rows", who);
  auto launch = [&](auto kern, size_t bytes, SmemLimit& limit, std::atomic<int>& regs) {
    const size_t smem = bytes + 1024;
    int e = raise_smem_limit(limit, reinterpret_cast<const void*>(kern), smem, who);
    if (e) return e;
    // the register split asks for what the launch has: a kernel that was built with fewer would wait for ever
    if (regs.load(std::memory_order_relaxed) == 0) {
      cudaFuncAttributes attr;
      if (cudaFuncGetAttributes(&attr, kern) != cudaSuccess) return fail(B200_ELAUNCH, "%s: cudaFuncGetAttributes", who);
      regs.store(attr.numRegs, std::memory_order_relaxed);
    }
    if (regs.load(std::memory_order_relaxed) < kLaunchRegs)
      return fail(B200_ELAUNCH, "%s: built with %d registers a thread, %d are needed", who, regs.load(), kLaunchRegs);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.slots);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = options().gemv_pdl ? 1 : 0;
    const cudaError_t r = cudaLaunchKernelEx(&cfg, kern, p);
    if (r != cudaSuccess) return fail(B200_ELAUNCH, "%s launch: %s", who, cudaGetErrorString(r));
    count_launch();
    return B200_OK;
  };
  const int form = !(a.scale > 0.f) || (a.cap > 0.f && a.slopes) ? kGeneral : a.cap > 0.f ? kCapped : a.slopes ? kSloped : kPlain;
  const bool wide = a.cap > 0.f && a.capped.wide();
  auto by_form = [&](auto type_, auto dim) {
    using T = decltype(type_);
    constexpr int N = decltype(dim)::value;
    static SmemLimit limit[6];
    static std::atomic<int> regs[6];
    const int at = form + (wide ? form == kCapped ? 3 : 2 : 0);
    auto kern = form == kPlain ? paged_prompt_kernel<T, N, kPlain, false>
              : form == kSloped ? paged_prompt_kernel<T, N, kSloped, false>
              : form == kCapped ? wide ? paged_prompt_kernel<T, N, kCapped, true> : paged_prompt_kernel<T, N, kCapped, false>
                                : wide ? paged_prompt_kernel<T, N, kGeneral, true> : paged_prompt_kernel<T, N, kGeneral, false>;
    return launch(kern, sizeof(Smem<N>), limit[at], regs[at]);
  };
  auto by_dim = [&](auto type_) {
    return c->head_dim == 128 ? by_form(type_, std::integral_constant<int, 128>()) : by_form(type_, std::integral_constant<int, 64>());
  };
  return c->dtype == B200_F16 ? by_dim(__half()) : by_dim(__nv_bfloat16());
}

#ifdef B200_PAGED_BYTES
int paged8_prompt_error_read_and_clear() {
#else
int paged_prompt_error_read_and_clear() {
#endif
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_prompt_error, sizeof(int)) != cudaSuccess) return 0xff;
  if (v) cudaMemcpyToSymbol(g_prompt_error, &zero, sizeof(int));
  return v;
}

}  // namespace b200
