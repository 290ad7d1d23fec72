// What the kernels over the paged key-value cache share: the descriptor as a launch gets it, the rows and the visible keys of a sequence.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "sm100_ptx.cuh"

namespace b200 {

struct PagedParams {
  void* k;                     // [pages, kv_heads, page, D]
  void* v;
  int64_t k_stride, v_stride;  // between pages
  const int* table;
  const int* lengths;
  const int* starts;           // may be null: row b is sequence b's only one
  int64_t table_stride, tokens;
  int batch, table_width, pages, kv_heads, page_log2;
};

struct Sequence {
  int first, rows, length;     // rows of this call, tokens in the cache
};

__device__ __forceinline__ Sequence sequence_of(const PagedParams& p, int b) {
  Sequence s;
  s.length = min(max(p.lengths[b], 0), p.table_width << p.page_log2);
  s.first = b;
  s.rows = 1;
  if (p.starts) {
    s.first = min(max(p.starts[b], 0), (int)p.tokens);
    s.rows = max(min(p.starts[b + 1], (int)p.tokens) - s.first, 0);
  }
  return s;
}

__device__ __forceinline__ int page_of(const PagedParams& p, int b, int index) {
  return min(max(p.table[(int64_t)b * p.table_stride + index], 0), p.pages - 1);
}

// Two values of the cache's type in 32 bits.
__device__ __forceinline__ float2 unpack2(__half, uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 unpack2(__nv_bfloat16, uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

using ptx::exp2_approx;
using ptx::kLog2e;

// cap * tanh(scale * x / cap) in the exponent of 2, u = scale * x / cap.
//   small  |u| <= 0.4, where nearly all scores are: a cubic in u^2 through the Chebyshev points of [0, 0.16] is tanh(u) / u to 1.0e-7
//          (Taylor's series needs two terms more)
//   any    two special functions; exact to a few 2^-23 of the cap, not of the score
//   of     each where it holds.  Up to a cap of 128 `any` alone changes a weight by 5e-5 at most, a tenth of its rounding to 16 bits; with
//          a cap of 10^4 it changes weights by 0.004, and far above that it leaves nothing of a score
struct Cap {
  float per_cap, log2_cap, c[4];
  Cap() = default;
  __host__ __device__ Cap(float scale, float cap) : per_cap(cap > 0.f ? scale / cap : 0.f), log2_cap(cap * kLog2e) {
    c[0] = 0.999999901f * log2_cap;
    c[1] = -0.333313563f * log2_cap;
    c[2] = 0.132708743f * log2_cap;
    c[3] = -0.0475493467f * log2_cap;
  }
  bool wide() const { return log2_cap > 128.f * kLog2e; }                       // `any` will not do
  // two of them, less a row's maximum
  __device__ __forceinline__ void small(float& x, float& y, float minus) const {
    ptx::mul2(x, y, per_cap, per_cap);
    float u = x, v = y, pu, pv;
    ptx::mul2(u, v, x, y);
    ptx::fma2(pu, pv, u, v, c[3], c[3], c[2], c[2]);
    ptx::fma2(pu, pv, pu, pv, u, v, c[1], c[1]);
    ptx::fma2(pu, pv, pu, pv, u, v, c[0], c[0]);
    ptx::fma2(x, y, x, y, pu, pv, minus, minus);
  }
  __device__ __forceinline__ float small(float x) const {
    const float u = x * per_cap, v = u * u;
    return u * fmaf(fmaf(fmaf(v, c[3], c[2]), v, c[1]), v, c[0]);
  }
  __device__ __forceinline__ float any(float x) const {
    return log2_cap * (1.f - __fdividef(2.f, exp2_approx(x * (2.f * kLog2e * per_cap)) + 1.f));
  }
  __device__ __forceinline__ float of(float x) const {
    float y;                                    // (both, and one of them: a branch for each score takes more than twice as long)
    asm("{\n.reg .pred p;\nsetp.le.f32 p, %1, 0f3ECCCCCD;\nselp.f32 %0, %2, %3, p;\n}" : "=f"(y) : "f"(fabsf(x * per_cap)), "f"(small(x)), "f"(any(x)));
    return y;
  }
};

// What both attention kernels get.
struct PagedAttnParams {
  PagedParams c;
  const void* q;
  void* out;
  int64_t q_stride;
  int heads, group, causal, window;
  float scale, cap;
  Cap capped;
  const float* slopes;
  const int* prefix;
  float* partial;              // few rows: [part][row][D]; many rows: [part][tile of two][D / 4][row][4]
  float* partial_ml;           // their rows' maxima and sums, in pairs
  const __half* k_scales;      // pages of 8 bits: [pages, kv_heads, page / 16]
  const __half* v_scales;
  int* arrived;                // few rows: [CTA]
  int slots;                   // CTAs that run at once
};
constexpr float kSlack = 8.f;  // how far above the running maximum a score may lie, log2

// Units of kUnit tokens that some row of a tile sees: those below `pre`, then those of [low, high).
template <int kUnit>
struct Range {
  int pre, low, high;          // tokens; low >= 0
  int pre_units, second, units;
  __device__ __forceinline__ void set(const PagedAttnParams& p, const Sequence& s, int b, int first_token, int last_token) {
    const int base = s.length - s.rows;
    pre = p.causal ? (p.prefix ? min(max(p.prefix[b], 0), s.length) : 0) : s.length;
    high = max(min(s.length, base + last_token + 1), 0);
    low = p.window ? max(base + first_token - p.window + 1, 0) : 0;
    if (high == 0) pre = 0;                     // (no row has a position)
    pre_units = (pre + kUnit - 1) / kUnit;
    second = max(pre_units, low / kUnit);
    units = pre_units + max((high + kUnit - 1) / kUnit - second, 0);
  }
  __device__ __forceinline__ int unit(int u) const { return u < pre_units ? u : u - pre_units + second; }
};

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// Scratch memory: counters of the few-rows kernel (32 bits), counters of the many-rows kernel's cut tiles (64 bits) and its words, and partial
// results.  Partial results of the many-rows kernel are 256 rows; of its items at most so many times as there are slots are cut.
constexpr int kFewCounters = 2048, kCutTiles = 1016, kPartsOfSlots = 4;
struct PromptWords {
  int next, through;           // the next item; CTAs that are through: zero between launches
  unsigned epoch;              // launches so far
};
static_assert(kFewCounters * 4 + kCutTiles * 8 + sizeof(PromptWords) <= B200_PAGED_ZEROED_BYTES, "the counters");

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }
// Four e4m3 codes (the low ones first) as fp16 values, which hold them exactly.
__device__ __forceinline__ void e4m3_to_half4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
// Two of them.
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
  return r;
}

// The kernel for many rows (paged_attn_prompt.cu).
int launch_paged_prompt(const char* who, const B200PagedCache* c, PagedAttnParams p, cudaStream_t stream);
int launch_paged8_prompt(const char* who, const B200PagedCache* c, PagedAttnParams p, cudaStream_t stream);    // over pages of 8 bits

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launch parameters of a checked descriptor; `who` names the entry point in messages.
int paged_params(const char* who, const B200PagedCache* c, PagedParams* out);
// The scales of pages of 8 bits, beside a checked descriptor.
int paged8_scales(const char* who, const B200PagedCache* c, const B200PagedScales* s);

}  // namespace b200
