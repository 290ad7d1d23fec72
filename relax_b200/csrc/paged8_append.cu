// Rotary positions for q and k, and the append of k and v to pages of 8 bits (e4m3) with a scale for 16 tokens of a head.
//
// k and v are first what the 16-bit cache would hold (fp32, rounded to the rows' type).  The scale of a block of 16 tokens is a power of two,
// the smallest by which the call's tokens fit, and never smaller than what earlier tokens of the block have.  Where it grows, their
// codes are scaled anew: powers of two change a code's exponent only, so that nothing is rounded twice but what falls below the
// format's smallest step.
//
// A block of the call is one for each token: it turns the token's query heads.  The keys and values of a block of 16 tokens are tasks, one
// for each key head and one for its values, dealt out to the thread blocks of its tokens, a warp each: so a prompt's block of 16 tokens has 16 thread
// blocks with a task or two each, and a single token has one with all.  A task's warp holds all its tokens, a lane D / 32 dims of each:
// the largest value is a shuffle away, and no other warp touches the block's codes or its scale.
#include <type_traits>

#include "paged_common.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kTokens = 16;                     // that share a scale
constexpr int kMinPower = -24, kMaxPower = 7;   // of a scale: fp16's smallest number; 448 * 2^7 is the last that fp16 holds

struct AppendParams {
  PagedParams c;
  const void* qkv;
  void* q_out;
  const float* cos_t;
  const float* sin_t;
  const int* positions;
  __half* k_scales;
  __half* v_scales;
  int64_t qkv_stride, table_rows;
  int heads, rotary;
};

// The exponent of the smallest power of two by which values up to `most` fit into e4m3: most = 2^e 1.f, 448 = 2^8 1.75.
__device__ __forceinline__ int power_for(float most) {
  const uint32_t u = __float_as_uint(most);
  const int e = (int)(u >> 23) - 127, power = e - 8 + ((u & 0x7fffffu) > 0x600000u);
  return most > 0.f ? min(max(power, kMinPower), kMaxPower) : kMinPower;
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }
// Two values' codes, to nearest even, at most 448 in size; NaN for what is no number.
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 values2(uint32_t codes) { return unpack2(__half(), e4m3_to_half2(codes)); }

// The words of a lane's share of a token: W 16-bit pairs.
template <int W>
struct Words {
  uint32_t w[W];
};
template <int W>
__device__ __forceinline__ Words<W> load_words(const void* p) {
  Words<W> r;
  if constexpr (W == 2) {
    const uint2 v = *static_cast<const uint2*>(p);
    r.w[0] = v.x;
    r.w[1] = v.y;
  } else {
    r.w[0] = *static_cast<const uint32_t*>(p);
  }
  return r;
}

// The table row of a token at `position`, row `row` of the call.
__device__ __forceinline__ int64_t table_row(const AppendParams& p, int row, int position) {
  const int64_t at = p.positions ? p.positions[row] : position;
  return at < 0 ? 0 : at >= p.table_rows ? p.table_rows - 1 : at;
}

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kThreads)
paged8_append_kernel(const AppendParams p) {
  constexpr int E = D / 32, W = E / 2;          // dims and words of a lane
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int kv = p.c.kv_heads, page = 1 << p.c.page_log2;
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.rotary / 2;
  T* q = static_cast<T*>(p.q_out) + (int64_t)row * p.heads * D;
  // the sequence of this row: the last one that starts at or before it
  int b = row;
  if (p.c.starts) {
    int lo = 0, hi = p.c.batch;                 // starts[lo] <= row < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.c.starts[mid] <= row) lo = mid; else hi = mid;
    }
    b = lo;
  }
  const Sequence s = sequence_of(p.c, b);
  const int place = row - s.first, base = s.length - s.rows, position = base + place;
  if (!(position >= 0 && place >= 0 && place < s.rows)) {
    for (int i = threadIdx.x; i < p.heads * D / 8; i += kThreads) reinterpret_cast<uint4*>(q)[i] = make_uint4(0, 0, 0, 0);
    return;
  }

  // ---- keys and values of the block of 16 tokens that this one lies in: tokens [first, first + n) are the call's ------------------
  const int begin = position & ~(kTokens - 1), first = max(begin, max(base, 0)), n = min(begin + kTokens, s.length) - first;
  const int64_t id = page_of(p.c, b, position >> p.c.page_log2);
  const int offset = begin & (page - 1), first_row = s.first + first - base;
#pragma unroll 1
  for (int task = position - first + n * warp; task < 2 * kv; task += n * kWarps) {
    const bool is_v = task >= kv;
    const int h = is_v ? task - kv : task;
    const T* in = static_cast<const T*>(p.qkv) + (int64_t)first_row * p.qkv_stride + (p.heads + task) * D + E * lane;
    unsigned char* codes = static_cast<unsigned char*>(is_v ? p.c.v : p.c.k) + id * (is_v ? p.c.v_stride : p.c.k_stride) +
                           ((int64_t)h * page + offset) * D + E * lane;
    __half* scale = (is_v ? p.v_scales : p.k_scales) + ((id * kv + h) * page + offset) / kTokens;
    const int earlier = first - begin;
    const float was = earlier ? __half2float(*scale) : 0.f;
    const bool turned = !is_v && E * lane < p.rotary;
    Words<W> x[kTokens];
    float most = 0.f;
    // (four tokens' loads at a time)
#pragma unroll
    for (int r0 = 0; r0 < kTokens; r0 += 4) {
      if (r0 >= n) break;
      Words<W> other[4];
      float cs[4][E], sn[4][E];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (r0 + r >= n) continue;
        const T* from = in + (r0 + r) * p.qkv_stride;
        x[r0 + r] = load_words<W>(from);
        if (turned) {
          const int64_t at = table_row(p, first_row + r0 + r, first + r0 + r) * half;
          const int d = E * lane;
          if (kInterleaved) {                   // pairs (2 i, 2 i + 1): the lane's own
#pragma unroll
            for (int i = 0; i < W; ++i) { cs[r][i] = p.cos_t[at + d / 2 + i]; sn[r][i] = p.sin_t[at + d / 2 + i]; }
          } else {                              // pairs (i, i + half): the other's in another lane
            const bool low = d < half;
            other[r] = load_words<W>(low ? from + half : from - half);
#pragma unroll
            for (int i = 0; i < E; ++i) {
              cs[r][i] = p.cos_t[at + (low ? d : d - half) + i];
              sn[r][i] = p.sin_t[at + (low ? d : d - half) + i];
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (r0 + r >= n) continue;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          uint32_t& w = x[r0 + r].w[i];
          if (turned) {
            const float2 a = unpack2(T(), w);
            if (kInterleaved) {
              w = pack2(T(), a.x * cs[r][i] - a.y * sn[r][i], a.y * cs[r][i] + a.x * sn[r][i]);
            } else {
              const float2 o = unpack2(T(), other[r].w[i]);
              const bool low = E * lane < half;
              const float s0 = low ? -sn[r][2 * i] : sn[r][2 * i], s1 = low ? -sn[r][2 * i + 1] : sn[r][2 * i + 1];
              w = pack2(T(), a.x * cs[r][2 * i] + o.x * s0, a.y * cs[r][2 * i + 1] + o.y * s1);
            }
          }
          const float2 v = unpack2(T(), w);
          // (what is no finite number does not count)
          if (fabsf(v.x) < INFINITY) most = fmaxf(most, fabsf(v.x));
          if (fabsf(v.y) < INFINITY) most = fmaxf(most, fabsf(v.y));
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float need = power_of_two(power_for(most)), now = fmaxf(was, need);
    const float per = 1.f / now;
    if (was < now && earlier) {                 // the earlier tokens' codes by the new scale
      const float ratio = was * per;
#pragma unroll 4
      for (int r = 0; r < earlier; ++r) {
        unsigned char* at = codes + r * D;
        if constexpr (E == 4) {
          const uint32_t c = *reinterpret_cast<const uint32_t*>(at);
          const float2 u = values2(c & 0xffffu), v = values2(c >> 16);
          *reinterpret_cast<uint32_t*>(at) = codes2(u.x * ratio, u.y * ratio) | codes2(v.x * ratio, v.y * ratio) << 16;
        } else {
          const float2 u = values2(*reinterpret_cast<const uint16_t*>(at));
          *reinterpret_cast<uint16_t*>(at) = (uint16_t)codes2(u.x * ratio, u.y * ratio);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kTokens; ++r) {
      if (r >= n) break;
      uint32_t c[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float2 v = unpack2(T(), x[r].w[i]);
        if (!(fabsf(v.x) < INFINITY)) v.x = NAN;
        if (!(fabsf(v.y) < INFINITY)) v.y = NAN;
        c[i] = codes2(v.x * per, v.y * per);
      }
      unsigned char* at = codes + (earlier + r) * D;
      if constexpr (E == 4) *reinterpret_cast<uint32_t*>(at) = c[0] | c[W - 1] << 16;
      else *reinterpret_cast<uint16_t*>(at) = (uint16_t)c[0];
    }
    if (lane == 0) *scale = __float2half_rn(now);
  }

  // ---- the token's queries: pairs of chunks of 8 values, turned or as they are ------------------------------------------------------
  const T* in = static_cast<const T*>(p.qkv) + (int64_t)row * p.qkv_stride;
  const int64_t at = table_row(p, row, position) * half;
  constexpr int kPairs = D / 16;
#pragma unroll 2
  for (int i = threadIdx.x; i < p.heads * kPairs; i += kThreads) {
    const int h = i / kPairs, c = i - h * kPairs;
    const bool turn = 16 * c < p.rotary;
    const int o0 = kInterleaved || !turn ? 16 * c : 8 * c, o1 = kInterleaved || !turn ? o0 + 8 : half + 8 * c;
    const uint4 x = *reinterpret_cast<const uint4*>(in + h * D + o0), y = *reinterpret_cast<const uint4*>(in + h * D + o1);
    uint32_t xo[4] = {x.x, x.y, x.z, x.w}, yo[4] = {y.x, y.y, y.z, y.w};
    if (turn) {
      float cs[8], sn[8];
      const float4* cp = reinterpret_cast<const float4*>(p.cos_t + at + 8 * c);
      const float4* sp = reinterpret_cast<const float4*>(p.sin_t + at + 8 * c);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 u = cp[j], w = sp[j];
        cs[4 * j] = u.x; cs[4 * j + 1] = u.y; cs[4 * j + 2] = u.z; cs[4 * j + 3] = u.w;
        sn[4 * j] = w.x; sn[4 * j + 1] = w.y; sn[4 * j + 2] = w.z; sn[4 * j + 3] = w.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = unpack2(T(), xo[j]), w = unpack2(T(), yo[j]);
        if (kInterleaved) {                     // a word is a pair: x holds pairs 0..3 of the eight, y 4..7
          xo[j] = pack2(T(), u.x * cs[j] - u.y * sn[j], u.y * cs[j] + u.x * sn[j]);
          yo[j] = pack2(T(), w.x * cs[4 + j] - w.y * sn[4 + j], w.y * cs[4 + j] + w.x * sn[4 + j]);
        } else {
          xo[j] = pack2(T(), u.x * cs[2 * j] - w.x * sn[2 * j], u.y * cs[2 * j + 1] - w.y * sn[2 * j + 1]);
          yo[j] = pack2(T(), w.x * cs[2 * j] + u.x * sn[2 * j], w.y * cs[2 * j + 1] + u.y * sn[2 * j + 1]);
        }
      }
    }
    *reinterpret_cast<uint4*>(q + h * D + o0) = make_uint4(xo[0], xo[1], xo[2], xo[3]);
    *reinterpret_cast<uint4*>(q + h * D + o1) = make_uint4(yo[0], yo[1], yo[2], yo[3]);
  }
}

}  // namespace

int paged8_scales(const char* who, const B200PagedCache* c, const B200PagedScales* s) {
  if (!s) return fail(B200_EINVAL, "%s: null descriptor of the scales", who);
  if (c->tokens == 0 || c->batch == 0) return B200_OK;
  if (!s->k_scales || !s->v_scales || (reinterpret_cast<uintptr_t>(s->k_scales) & 1u) || (reinterpret_cast<uintptr_t>(s->v_scales) & 1u))
    return fail(B200_EINVAL, "%s: the scales must be non-null and aligned to their type", who);
  if (c->k_page_stride % 16 || c->v_page_stride % 16) return fail(B200_EINVAL, "%s: page strides of 8-bit pages are multiples of 16", who);
  return B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_paged8_rope_append(const B200PagedCache* cache, const B200PagedScales* scales, const void* qkv, int64_t qkv_stride,
                                       int32_t heads, const void* cos_t, const void* sin_t, int64_t table_rows, int32_t rotary,
                                       int32_t interleaved, const void* positions, void* q_out, void* stream) {
  const char* who = "paged8_rope_append";
  AppendParams p = {};
  int rc = paged_params(who, cache, &p.c);
  if (rc) return rc;
  if ((rc = paged8_scales(who, cache, scales))) return rc;
  if (heads <= 0 || heads > 65536) return fail(B200_EINVAL, "%s: heads in 1..65536, got %d", who, heads);
  if (rotary <= 0 || rotary % 16 || rotary > cache->head_dim)
    return fail(B200_EINVAL, "%s: rotary is a multiple of 16 up to head_dim, got %d", who, rotary);
  if (cache->tokens == 0) return B200_OK;
  if (cache->batch == 0) return fail(B200_EINVAL, "%s: rows without sequences", who);
  if (table_rows <= 0) return fail(B200_EINVAL, "%s: empty tables", who);
  if (qkv_stride < (int64_t)(heads + 2 * cache->kv_heads) * cache->head_dim || qkv_stride % 8)
    return fail(B200_EINVAL, "%s: qkv_stride is a multiple of 8 and at least a row", who);
  if (!qkv || !q_out || !cos_t || !sin_t || !aligned16(qkv) || !aligned16(q_out) || !aligned16(cos_t) || !aligned16(sin_t))
    return fail(B200_EINVAL, "%s: qkv, q_out and the tables must be non-null and 16-byte aligned", who);
  if ((rc = ensure_device())) return rc;
  p.qkv = qkv;
  p.q_out = q_out;
  p.cos_t = static_cast<const float*>(cos_t);
  p.sin_t = static_cast<const float*>(sin_t);
  p.positions = static_cast<const int*>(positions);
  p.k_scales = static_cast<__half*>(scales->k_scales);
  p.v_scales = static_cast<__half*>(scales->v_scales);
  p.qkv_stride = qkv_stride;
  p.table_rows = table_rows;
  p.heads = heads;
  p.rotary = rotary;
  auto launch = [&](auto kern) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cache->tokens);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = options().gemv_pdl ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(B200_ELAUNCH, "%s launch: %s", who, cudaGetErrorString(e));
    count_launch();
    return B200_OK;
  };
  auto by_layout = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    return interleaved ? launch(paged8_append_kernel<T, D, true>) : launch(paged8_append_kernel<T, D, false>);
  };
  auto by_dim = [&](auto type) {
    return cache->head_dim == 128 ? by_layout(type, std::integral_constant<int, 128>()) : by_layout(type, std::integral_constant<int, 64>());
  };
  return cache->dtype == B200_F16 ? by_dim(__half()) : by_dim(__nv_bfloat16());
}
