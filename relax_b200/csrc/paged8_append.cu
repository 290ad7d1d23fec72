// Rotary positions for q and k, and the append of k and v to pages of 8 bits (e4m3) with a scale for 16 tokens of a head.
//
// k and v are first what the 16-bit cache would hold (fp32, rounded to the rows' type).  The scale of a block of 16 tokens is a power of two,
// the smallest by which the call's tokens fit, and never smaller than what earlier tokens of the block have.  Where it grows, their
// codes are scaled anew: powers of two change a code's exponent only, so that nothing is rounded twice but what falls below the
// format's smallest step.
//
// A thread block takes one token: its query heads, and a share of the keys and values of the 16 tokens that it lies in.  A task is a key head's
// keys or its values; the thread blocks of the call's n tokens there deal the tasks out among themselves, so that each has as many (token, task)
// pairs as a token has keys and values, whatever n is.  No other thread block touches a task's codes or its scale.
// A thread has two chunks of 8 values of a pair, those that are turned together, as it has of the queries; the largest value of a task comes
// together in shared memory.
//
// What bounds it: HBM for prompts, latency for single tokens (64 of them 5.0 us a call).  us for 8.4k tokens of 32 heads and 8 key heads, 190 MB: 40.3
// (4.8 TB/s, 0.73 of a copy) with eight blocks an SM, 42.6 with six, 51.8 with the four that fit without a limit on registers.  Before: a warp for all
// tokens of a task 164; a warp for a (token, task) pair, 4 values a lane, 68 (5000 instructions a token instead of 3100).
#include <type_traits>

#include "paged_common.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 128;
constexpr int kEarly = 2;                       // of the queries' chunk pairs that are asked for before it is known where the token lies
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
// Two values' codes, to nearest even, at most 448 in size; NaN for what is no number.
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 values2(uint32_t codes) { return unpack2(__half(), e4m3_to_half2(codes)); }

// 8 neighbouring numbers of a table.
__device__ __forceinline__ void load8_floats(const float* p, float (&to)[8]) {
  const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
  to[0] = u.x; to[1] = u.y; to[2] = u.z; to[3] = u.w;
  to[4] = v.x; to[5] = v.y; to[6] = v.z; to[7] = v.w;
}

// The table row of a token at `position`, row `row` of the call.
__device__ __forceinline__ int64_t table_row(const AppendParams& p, int row, int position) {
  const int64_t at = p.positions ? p.positions[row] : position;
  return at < 0 ? 0 : at >= p.table_rows ? p.table_rows - 1 : at;
}

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 8)
paged8_append_kernel(const AppendParams p) {
  constexpr int kChunks = D / 16;               // chunk pairs of a row of D values
  constexpr int kPairs = kThreads / kChunks;    // (token, task) pairs at a time
  constexpr uint32_t kInfinite = std::is_same<T, __half>::value ? 0x7c00 : 0x7f80;
  __shared__ int sm_most[3][kPairs];            // largest values of the tasks at hand; the next round's are cleared a barrier before
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int kv = p.c.kv_heads, page = 1 << p.c.page_log2;
  const int row = blockIdx.x, c = threadIdx.x % kChunks;
  const int half = p.rotary / 2;
  const bool turns = 16 * c < p.rotary;         // this thread's chunk pairs, of queries and keys
  const int o0 = !kInterleaved && turns ? 8 * c : 16 * c, o1 = !kInterleaved && turns ? half + o0 : o0 + 8;
  const T* in = static_cast<const T*>(p.qkv) + (int64_t)row * p.qkv_stride;
  T* q = static_cast<T*>(p.q_out) + (int64_t)row * p.heads * D;
  auto chunk = [](const T* from) { return *reinterpret_cast<const uint4*>(from); };
  uint4 qx[kEarly], qy[kEarly];
  int head = threadIdx.x / kChunks;
#pragma unroll
  for (int k = 0; k < kEarly; ++k)
    if (head + k * kPairs < p.heads) {
      qx[k] = chunk(in + (head + k * kPairs) * D + o0);
      qy[k] = chunk(in + (head + k * kPairs) * D + o1);
    }
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
  // a chunk pair turned by the angles of table row `at`
  auto turn = [&](uint4& x, uint4& y, int64_t at) {
    float cs[8], sn[8];
    load8_floats(p.cos_t + at * half + 8 * c, cs);
    load8_floats(p.sin_t + at * half + 8 * c, sn);
    uint32_t* xo = &x.x;
    uint32_t* yo = &y.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 u = unpack2(T(), xo[j]), w = unpack2(T(), yo[j]);
      if (kInterleaved) {                       // a word is a pair: x holds pairs 0..3 of the eight, y 4..7
        xo[j] = pack2(T(), u.x * cs[j] - u.y * sn[j], u.y * cs[j] + u.x * sn[j]);
        yo[j] = pack2(T(), w.x * cs[4 + j] - w.y * sn[4 + j], w.y * cs[4 + j] + w.x * sn[4 + j]);
      } else {
        xo[j] = pack2(T(), u.x * cs[2 * j] - w.x * sn[2 * j], u.y * cs[2 * j + 1] - w.y * sn[2 * j + 1]);
        yo[j] = pack2(T(), w.x * cs[2 * j] + u.x * sn[2 * j], w.y * cs[2 * j + 1] + u.y * sn[2 * j + 1]);
      }
    }
  };
  const int64_t mine = table_row(p, row, position);
  auto put_query = [&](int h, uint4 x, uint4 y) {
    if (turns) turn(x, y, mine);
    *reinterpret_cast<uint4*>(q + h * D + o0) = x;
    *reinterpret_cast<uint4*>(q + h * D + o1) = y;
  };
  auto put_queries = [&]() {
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
      if (head + k * kPairs < p.heads) put_query(head + k * kPairs, qx[k], qy[k]);
#pragma unroll 1
    for (head += kEarly * kPairs; head < p.heads; head += kPairs) put_query(head, chunk(in + head * D + o0), chunk(in + head * D + o1));
  };

  // ---- keys and values of the block of 16 tokens that this one lies in: tokens [first, first + n) are the call's ------------------
  const int begin = position & ~(kTokens - 1), first = max(begin, max(base, 0)), n = min(begin + kTokens, s.length) - first;
  const int64_t id = page_of(p.c, b, position >> p.c.page_log2);
  const int offset = begin & (page - 1), first_row = s.first + first - base, earlier = first - begin;
  const int inverse = (65536 + n - 1) / n;      // (of numbers below 64 by n)
  const int per_round = kPairs * inverse >> 16; // tasks at a time
  const int slot = (threadIdx.x / kChunks) * inverse >> 16, r = threadIdx.x / kChunks - slot * n;
  const T* from = static_cast<const T*>(p.qkv) + (int64_t)(first_row + r) * p.qkv_stride + p.heads * D;
  if (threadIdx.x < kPairs) sm_most[0][threadIdx.x] = 0;
  __syncthreads();
  int round = 0;
  bool queries = true;
#pragma unroll 1
  for (int done = 0; position - first + n * done < 2 * kv; done += per_round) {
    const int next = round == 2 ? 0 : round + 1;
    if (threadIdx.x < kPairs) sm_most[next][threadIdx.x] = 0;
    const int task = position - first + n * (done + slot);
    const bool some = slot < per_round && task < 2 * kv, is_v = task >= kv;
    const int h = is_v ? task - kv : task;
    __half* scale = (is_v ? p.v_scales : p.k_scales) + ((id * kv + h) * page + offset) / kTokens;
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    float was = 0.f;
    if (some) {
      x = chunk(from + task * D + o0);
      y = chunk(from + task * D + o1);
      if (earlier) was = __half2float(*scale);
    }
    if (queries) put_queries();                 // (the loads above are on their way)
    queries = false;
    uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    if (some) {
      if (turns && !is_v) {
        turn(x, y, table_row(p, first_row + r, first + r));
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
      }
      // sizes are in the order of their bits; what is no finite number does not count
      uint32_t most = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = __vmaxu2(most, w[e] & 0x7fff7fffu);
      most = max(most & 0xffffu, most >> 16);
      if (most >= kInfinite) {
        most = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t v = (e & 1 ? w[e / 2] >> 16 : w[e / 2]) & 0x7fffu;
          if (v < kInfinite) most = max(most, v);
        }
      }
      atomicMax(&sm_most[round][slot], (int)most);
    }
    __syncthreads();
    if (some) {
      unsigned char* codes = static_cast<unsigned char*>(is_v ? p.c.v : p.c.k) + id * (is_v ? p.c.v_stride : p.c.k_stride) + ((int64_t)h * page + offset) * D;
      const float most = unpack2(T(), (uint32_t)sm_most[round][slot]).x;
      const float now = fmaxf(was, power_of_two(power_for(most))), per = 1.f / now;
      if (r == 0) {                             // the task's scale, and the earlier tokens' codes by it
        if (was < now && earlier) {
          const float ratio = was * per;
          auto again = [&](uint32_t codes4) {
            const float2 u = values2(codes4 & 0xffffu), v = values2(codes4 >> 16);
            return codes2(u.x * ratio, u.y * ratio) | codes2(v.x * ratio, v.y * ratio) << 16;
          };
#pragma unroll 5
          for (int t = 0; t < earlier; ++t) {
            uint4* old = reinterpret_cast<uint4*>(codes + t * D) + c;
            const uint4 v = *old;
            *old = make_uint4(again(v.x), again(v.y), again(v.z), again(v.w));
          }
        }
        if (c == 0) *scale = __float2half_rn(now);
      }
      uint32_t out[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float2 v = unpack2(T(), w[e]);
        if ((w[e] & 0x7fffu) == kInfinite) v.x = NAN;                     // (a NaN's code is one anyway)
        if ((w[e] >> 16 & 0x7fffu) == kInfinite) v.y = NAN;
        const uint32_t two = codes2(v.x * per, v.y * per);
        out[e / 2] = e & 1 ? out[e / 2] | two << 16 : two;
      }
      unsigned char* to = codes + (earlier + r) * D;
      *reinterpret_cast<uint2*>(to + o0) = make_uint2(out[0], out[1]);
      *reinterpret_cast<uint2*>(to + o1) = make_uint2(out[2], out[3]);
    }
    round = next;
  }
  if (queries) put_queries();                   // (more tokens than tasks: this one has none)
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
