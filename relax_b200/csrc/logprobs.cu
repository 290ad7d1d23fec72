// What the logits of a row say: log probability of a given token, entropy of the distribution, the likeliest entries.
//
// One pass over the row: with w_i = 2^t_i, t_i = (x_i - m) log2 e and m the running maximum of a thread, a thread keeps
// L = sum w and E = sum w t; a new maximum shifts all t by d: L' = L 2^d, E' = (E + d L) 2^d.  Then log p_i = (x_i - m) - ln L and
// the entropy is ln L - ln 2 E / L, neither of which suffers from a common offset of the logits.
//
// The likeliest k without a second pass over everything: the maxima of groups of four threads bound the k-th largest value from below
// (k of the groups have an element at or above the k-th largest group maximum), and only threads whose own maximum reaches that
// bound saw anything that counts: their parts, which are in cache, are looked through again by all.  What is found, a few more than k, is put
// in order by counting.
// Equal values go by index; where more elements equal the bound than the list holds, their lowest indices are found by a scan in order.
//
// A row is one CTA of 256 threads; few rows are spread over a cluster of up to 8, joined through shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kCtasPerSm = 5;
constexpr int kMaxTop = 32, kMaxCluster = 8;
constexpr int kGroups = 64;                     // of four neighbouring threads
constexpr int kList = 512;                      // elements above the bound, elements equal to it
constexpr float kLn2 = 0.6931471805599453f;
using ptx::exp2_approx;
using ptx::kLog2e;

struct LogprobParams {
  const void* logits;
  const int* tokens;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int* top_token;
  int64_t stride, rows;
  int V, top;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[Vec<T>::N]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// Values in the order of unsigned numbers; both zeros are one value.  0: smaller than every value (-inf is 0x007fffff).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kKeyNegInf = 0x007fffffu;

struct Stats {
  float m, l, e;                                // m = -inf: nothing but excluded entries
  __device__ __forceinline__ void raise(float to) {
    if (!(to > m)) return;
    const float d = fmaxf((m - to) * kLog2e, -1000.f), f = exp2_approx(d);     // (from -inf: l = e = 0)
    e = (e + d * l) * f;
    l *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {        // x <= m, m > -inf
    const float t = (x - m) * kLog2e, w = exp2_approx(t);
    l += w;
    e = fmaf(w, fmaxf(t, -1000.f), e);          // (an excluded entry is 0 * -1000, a NaN stays in w)
  }
  __device__ __forceinline__ void join(Stats o) {
    if (o.m == -INFINITY && o.l == 0.f) return;
    const float to = fmaxf(m, o.m);
    raise(to);
    o.raise(to);
    l += o.l;
    e += o.e;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
token_logprobs_kernel(const LogprobParams p) {
  constexpr int N = Vec<T>::N;
  constexpr int U = 4;                          // loads in flight
  __shared__ Stats sm_stats[kWarps];
  __shared__ __align__(16) uint32_t sm_group[kGroups];
  __shared__ uint32_t sm_bound;
  __shared__ int sm_above, sm_equal, sm_count, sm_hots;
  __shared__ uint8_t sm_hot[kThreads];
  __shared__ unsigned long long sm_list[kList];         // key << 32 | ~index
  __shared__ int sm_equal_at[kList];
  __shared__ unsigned long long sm_best[kMaxTop];       // this CTA's, in order
  __shared__ Stats in_stats[kMaxCluster];               // of the cluster, in CTA 0
  __shared__ int in_count[kMaxCluster];                 // how many of its likeliest a CTA has
  __shared__ unsigned long long in_best[kMaxCluster * kMaxTop];
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int c = gridDim.x, rank = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= p.rows) return;                            // (whole clusters)
  if (c > 1) ptx::cluster_arrive_relaxed();             // (every CTA of the cluster runs before anything is stored in it)
  const T* x = static_cast<const T*>(p.logits) + row * p.stride;
  // this CTA's slice, cut at 16-byte boundaries: [head, body of whole vectors, tail]
  const int per = (((p.V + c - 1) / c) + N - 1) / N * N;
  const int lead = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));   // elements in front of the first boundary
  int begin = rank * per + (rank ? lead : 0), end = min((rank + 1) * per + lead, p.V);
  if (rank == c - 1) end = p.V;
  begin = min(begin, p.V);
  const int body = min(rank ? begin : lead, end), vecs = max(end - body, 0) / N, tail = body + vecs * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + body);

  Stats s = {-INFINITY, 0.f, 0.f};
  auto one = [&](float v) {
    s.raise(v);
    if (s.m > -INFINITY || v != v) s.add(v);
  };
  // Several vectors at a time: one maximum.  Where it is not near the type's lowest value, entries below kFloor, excluded ones among them,
  // count as kFloor: weight 0, and 0 times a number instead of 0 times infinity.  Then four operations an entry beside the special
  // function, two entries an instruction.
  constexpr float kFloor = std::is_same<T, __half>::value ? -65504.f : -1e30f, kFar = std::is_same<T, __half>::value ? -65000.f : -1e29f;
  // (Where it is near the type's largest value, the distance to others in the exponent of 2 leaves fp32: that goes entry by entry too.)
  auto amid = [](float m) { return m > kFar && (std::is_same<T, __half>::value || m < 2e38f); };
  auto many = [&](auto& v) {                            // uint4 [n]
    constexpr int n = sizeof(v) / sizeof(uint4);
    float top;
    if constexpr (sizeof(T) == 2) {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      T2* w = reinterpret_cast<T2*>(v);
      T2 most[4] = {w[0], w[1], w[2], w[3]};
#pragma unroll
      for (int i = 4; i < 4 * n; ++i) most[i & 3] = __hmax2(most[i & 3], w[i]);
      const T2 all = __hmax2(__hmax2(most[0], most[1]), __hmax2(most[2], most[3]));
      top = fmaxf(to_float(T(all.x)), to_float(T(all.y)));
      s.raise(top);
      if (amid(s.m)) {
        const T lowest = T(kFloor);
        const T2 lowest2 = T2(lowest, lowest);
#pragma unroll
        for (int i = 0; i < 4 * n; ++i) w[i] = __hmax2_nan(w[i], lowest2);
      }
    } else {
      float* w = reinterpret_cast<float*>(v);
      float most[4] = {w[0], w[1], w[2], w[3]};
#pragma unroll
      for (int i = 4; i < 4 * n; ++i) most[i & 3] = fmaxf(most[i & 3], w[i]);
      top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
      s.raise(top);
      if (amid(s.m)) {
#pragma unroll
        for (int i = 0; i < 4 * n; ++i) w[i] = w[i] < kFloor ? kFloor : w[i];   // (a NaN stays)
      }
    }
    if (amid(s.m)) {
#pragma unroll
      for (int q = 0; q < n; ++q) {
        float f[N], l0 = 0.f, l1 = 0.f, e0 = 0.f, e1 = 0.f;       // (sums of a few, so that a thread's thousands do not lose bits)
        unpack<T>(v[q], f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          float a = f[i], b = f[i + 1];
          ptx::add2(a, b, -s.m, -s.m);
          ptx::mul2(a, b, kLog2e, kLog2e);
          const float wa = exp2_approx(a), wb = exp2_approx(b);
          ptx::add2(l0, l1, wa, wb);
          ptx::fma2(e0, e1, wa, wb, a, b, e0, e1);
        }
        s.l += l0 + l1;
        s.e += e0 + e1;
      }
      return;
    }
#pragma unroll 1
    for (int q = 0; q < n; ++q) {
      float f[N];
      unpack<T>(v[q], f);
      if (s.m > -INFINITY) {
        Stats part = {s.m, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) part.add(f[i]);
        s.l += part.l;
        s.e += part.e;
      } else {                                          // nothing but excluded entries so far, or NaN
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (f[i] != f[i]) s.l = f[i];
      }
    }
  };
  for (int i = begin + tid; i < body; i += kThreads) one(to_float(x[i]));
  int i = tid;
  for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = __ldg(xv + i + u * kThreads);
    many(v);
  }
  for (; i < vecs; i += kThreads) {
    uint4 v[1] = {__ldg(xv + i)};
    many(v);
  }
  for (int j = tail + tid; j < end; j += kThreads) one(to_float(x[j]));

  // ---- statistics of the CTA ------------------------------------------------------------------------------------------
  const float own = s.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stats other = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.l, o), __shfl_xor_sync(0xffffffffu, s.e, o)};
    s.join(other);
  }
  if (lane == 0) sm_stats[warp] = s;

  // ---- its likeliest entries ----------------------------------------------------------------------------------------------
  const int k = p.top;
  if (k > 0) {
    const uint32_t mine = key_of(own);
    uint32_t gk = mine;
    gk = max(gk, __shfl_xor_sync(0xffffffffu, gk, 1));
    gk = max(gk, __shfl_xor_sync(0xffffffffu, gk, 2));
    if ((lane & 3) == 0) sm_group[tid >> 2] = gk;
    if (tid == 0) sm_above = sm_equal = sm_count = sm_hots = 0;
    if (tid < k) sm_best[tid] = 0;
    __syncthreads();
    if (tid < kGroups) {                                // the k-th largest of the 64 groups, by counting
      const uint32_t key = sm_group[tid];
      int r = 0;
#pragma unroll
      for (int j = 0; j < kGroups; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(sm_group + j);
        r += (o.x > key || (o.x == key && j < tid)) + (o.y > key || (o.y == key && j + 1 < tid)) + (o.z > key || (o.z == key && j + 2 < tid)) +
             (o.w > key || (o.w == key && j + 3 < tid));
      }
      // -inf (an excluded entry, or a group without elements): nothing but real values is collected
      if (r == k - 1) sm_bound = max(key, kKeyNegInf);
    }
    __syncthreads();
    const uint32_t bound = sm_bound;
    auto look = [&](float v, int at) {
      const uint32_t key = key_of(v);
      if (key > bound) {
        const int n = atomicAdd(&sm_above, 1);
        if (n < kList) sm_list[n] = (unsigned long long)key << 32 | (uint32_t)~at;
      } else if (key == bound && bound > kKeyNegInf) {
        const int n = atomicAdd(&sm_equal, 1);
        if (n < kList) sm_equal_at[n] = at;
      }
    };
    // The threads that saw such an element; all of them look through those threads' vectors together.
    const bool hot = mine >= bound;
    if (hot) {
      for (int j = begin + tid; j < body; j += kThreads) look(to_float(x[j]), j);
      for (int j = tail + tid; j < end; j += kThreads) look(to_float(x[j]), j);
      sm_hot[atomicAdd(&sm_hots, 1)] = tid;
    }
    __syncthreads();
    const int rounds = (vecs + kThreads - 1) / kThreads, hots = sm_hots;
    for (int j = tid; j < hots * rounds; j += kThreads) {
      const int who = j / rounds, i = sm_hot[who] + (j - who * rounds) * kThreads;
      if (i >= vecs) continue;
      float f[N];
      unpack<T>(__ldg(xv + i), f);
      float top = f[0];
#pragma unroll
      for (int u = 1; u < N; ++u) top = fmaxf(top, f[u]);
      if (key_of(top) < bound) continue;
#pragma unroll
      for (int u = 0; u < N; ++u) look(f[u], body + i * N + u);
    }
    __syncthreads();
    const int above = sm_above, equal = sm_equal;
    if (above <= kList) {
      // rank among those above the bound: fewer than k groups reach above it, but a group may hold many
      for (int j = tid; j < above; j += kThreads) {
        const unsigned long long v = sm_list[j];
        int r = 0;
        for (int u = 0; u < above; ++u) r += sm_list[u] > v;
        if (r < k) sm_best[r] = v;
      }
      const int want = k - above;                       // of those equal to it, by index
      if (want > 0 && equal > 0) {
        if (equal <= kList) {
          for (int j = tid; j < equal; j += kThreads) {
            const int at = sm_equal_at[j];
            int r = 0;
            for (int u = 0; u < equal; ++u) r += sm_equal_at[u] < at;
            if (r < want) sm_best[above + r] = (unsigned long long)bound << 32 | (uint32_t)~at;
          }
        } else {                                        // in order, 256 at a time, until there are enough
          __shared__ int sm_warp[kWarps];
          for (int from = begin; from < end; from += kThreads) {
            const int at = from + tid;
            const bool hit = at < end && key_of(to_float(x[at])) == bound;
            const unsigned hits = __ballot_sync(0xffffffffu, hit);
            if (lane == 0) sm_warp[warp] = __popc(hits);
            __syncthreads();
            int before = sm_count;
            for (int w = 0; w < warp; ++w) before += sm_warp[w];
            before += __popc(hits & ((1u << lane) - 1));
            if (hit && before < want) sm_best[above + before] = (unsigned long long)bound << 32 | (uint32_t)~at;
            int all = sm_count;
            for (int w = 0; w < kWarps; ++w) all += sm_warp[w];
            __syncthreads();
            if (tid == 0) sm_count = all;
            __syncthreads();
            if (all >= want) break;
          }
        }
      }
    } else {
      // a group holds more than the list does: the largest below the last one found, k times
      __shared__ unsigned long long sm_next[kWarps];
      unsigned long long last = ~0ull;
      for (int j = 0; j < k; ++j) {
        unsigned long long best = 0;
        for (int at = begin + tid; at < end; at += kThreads) {
          const unsigned long long v = (unsigned long long)key_of(to_float(x[at])) << 32 | (uint32_t)~at;
          if (v < last && v > best) best = v;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) sm_next[warp] = best;
        __syncthreads();
        best = 0;
        for (int w = 0; w < kWarps; ++w) best = max(best, sm_next[w]);
        if (tid == 0) sm_best[j] = best;
        last = best;
        __syncthreads();
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    s = lane < kWarps ? sm_stats[lane] : Stats{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      const Stats other = {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.l, o), __shfl_xor_sync(0xffffffffu, s.e, o)};
      s.join(other);
    }
    if (lane == 0) sm_stats[0] = s;
  }
  __syncthreads();

  // ---- the cluster --------------------------------------------------------------------------------------------------------
  if (c > 1) {
    ptx::cluster_wait();                                // (the one at the start)
    if (tid < k) {
      const uint32_t to = ptx::map_to_rank(ptx::smem_u32(&in_best[rank * kMaxTop + tid]), 0);
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(sm_best[tid]) : "memory");
    }
    if (tid == 0) {
      const uint32_t to = ptx::map_to_rank(ptx::smem_u32(&in_stats[rank]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(sm_stats[0].m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(sm_stats[0].l) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(sm_stats[0].e) : "memory");
      int n = 0;
      while (n < k && sm_best[n] != 0) ++n;
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ptx::map_to_rank(ptx::smem_u32(&in_count[rank]), 0)), "r"(n) : "memory");
    }
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (rank != 0) return;
    s = in_stats[0];
    for (int r = 1; r < c; ++r) s.join(in_stats[r]);
    int real = 0;
    for (int o = 0; o < c; ++o) real += in_count[o];
    for (int n = warp; n < c; n += kWarps) {            // a warp has a CTA's list, a lane an entry
      if (lane >= in_count[n]) continue;
      const unsigned long long v = in_best[n * kMaxTop + lane];
      int r = lane;                                     // those before it in its own list, and those above it in the others
      for (int o = 0; o < c; ++o) {
        if (o == n) continue;
        int lo = 0, hi = in_count[o];
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (in_best[o * kMaxTop + mid] > v) lo = mid + 1; else hi = mid;
        }
        r += lo;
      }
      if (r < k) sm_best[r] = v;
    }
    if (tid < k && tid >= real) sm_best[tid] = 0;       // (fewer real values than k)
    __syncthreads();
  } else {
    s = sm_stats[0];
  }
  const float log_l = logf(s.l);
  const bool none = s.m == -INFINITY && s.l == 0.f, bad = !(s.l < INFINITY) || s.m == INFINITY;
  auto log_of = [&](float v) { return bad ? NAN : none ? -INFINITY : (v - s.m) - log_l; };
  if (tid == 0) {
    if (p.logprob) {
      const int at = p.tokens[row];
      p.logprob[row] = bad ? NAN : at < 0 || at >= p.V ? -INFINITY : log_of(to_float(x[at]));
    }
    if (p.entropy) p.entropy[row] = bad ? NAN : none ? 0.f : log_l - kLn2 * s.e / s.l;
  }
  if (tid < k) {
    const unsigned long long v = sm_best[tid];
    float value = value_of((uint32_t)(v >> 32));
    int at = (int)~(uint32_t)v;
    if (bad) {
      at = tid;
    } else if ((v >> 32) <= kKeyNegInf) {
      // excluded entries, by index: all but fewer than k of the first k entries
      value = -INFINITY;
      int real = 0;
      for (int j = 0; j < k; ++j) real += (sm_best[j] >> 32) > kKeyNegInf;
      int want = tid - real;
      at = 0;
      for (int j = 0; j < p.V; ++j)
        if (to_float(x[j]) == -INFINITY && want-- == 0) { at = j; break; }
    }
    p.top_logprob[row * k + tid] = log_of(value);
    p.top_token[row * k + tid] = at;
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_token_logprobs(const void* logits, int32_t dtype, int64_t stride, const void* tokens, void* logprob, void* entropy,
                                   void* top_logprob, void* top_token, int64_t rows, int64_t V, int32_t top, void* stream) {
  const char* who = "token_logprobs";
  if (dtype != B200_F16 && dtype != B200_BF16 && dtype != B200_F32) return fail(B200_EINVAL, "%s: dtype %d is not fp16, bf16 or fp32", who, dtype);
  // (an index runs past the row's end by up to a step of all threads before it is looked at: that has to fit in 31 bits)
  if (rows < 0 || V <= 0 || V >= (1LL << 31) - 4096) return fail(B200_EINVAL, "%s: bad sizes %lld x %lld", who, (long long)rows, (long long)V);
  if (top < 0 || top > kMaxTop || top > V) return fail(B200_EINVAL, "%s: top is at most %d and V, got %d", who, kMaxTop, top);
  if (rows == 0) return B200_OK;
  const unsigned size = dtype == B200_F32 ? 4 : 2;
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & (size - 1))) return fail(B200_EINVAL, "%s: logits must be non-null and aligned to their type", who);
  if (stride < V && rows > 1) return fail(B200_EINVAL, "%s: rows overlap", who);
  if (logprob && !tokens) return fail(B200_EINVAL, "%s: log probabilities need tokens", who);
  if (top > 0 && (!top_logprob || !top_token)) return fail(B200_EINVAL, "%s: null output of the likeliest entries", who);
  if (rows > 0x7fffffffLL) return fail(B200_EINVAL, "%s: too many rows", who);
  int rc = ensure_device();
  if (rc) return rc;
  LogprobParams p = {logits, static_cast<const int*>(tokens), static_cast<float*>(logprob), static_cast<float*>(entropy),
                     static_cast<float*>(top_logprob), static_cast<int*>(top_token), stride, rows, (int)V, top};
  // CTAs of a row: the fewest rounds of CTAs, each as long as its slice of the row and what begins and ends it (about 14000 entries, and
  // 2000 for each CTA of the cluster).  us, fp16, 20 alternatives: one row of 32000 8.9 with four CTAs, 10.1 with eight; 64 rows 9.6 with
  // four, 14.8 with eight.  Threads, CTAs an SM and loads in flight, 2048 rows: 256, 5, 4 42.5 (31.2 without
  // alternatives); 256, 6, 4 42; 256, 4, 4 47; 128, 12, 4 50.
  const int64_t slots = (int64_t)sm_count() * kCtasPerSm;
  int c = 1;
  int64_t least = 0;
  for (int w = 1; w <= kMaxCluster && (w == 1 || V / w >= 2048); w *= 2) {
    const int64_t cost = (rows * w + slots - 1) / slots * (V / w + 14000 + 2000 * w);
    if (w == 1 || cost < least) {
      least = cost;
      c = w;
    }
  }
  auto launch = [&](auto kern) {
    const int64_t y = rows < 32768 ? rows : 32768;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c, (unsigned)y, (unsigned)((rows + y - 1) / y));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = options().gemv_pdl ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(B200_ELAUNCH, "%s launch: %s", who, cudaGetErrorString(e));
    count_launch();
    return B200_OK;
  };
  return dtype == B200_F16 ? launch(token_logprobs_kernel<__half>)
       : dtype == B200_BF16 ? launch(token_logprobs_kernel<__nv_bfloat16>) : launch(token_logprobs_kernel<float>);
}
