// A token of every row of logits, drawn with a given random number: temperature, top-k, top-p, min-p.
//
// In the order (logit downwards, index upwards) what stays is a beginning: of top_k entries, of the fewest whose weights reach top_p of those
// of the top_k, of those with min_p of the largest one's weight.  So all that is wanted of the row is one place in that order, a border:
// the key (value, index) of the last entry that stays.  Then the token is the first one that stays whose sum of weights, in the order of the index,
// is above the random number times the whole.
//
// Which token it is hangs on comparisons of sums: with weights in 32 bits one row in eight of 32000 entries would have a border within the rounding
// of its sum.  Sums are fp64 and weights 2^-37 exact, by Tang's method: (x - max) log2(e) / T = (n + r) / 64, 2^n/64 from a table of 2^(j / 64),
// 2^r/64 = 1 + r (c1 + r (c2 + r c3)) with the least largest relative error on |r| <= 0.51 (found by linear programming: 6.7e-12; 1 stays
// exact, so that sums of equal largest logits are whole numbers).  Nine fp64 operations an entry and one a sum: the GPU has half as many fp64
// units as fp32 ones, and a pass that took n and the exponents through whole numbers waited for the issue of 49 instructions an entry.
//
// Passes over the row, out of L2 but for the first:
//   1  the maximum
//   2  with top_k or top_p: how many entries lie in each of 2048 bins of T / 92 below the maximum (n, but from fp32)
//   3  top_k: a list of the k largest and a few more, bounded by the threads' maxima (without pass 2) or by the bins, in order; all the rest
//      happens on it.  Where k is more than a list holds, the bin with the border is known and its entries are put in order.
//      top_p: the counts times the bins' weights tell the bin but for an error in the fourth digit; the exact sum in front of it, and its entries
//      in order, find the border or say on which side it lies.  Where the bin, with the neighbour that may have the border instead, holds more
//      entries than the list, the border is found by bisection of the keys, 64 passes.  That is so for equal logits, and for some rows that
//      are long and flat: of normal logits of size 2.5 over 152000 entries none at T = 1, one in five or more from T = 2 on (top_p 0.9); one in eight
//      of size 1 at T = 1.  Such a row takes 0.5 ms alone, not 30 us, and 64 rows with some of them 1.2 ms, not 58 us.
//   4  the sum of what stays, a segment a warp (top_p's pass has it); then the segment in which the random number falls, a vector a thread
// A row is a CTA of 512 threads, or of 256 with four on an SM where there are many rows, or a cluster of CTAs that tell each other their sums.
//
// What bounds it: latency for few rows (one of 32000, top_k 50 and top_p 0.9: 12.1 us; before, with all passes apart, 58); the issue of whole-number
// and comparing instructions, which have half the rate of others, for many (512 rows of 32000 fp32, top_p and min_p: 72 us, 0.9 TB/s; by the units'
// rates alone the counts' additions in shared memory would be 8 and the weights' fp64 operations 10 of it; 2048 rows of fp16: 39 without weights, 100 with all of them, 69 with top_k 50, 200
// with top_p).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

constexpr int kFew = 512, kMany = 256;          // threads of a CTA where there are few rows, or many
constexpr int kMaxCluster = 8;
constexpr int kBins = 2048;                     // 22 nats; counted again where that is not enough:
constexpr int kWide = 32;                       // bins so many times as wide, 710 nats
constexpr int kFewEnough = 600;                 // of 4 x 256 maxima 905 values, of 4 x 512 711: they fit the list
constexpr int kAhead = 2;                       // vectors under way while one is worked on
constexpr int kList = 1024;                     // entries of the bins around a border
constexpr int kTableLog2 = 6, kTable = 1 << kTableLog2;                  // 2^(j / 64)
constexpr int kCopies = 8;                      // of the table: fewer lanes ask the same bank for different entries
constexpr double kLog2e = 1.4426950408889634074;
constexpr double kDepth = 690.;                 // weights from e^-690 on are normal numbers

using ptx::exp2_approx;
typedef unsigned long long u64;

struct SampleParams {
  const void* logits;
  const float* uniform;
  int* token;
  float* logprob;
  const float* temperatures;                    // of every row, or null: the number below
  const int* top_ks;
  const float* top_ps;
  const float* min_ps;
  int64_t stride, rows;
  int V;
  float temperature, top_p, min_p;
  int top_k;
};

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Values in the order of unsigned numbers; both zeros are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ u64 entry_of(float v, int index) { return (u64)key_of(v) << 32 | (uint32_t)~index; }

// A row as vectors of 16 bytes on their own grid: its first element is element `lead` of vector 0.  The first and the last vector may reach
// beyond the row (not beyond the 16 bytes that hold its ends, so not beyond the memory that it lies in); what they hold there becomes -inf, an
// excluded entry.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const uint4* vectors;
  const T* x;
  int lead, V, count;
  __device__ __forceinline__ Row(const T* row, int size) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    vectors = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15);
    x = row;
    V = size;
    count = (int)(((int64_t)lead + size + N - 1) / N);
  }
  __device__ __forceinline__ int first(int j) const { return j * N - lead; }          // index of a vector's first element
  __device__ __forceinline__ uint4 load(int j) const {
    uint4 v = __ldg(vectors + j);
    const int at = first(j);
    if (at < 0 || at > V - N) {
      constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (at + i >= 0 && at + i < V) continue;
        if (sizeof(T) == 4) w[i & 3] = kNone;
        else w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | kNone << 16 : (w[i / 2] & 0xffff0000u) | kNone;
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
  }
  __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = u.x;
        f[2 * i + 1] = u.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  // the largest (the least) value of a vector, NaN where there is one
  template <bool kLeast>
  __device__ __forceinline__ static float extreme(const uint4& v) {
    if constexpr (sizeof(T) == 4) {
      float a = __uint_as_float(v.x);
      for (const uint32_t u : {v.y, v.z, v.w}) {
        if (kLeast) asm("min.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(__uint_as_float(u)));
        else asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(__uint_as_float(u)));
      }
      return a;
    } else {
      using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      const T2* w = reinterpret_cast<const T2*>(&v);
      const T2 a = kLeast ? __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3])) : __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
      return to_float(kLeast ? __hmin_nan(T(a.x), T(a.y)) : __hmax_nan(T(a.x), T(a.y)));
    }
  }
  // The type's least number that is not below an fp32 one; the elements of a vector (bits) that reach `from` and do not reach `to`.
  __device__ __forceinline__ static T up(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_ru(v);
    else return __float2bfloat16_ru(v);
  }
  __device__ __forceinline__ static unsigned between(const uint4& v, T from, T to) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t in[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        in[i] = __uint_as_float(w[i]) >= from && __uint_as_float(w[i]) < to ? 1u << i : 0u;
      } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2 x = *reinterpret_cast<const T2*>(&w[i]);
        in[i] = __hge2_mask(x, T2(from, from)) & __hlt2_mask(x, T2(to, to));
      }
    }
    if ((in[0] | in[1] | in[2] | in[3]) == 0) return 0;
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= sizeof(T) == 4 ? in[i] : (in[i] & 1u) << (2 * i) | (in[i] >> 31) << (2 * i + 1);
    return bits;
  }
  __device__ __forceinline__ static float highest(const uint4& v) { return extreme<false>(v); }
  __device__ __forceinline__ static float lowest(const uint4& v) { return extreme<true>(v); }
};

// An entry's value.
__device__ __forceinline__ float value_of(u64 e) {
  const uint32_t k = (uint32_t)(e >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// The last entry that stays, as a pass compares with it: values from `value` on up to the index, from `next` on behind it.
struct Border {
  float value, next;
  int index;
  __device__ __forceinline__ explicit Border(u64 e) : value(value_of(e)), next(value_of(e + (1ull << 32))), index((int)min(~(uint32_t)e, 0x7fffffffu)) {}
};
// sum += w where v >= from
__device__ __forceinline__ void add_from(double& sum, double w, float v, float from) {
  asm("{\n.reg .pred p;\nsetp.ge.f32 p, %1, %2;\n@p add.f64 %0, %0, %3;\n}" : "+d"(sum) : "f"(v), "f"(from), "d"(w));
}

__device__ __forceinline__ int mul(int a, int b) {
  int r;
  asm("mul.lo.s32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// What the CTAs of a row tell each other.
struct Note {
  double a, b;
  int n, m;
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
sample_tokens_kernel(const SampleParams p) {
  constexpr int kWarps = kThreads / 32, kBuckets = 2 * kThreads, kEach = kList / kThreads;
  static_assert(2 * kBuckets <= kBins, "buckets");
  constexpr int N = Vec<T>::N;
  __shared__ double sm_table[kTable * kCopies];
  __shared__ __align__(16) int sm_bins[kBins];
  __shared__ __align__(16) u64 sm_own[2][kList], sm_list[kList];          // this CTA's part of the list; all of it
  __shared__ __align__(16) u64 sm_sorted[kList];
  int* sm_bucket = sm_bins;                     // [2][kBuckets], when the bins are no longer wanted
  __shared__ Note sm_notes[2][kMaxCluster];
  __shared__ double sm_warp[kWarps], sm_segment[kWarps];
  __shared__ float2 sm_extreme[kWarps];
  __shared__ int sm_warp_n[kWarps], sm_count, sm_index, sm_border[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = gridDim.x, rank = blockIdx.x;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (tid < kTable) {
    const double w = exp2((double)tid / kTable);
#pragma unroll
    for (int i = 0; i < kCopies; ++i)
      sm_table[tid * kCopies + i] = __hiloint2double(__double2hiint(w) - (tid << (20 - kTableLog2)), __double2loint(w));
  }
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  if (row >= p.rows) return;                    // (whole clusters)
  if (ranks > 1) ptx::cluster_arrive_relaxed(); // (every CTA of the cluster runs before anything is stored in it)
  auto meet = [&]() {                           // all threads of the row
    if (ranks > 1) {
      __syncwarp();                             // (the barrier wants whole warps)
      ptx::cluster_arrive();
      ptx::cluster_wait();
    } else {
      __syncthreads();
    }
  };
  // the same variable of another CTA of the row
  auto remote = [&](auto* at, int r) {
    u64 a;
    asm("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"(at), "r"(r));
    return reinterpret_cast<decltype(at)>(a);
  };
  // Everybody's notes, in the order of the CTAs.  One meeting: the next notes go to the other place, and those after them are written behind
  // the next meeting, when these have been read.
  int turn = 0;
  auto exchange = [&](Note mine) {
    if (tid < ranks) *remote(&sm_notes[turn][rank], tid) = mine;
    meet();
    const Note* all = sm_notes[turn];
    turn ^= 1;
    return all;
  };
  // the sum of all threads of the CTA
  auto block_sum = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sm_warp[warp] = v;
    __syncthreads();
    double s = 0.;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sm_warp[w];
    return s;
  };
  auto row_sum = [&](double v) {
    const Note* notes = exchange({block_sum(v), 0., 0, 0});
    double s = 0.;
    for (int r = 0; r < ranks; ++r) s += notes[r].a;
    return s;
  };

  // Every CTA has a slice of the row's vectors, every warp a segment of it.
  const Row<T> x(static_cast<const T*>(p.logits) + row * p.stride, p.V);
  const int per = (x.count + ranks - 1) / ranks, begin = min(rank * per, x.count), end = min(begin + per, x.count);
  const int share = (per + kWarps - 1) / kWarps;
  const int from = min(begin + warp * share, end), to = min(from + share, end);

  // ---- 1: the maximum, NaN where there is one --------------------------------------------------------------------------------------
  auto join = [](float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
  };
  float own_most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};       // of four sets of this thread's vectors
  for (int j = from + lane; j < to; j += 128) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x.load(min(j + 32 * i, to - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + 32 * i < to) own_most[i] = join(own_most[i], x.highest(v[i]));       // (a vector is one set's)
  }
  float m = join(join(own_most[0], own_most[1]), join(own_most[2], own_most[3]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = join(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sm_warp[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = join(m, (float)sm_warp[w]);
  {
    if (ranks > 1) ptx::cluster_wait();         // (the one at the start)
    const Note* notes = exchange({(double)m, 0., 0, 0});
    for (int r = 0; r < ranks; ++r) m = join(m, (float)notes[r].a);
  }
  const bool writes = rank == 0 && tid == 0;
  const float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
  const int want_k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float want_p = p.top_ps ? p.top_ps[row] : p.top_p, want_min = p.min_ps ? p.min_ps[row] : p.min_p;
  if (!(m < INFINITY) || m == -INFINITY) {      // a NaN, an infinity, nothing that is allowed
    if (writes) {
      p.token[row] = -1;
      if (p.logprob) p.logprob[row] = m == -INFINITY ? -INFINITY : NAN;
    }
    return;
  }
  if (!(temperature > 0.f) || want_p <= 0.f || want_k == 1) {             // the first of the largest
    int at = 0x7fffffff;
    for (int j = from + lane; j < to; j += 32) {
      const uint4 v = x.load(j);
      if (x.highest(v) != m) continue;
      float f[N];
      x.unpack(v, f);
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (f[i] == m) at = min(at, x.first(j) + i);
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) sm_warp_n[warp] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) at = min(at, sm_warp_n[w]);
    const Note* notes = exchange({0., 0., at, 0});
    if (writes) {
      for (int r = 1; r < ranks; ++r) at = min(at, notes[r].n);
      p.token[row] = at;
      if (p.logprob) p.logprob[row] = 0.f;
    }
    return;
  }

  const double top = m, t_eff = temperature, scale = kLog2e * kTable / t_eff;
  const char* table = reinterpret_cast<const char*>(sm_table + (lane & (kCopies - 1)));
  // The bin of a value, which only grows as the value falls, as a number above 1.5 * 2^23; its low bits count.
  constexpr float kBase = 12582912.f;
  float bins_per = fminf((float)scale, 1e30f);
  int unit = 1;                                 // n of a bin
  auto bin_of = [&](float v) { return fmaf(m - v, bins_per, kBase); };
  // 2^((x - max) log2(e) / T) = 2^n/64 2^r/64, for values from `low` on.  The maximum is taken off first, so that its own weight is 1 to the bit.
  auto weight = [&](float v) {
    constexpr double c1 = 0.0108304246963882758, c2 = 0.000058649173078506538, c3 = 2.1173088255274404e-7;
    constexpr double kMagic = 6755399441055744.;         // 1.5 * 2^52: its sum with a number has the nearest whole one in its low bits
    const double d = (double)v - top, shifted = fma(d, scale, kMagic), r = fma(d, scale, kMagic - shifted);
    const int n = __double2loint(shifted);
    // (multiplications take the other pipe; the table's entries come without their own part of the exponent that n << 14 adds)
    const double of = *reinterpret_cast<const double*>(table + mul(n & (kTable - 1), kCopies * 8));
    return fma(fma(fma(r, c3, c2), r, c1), r, 1.) * __hiloint2double(mul(n, 1 << (20 - kTableLog2)) + __double2hiint(of), __double2loint(of));
  };
  // (less weight is as good as excluded, and so is what lies further below the maximum than fp32 can say)
  const float low = fmaxf(__double2float_ru(top - kDepth * t_eff), fmaxf(m - 3.402823466e38f, -3.402823466e38f));
  const bool has_k = want_k > 0 && want_k < p.V, has_p = want_p < 1.f;
  u64 border = (u64)key_of(low) << 32;          // the smallest entry that stays
  const u64 all_of_weight = border;
  if (want_min > 0.f) {                         // w >= min_p: a value, rounded up to the next fp32 number
    // (an infinite temperature makes all weights 1)
    const double least = temperature == INFINITY ? -INFINITY : want_min < 1.f ? top + t_eff * log((double)want_min) : top;
    border = max(border, (u64)key_of(__double2float_ru(least)) << 32);
  }
  int listed = 0, own_turn = 0;
  double sum_all, sum_above;
  // The first n entries of the list, those with the largest key(entry) first: by buckets that fall with the key, and within a bucket an entry's
  // place is the number of larger ones.
  auto order = [&](int n, auto key, auto bucket) {
    int* start = sm_bucket;
    int* end = sm_bucket + kBuckets;
    for (int i = tid; i < kBuckets; i += kThreads) end[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) atomicAdd(&end[bucket(sm_list[i])], 1);
    __syncthreads();
    const int2 mine = reinterpret_cast<const int2*>(end)[tid];
    int upto = mine.x + mine.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sm_warp_n[warp] = upto;
    __syncthreads();
    int before = upto - mine.x - mine.y;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) before += sm_warp_n[w];
    reinterpret_cast<int2*>(start)[tid] = make_int2(before, before + mine.x);
    reinterpret_cast<int2*>(end)[tid] = make_int2(before, before + mine.x);
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const u64 e = sm_list[i];
      sm_sorted[atomicAdd(&end[bucket(e)], 1)] = e;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const u64 e = sm_sorted[i], k = key(e);
      const int b = bucket(e), from = start[b], to = end[b];
      int place = from;
      for (int q = from; q < to; ++q) place += key(sm_sorted[q]) > k;
      sm_list[place] = e;
    }
    __syncthreads();
  };
  auto order_by_value = [&](int n) {
    // buckets between the list's largest and its least value
    float hi = -INFINITY, lo = INFINITY;
    for (int i = tid; i < n; i += kThreads) {
      const float v = value_of(sm_list[i]);
      hi = fmaxf(hi, v);
      lo = fminf(lo, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (lane == 0) sm_extreme[warp] = make_float2(hi, lo);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      hi = fmaxf(hi, sm_extreme[w].x);
      lo = fminf(lo, sm_extreme[w].y);
    }
    const float per = hi > lo ? fminf((kBuckets - 1) / (hi - lo), 1e30f) : 0.f;
    order(n, [](u64 e) { return e; }, [&](u64 e) { return (int)fminf((hi - value_of(e)) * per, kBuckets - 1.f); });
  };
  // The parts of the list that the CTAs have (sm_own, their lengths the notes' n) in order.
  auto put_in_order = [&](const Note* notes) {
    listed = 0;
    for (int r = 0; r < ranks; ++r) {
      const int n = min(notes[r].n, kList + 1);
      if (listed + n <= kList) {
        const u64* other = remote(sm_own[own_turn], r);
        for (int i = tid; i < n; i += kThreads) sm_list[listed + i] = other[i];
      }
      listed = min(listed + n, kList + 1);
    }
    own_turn ^= 1;                              // (others may still read this one)
    __syncthreads();
    if (listed > kList) return false;
    order_by_value(listed);
    return true;
  };
  // The values from which a bin is reached, in the row's type: all values from edge(b) on, and no others, lie in bins in front of b.  (But for
  // fp32's last bits, in which the counts may see it differently.)
  auto edge = [&](int b) { return b <= 0 ? T(INFINITY) : x.up(b >= kBins ? low : fmaxf(m - ((float)b - 0.5f) / bins_per, low)); };
  // The entries of a vector whose bits are set, to this CTA's part of the list.
  auto push = [&](unsigned hits, int first, auto also) {
    while (hits) {
      const int at = first + __ffs(hits) - 1;
      hits &= hits - 1;
      const float v = to_float(x.x[at]);
      if (!also(v, at)) continue;
      const int n = atomicAdd(&sm_count, 1);
      if (n < kList) sm_own[own_turn][n] = entry_of(v, at);
    }
  };
  // Without sums: the entries from `reach` on for which `also` holds.
  auto gather_from = [&](T reach, auto also) {
    if (tid == 0) sm_count = 0;
    __syncthreads();
#pragma unroll 1
    for (int j = from + lane; j < to; j += 128) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = x.load(min(j + 32 * i, to - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + 32 * i < to) push(x.between(v[i], reach, T(INFINITY)), x.first(j + 32 * i), also);
    }
    __syncthreads();
    return put_in_order(exchange({0., 0., sm_count, 0}));
  };
  // The entries of bins [first, last], those of the counts.
  auto gather = [&](int first, int last) {
    const float from_bin = kBase + (float)first, to_bin = last == kBins - 1 ? INFINITY : kBase + (float)last;
    return gather_from(edge(last + 2), [&](float v, int) {               // (a bin to spare)
      const float bin = bin_of(v);
      return bin >= from_bin && bin <= to_bin && v >= low;
    });
  };
  // The k largest, and some more: the k-th largest of the maxima that the threads have of sets of vectors bounds the k-th largest value from below.
  // It is found to a part of the maxima's range.  Of n maxima, values from there on are about -n log(1 - k / n).
  auto gather_few = [&](int k) {
    float lo = INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (own_most[i] >= low) lo = fminf(lo, own_most[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    if (lane == 0) sm_extreme[warp].x = lo;
    for (int i = tid; i < kBuckets; i += kThreads) sm_bucket[i] = 0;
    if (tid == 0) sm_index = kBuckets;          // (fewer maxima than k: everything)
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) lo = fminf(lo, sm_extreme[w].x);
    const float per = m > lo ? fminf((kBuckets - 1) / (m - lo), 1e30f) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (own_most[i] >= low) atomicAdd(&sm_bucket[(int)fminf((m - own_most[i]) * per, kBuckets - 1.f)], 1);
    __syncthreads();
    const int2 mine = reinterpret_cast<const int2*>(sm_bucket)[tid];
    int upto = mine.x + mine.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sm_warp_n[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) upto += sm_warp_n[w];
    const int before = upto - mine.x - mine.y;
    if (before < k && upto >= k) sm_index = 2 * tid + (before + mine.x < k);
    __syncthreads();
    const int bucket = sm_index;
    return gather_from(x.up(bucket >= kBuckets - 1 || !(per > 0.f) ? low : fmaxf(m - ((float)bucket + 1.01f) / per, low)),
                       [&](float v, int) { return v >= low; });
  };
  // Sums up to every thread's kEach entries, in order; the sum of all.
  auto scan = [&](const double (&w)[kEach], double& before) {
    double own = 0., all = 0.;
#pragma unroll
    for (int i = 0; i < kEach; ++i) own += w[i];
    double upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 31) sm_warp[warp] = upto;
    if (tid == 0) sm_index = 0x7fffffff;
    __syncthreads();
    before = upto - own;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) {
      if (q < warp) before += sm_warp[q];
      all += sm_warp[q];
    }
    return all;
  };
  // What a pass finds: sums over the row of all that the border `lowest` keeps and of those from `above` on; the second of each warp's segment in
  // sm_segment; the entries from `near` on below `above` that it keeps, of the whole row and in order, in sm_list, if they fit.
  auto pass = [&](T above, T near, u64 lowest) {
    const Border kept(lowest);
    const float above_f = to_float(above);
    if (tid == 0) sm_count = 0;
    __syncthreads();
    double s = 0., a = 0.;
    uint4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (from + lane + 32 * i < to) ahead[i] = x.load(from + lane + 32 * i);
#pragma unroll 1
    for (int j = from + lane; j < to; j += 32) {
      const uint4 v = ahead[0];
#pragma unroll
      for (int i = 0; i + 1 < kAhead; ++i) ahead[i] = ahead[i + 1];
      if (j + 32 * kAhead < to) ahead[kAhead - 1] = x.load(j + 32 * kAhead);
      if (x.highest(v) < kept.value) continue;
      float f[N];
      x.unpack(v, f);
      const int at = x.first(j);
      if (at <= kept.index && at + N - 1 > kept.index) {           // the border's own index is among these
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i > kept.index && f[i] == kept.value) f[i] = -INFINITY;
      }
      const float least = at > kept.index ? kept.next : kept.value;
      // (no branch an entry: the chains of fp64 operations of several run side by side)
#pragma unroll
      for (int i = 0; i < N; ++i)
        asm("{\n.reg .pred p, q;\nsetp.ge.f32 p, %2, %3;\n@p add.f64 %0, %0, %5;\nsetp.ge.and.f32 q, %2, %4, p;\n@q add.f64 %1, %1, %5;\n}"
            : "+d"(s), "+d"(a) : "f"(f[i]), "f"(least), "f"(above_f), "d"(weight(f[i])));
      push(x.between(v, near, above), at, [&](float v, int i) { return v >= (i > kept.index ? kept.next : kept.value); });
    }
    // the segments' sums, the CTA's and the row's
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      a += __shfl_xor_sync(0xffffffffu, a, o);
    }
    if (lane == 0) {
      sm_warp[warp] = s;
      sm_segment[warp] = a;
    }
    __syncthreads();
    Note mine = {0., 0., sm_count, 0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      mine.a += sm_warp[w];
      mine.b += sm_segment[w];
    }
    const Note* notes = exchange(mine);
    sum_all = sum_above = 0.;
    for (int r = 0; r < ranks; ++r) {
      sum_all += notes[r].a;
      sum_above += notes[r].b;
    }
    return put_in_order(notes);
  };
  // The largest entry e for which what(entries >= e), a sum over the row, reaches `goal`: by bisection, for rows that fit no list.
  auto bisect = [&](u64 lowest, double goal, auto what) {
    u64 lo = lowest, hi = ~0ull;                // what(>= lo) reaches it, what(>= hi) does not
    while (hi - lo > 1) {
      const u64 mid = lo + (hi - lo) / 2;
      double s = 0.;
      for (int j = from + lane; j < to; j += 32) {
        float f[N];
        x.unpack(x.load(j), f);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (f[i] >= low && entry_of(f[i], x.first(j) + i) >= mid) s += what(f[i]);
      }
      if (row_sum(s) >= goal) lo = mid; else hi = mid;
    }
    return lo;
  };

  bool segments = false;                        // sm_segment has the sums above the list, and the list what lies around the border
  if (has_k || has_p) {
    // ---- 2: how many entries lie how far below the maximum, and the bin in which the border lies ----------------------------------------
    constexpr int kMost = kBins / kThreads;
    int mine = max(kMost / ranks, 1);           // of the whole row every CTA has a part of the bins, every thread a few neighbours
    const int bin0 = rank * (kBins / ranks) + tid * mine;
    if (tid * mine >= kBins / ranks) mine = 0;
    int n_of[kMost], sum;
    float mass_of[kMost], mass = 0.f;           // the bins' weights, an estimate in fp32 by their middles
    auto masses = [&](int n, int most) {
      mass = 0.f;
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        mass_of[i] = i < mine ? (float)min(n_of[i], max(most - n, 0)) * exp2_approx((float)((bin0 + i) * unit) * (-1.f / kTable)) : 0.f;
        mass += mass_of[i];
        n += n_of[i];
      }
    };
    int before = 0, all = 0;                    // entries in front of this thread's bins, of the row
    float mass_before = 0.f, mass_end = 0.f, mass_all = 0.f;         // (a thread's end is the next one's beginning to the bit)
    auto totals = [&]() {
      int upto = sum;
      float mass_upto = mass;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        const float f = __shfl_up_sync(0xffffffffu, mass_upto, o);
        if (lane >= o) { upto += v; mass_upto += f; }
      }
      __syncthreads();
      if (lane == 31) { sm_warp_n[warp] = upto; sm_warp[warp] = mass_upto; }
      if (tid == 0) sm_border[0] = -1;
      __syncthreads();
      before = upto - sum;
      mass_end = mass_upto;
      mass_before = __shfl_up_sync(0xffffffffu, mass_upto, 1);
      if (lane == 0) mass_before = 0.f;
      float mass_base = 0.f;
      int slice = 0;
      float mass_slice = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = (float)sm_warp[w];
        if (w < warp) { before += sm_warp_n[w]; mass_base += f; }
        slice += sm_warp_n[w];
        mass_slice += f;
      }
      const Note* notes = exchange({(double)mass_slice, 0., slice, 0});    // (and everybody has read the bins)
      mass_before += mass_base;
      mass_end += mass_base;
      all = 0;
      mass_all = 0.f;
      for (int r = 0; r < ranks; ++r) {
        if (r == rank) { mass_before += mass_all; mass_end += mass_all; }
        if (r < rank) before += notes[r].n;
        all += notes[r].n;
        mass_all += (float)notes[r].a;
      }
    };
    auto count = [&]() {
      for (int i = tid; i < kBins / 4; i += kThreads) reinterpret_cast<int4*>(sm_bins)[i] = make_int4(0, 0, 0, 0);
      __syncthreads();
      auto place_of = [&](float v) { return (int)(min(__float_as_uint(bin_of(v)), 0x4b400000u + kBins - 1) - 0x4b400000u); };
#pragma unroll 1
      for (int j = from + lane; j < to; j += 128) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = x.load(min(j + 32 * i, to - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (j + 32 * i >= to) break;
          float f[N];
          x.unpack(v[i], f);
          if (x.lowest(v[i]) >= low) {
#pragma unroll
            for (int q = 0; q < N; ++q) atomicAdd(&sm_bins[place_of(f[q])], 1);
          } else {
#pragma unroll
            for (int q = 0; q < N; ++q)
              if (f[q] >= low) atomicAdd(&sm_bins[place_of(f[q])], 1);
          }
        }
      }
      meet();
      sum = 0;
#pragma unroll
      for (int i = 0; i < kMost; ++i) n_of[i] = 0;
      if (ranks == 1) {
#pragma unroll
        for (int i = 0; i < kMost; i += 4) {
          const int4 v = *reinterpret_cast<const int4*>(sm_bins + bin0 + i);
          n_of[i] = v.x; n_of[i + 1] = v.y; n_of[i + 2] = v.z; n_of[i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kMost / 2; ++i) {
          int v[kMaxCluster];
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r) v[r] = i < mine && r < ranks ? *remote(&sm_bins[bin0 + i], r) : 0;
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r) n_of[i] += v[r];
        }
      }
#pragma unroll
      for (int i = 0; i < kMost; ++i) sum += n_of[i];
      if (!has_k) masses(0, 0x7fffffff);
      totals();
    };
    // what one thread of the row has found, to everybody
    auto everybody = [&](int& bin, int& more) {
      __syncthreads();
      const Note* notes = exchange({0., 0., sm_border[0], sm_border[1]});
      bin = -1;
      for (int r = 0; r < ranks; ++r)
        if (notes[r].n >= 0) {
          bin = notes[r].n;
          more = notes[r].m;
        }
      if (tid == 0) sm_border[0] = -1;
      __syncthreads();
    };
    // the bin in which the k-th entry lies, and how many lie above it
    auto find_k = [&](int& bin, int& above) {
      int n = before;
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        if (i < mine && n < want_k && n + n_of[i] >= want_k) {
          sm_border[0] = bin0 + i;
          sm_border[1] = n;
        }
        n += n_of[i];
      }
      everybody(bin, above);
    };
    // the bin in which the estimated weights reach top_p, and on which side a border so near its edge that the neighbour may have it
    auto find_p = [&](int& bin, int& edge) {
      const float goal = mass_all * want_p;
      float at = mass_before;
      if (at < goal && mass_end >= goal) {
        int in = bin0 + mine - 1, side = 0;
        bool open = true;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          if (open && i < mine && at + mass_of[i] >= goal) {
            in = bin0 + i;
            side = goal - at < mass_of[i] * 0.1f ? -1 : at + mass_of[i] - goal < mass_of[i] * 0.1f ? 1 : 0;
            open = false;
          }
          at += mass_of[i];
        }
        sm_border[0] = in;
        sm_border[1] = side;
      }
      edge = 0;
      everybody(bin, edge);
      if (bin < 0) bin = kBins - 1;             // (the sums' last bits)
    };

    int bin = 0, more = 0;
    auto find = [&]() {
      count();
      if (has_k && want_k < all) find_k(bin, more);
      else if (has_p && !has_k) find_p(bin, more);
    };
    // ---- 3, top_k: a list of all that can stay --------------------------------------------------------------------------------------------
    bool on_list = has_k && want_k <= kFewEnough / ranks && gather_few(want_k);
    if (!on_list) {
      find();
      if (bin == kBins - 1) {                   // further away than the bins reach
        unit = kWide;
        bins_per *= 1.f / kWide;
        find();
      }
      on_list = has_k && want_k < all && want_k <= kList && gather(0, bin);
    }
    if (on_list) {
      // All that can stay is on the list, and everybody has it.
      int stay = min(want_k, listed);
      double w[kEach], before_w;
#pragma unroll
      for (int i = 0; i < kEach; ++i) w[i] = tid * kEach + i < stay ? weight(value_of(sm_list[tid * kEach + i])) : 0.;
      if (has_p) {
        const double need = (double)want_p * scan(w, before_w);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          before_w += w[i];
          if (tid * kEach + i < stay && before_w >= need) {
            atomicMin(&sm_index, tid * kEach + i);
            break;
          }
        }
        __syncthreads();
        stay = min(stay, sm_index == 0x7fffffff ? stay : sm_index + 1);
      }
      // those below min_p's border
      if (tid == 0) sm_count = stay;
      __syncthreads();
      for (int i = tid; i < stay; i += kThreads)
        if (sm_list[i] < border) atomicMin(&sm_count, i);
      __syncthreads();
      stay = max(sm_count, 1);
      // in the order of the index
      const float per = (float)kBuckets / p.V;
      order(stay, [](u64 e) { return (uint32_t)e; }, [&](u64 e) { return min((int)((float)~(uint32_t)e * per), kBuckets - 1); });
#pragma unroll
      for (int i = 0; i < kEach; ++i) w[i] = tid * kEach + i < stay ? weight(value_of(sm_list[tid * kEach + i])) : 0.;
      const double whole = scan(w, before_w);
      const float u = p.uniform[row];
      const double goal = u > 0.f ? fmin((double)u, 1.) * whole : 0.;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        before_w += w[i];
        if (tid * kEach + i < stay && before_w > goal) {
          atomicMin(&sm_index, tid * kEach + i);
          break;
        }
      }
      __syncthreads();
      if (writes) {
        const u64 e = sm_list[min(sm_index, stay - 1)];
        p.token[row] = (int)~(uint32_t)e;
        if (p.logprob) p.logprob[row] = (float)log(weight(value_of(e)) / whole);
      }
      meet();                                 // (others may still read this CTA's part of the list)
      return;
    }
    u64 border_k = all_of_weight;
    if (has_k && want_k < all) {                // more than the list holds: the last one that stays, by its bin
      const int above = more;
      if (gather(bin, bin)) border_k = sm_list[want_k - above - 1];
      else border_k = bisect(all_of_weight, (double)want_k, [](float) { return 1.; });
      __syncthreads();
    }
    u64 border_p = 0;
    bool by_min_p = false;                      // min_p's is the border, and the sums are those above it
    if (has_p) {
      // ---- 3, top_p ----------------------------------------------------------------------------------------------------------------------
      int side = more;
      if (has_k) {
        masses(before, min(want_k, all));
        totals();
        find_p(bin, side);
      }
      int first = max(bin + min(side, 0), 0), last = min(bin + max(side, 0), kBins - 1);
      // Where min_p's border seems to lie above top_p's: what it leaves is less than top_p, or top_p's is the higher one after all.
      const float min_border = value_of(border);
      if (min_border >= to_float(edge(first))) {
        const T from_there = x.up(min_border);
        segments = pass(from_there, from_there, border_k);
        by_min_p = sum_above < (double)want_p * sum_all;
      }
      bool found = by_min_p;
      for (int attempt = 0; attempt < 16 && !found; ++attempt) {
        segments = pass(edge(first), edge(last + 1), border_k);
        if (!segments) break;
        const double need = (double)want_p * sum_all;
        if (sum_above >= need && first > 0) {   // it lies further up
          last = first - 1;
          first = max(first - 2, 0);
          continue;
        }
        // the list's sums, in order
        double w[kEach], here;
#pragma unroll
        for (int i = 0; i < kEach; ++i) w[i] = tid * kEach + i < listed ? weight(value_of(sm_list[tid * kEach + i])) : 0.;
        scan(w, here);
        here += sum_above;
        // the first place whose sum reaches what is wanted
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          here += w[i];
          if (tid * kEach + i < listed && here >= need) {
            atomicMin(&sm_index, tid * kEach + i);
            break;
          }
        }
        __syncthreads();
        const int place = sm_index;
        if (place == 0x7fffffff) {
          if (last == kBins - 1) {              // the sums differ in their last bits: everything stays
            found = true;
            break;
          }
          first = last + 1;
          last = min(last + 2, kBins - 1);
          continue;
        }
        border_p = sm_list[place];
        found = true;
      }
      if (!found) {
        segments = false;
        double s = 0.;
        for (int j = from + lane; j < to; j += 32) {
          float f[N];
          x.unpack(x.load(j), f);
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (f[i] >= low && entry_of(f[i], x.first(j) + i) >= border_k) s += weight(f[i]);
        }
        const double need = (double)want_p * row_sum(s);
        border_p = bisect(border_k, need, weight);
      }
    }
    // (where min_p leaves less than the bins in front of the list, their sums are of no use)
    if (!by_min_p && (listed == 0 || border > sm_list[0])) segments = false;
    border = max(border, max(border_k, border_p));
  }

  // ---- 4: the sums of what stays, a segment a warp; where the random number falls in them ----------------------------------------------
  const Border stays(border);
  if (segments) {
    // what stays of the list, each to its segment, in order
    double s = 0.;
    for (int i = lane; i < listed; i += 32) {
      const u64 e = sm_list[i];
      const int j = ((int)~(uint32_t)e + x.lead) / N;
      if (e >= border && j >= from && j < to) s += weight(value_of(e));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sm_segment[warp] += s;
  } else {
    double s = 0.;
#pragma unroll 1
    for (int j = from + lane; j < to; j += 32) {
      const uint4 v = x.load(j);
      if (x.highest(v) < stays.value) continue;
      float f[N];
      x.unpack(v, f);
      const int at = x.first(j);
      if (at <= stays.index && at + N - 1 > stays.index) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at + i > stays.index && f[i] == stays.value) f[i] = -INFINITY;
      }
      const float least = at > stays.index ? stays.next : stays.value;
#pragma unroll
      for (int i = 0; i < N; ++i) add_from(s, weight(f[i]), f[i], least);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sm_segment[warp] = s;
  }
  __syncthreads();
  double own = 0.;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) own += sm_segment[w];
  const Note* notes = exchange({own, 0., 0, 0});
  double sums[kMaxCluster], whole = 0.;
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) {
    sums[r] = r < ranks ? notes[r].a : 0.;
    whole += sums[r];
  }
  const float u = p.uniform[row];
  const double goal = u > 0.f ? fmin((double)u, 1.) * whole : 0.;
  int holder = -1, last = 0;                    // the CTA in which it falls; the last one with anything that stays
  double run = 0., before = -1.;
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) {
    if (sums[r] > 0.) last = r;
    if (holder < 0 && run + sums[r] > goal) {
      holder = r;
      before = run;
    }
    run += sums[r];
  }
  if (holder < 0) holder = last;                // u = 1, or the sums' last bits: the last entry that stays
  if (rank != holder) return;
  int segment = -1, last_segment = 0;
  double at = before;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const double v = sm_segment[w];
    if (v > 0.) last_segment = w;
    if (segment < 0 && before >= 0. && at + v > goal) segment = w;
    if (segment < 0) at += v;
  }
  const bool at_end = segment < 0;
  if (at_end) segment = last_segment;
  const int first = min(begin + segment * share, end), behind = min(first + share, end);
  if (tid == 0) {
    sm_index = 0x7fffffff;
    sm_count = -1;
  }
  __syncthreads();
  // as many vectors as threads at a time, in order
  for (int base = first; base < behind; base += kThreads) {
    const int j = base + tid;
    double w[N], mine = 0.;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0.;
    if (j < behind) {
      float f[N];
      x.unpack(x.load(j), f);
      const int at = x.first(j);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (f[i] >= (at + i > stays.index ? stays.next : stays.value)) w[i] = weight(f[i]);
        mine += w[i];
      }
    }
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 31) sm_warp[warp] = upto;
    __syncthreads();
    double sum = at + (upto - mine), next = at;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) {
      if (q < warp) sum += sm_warp[q];
      next += sm_warp[q];
    }
    at = next;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      sum += w[i];
      if (w[i] > 0.) {
        if (!at_end && sum > goal) atomicMin(&sm_index, x.first(j) + i);
        atomicMax(&sm_count, x.first(j) + i);
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    const int token = sm_index != 0x7fffffff ? sm_index : sm_count;
    p.token[row] = token;
    if (p.logprob) p.logprob[row] = token >= 0 ? (float)log(weight(to_float(x.x[token])) / whole) : NAN;
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_sample_tokens(const void* logits, int32_t dtype, int64_t stride, const void* uniform, const B200Sampling* how, void* token,
                                  void* logprob, int64_t rows, int64_t V, void* stream) {
  const char* who = "sample_tokens";
  if (dtype != B200_F16 && dtype != B200_BF16 && dtype != B200_F32) return fail(B200_EINVAL, "%s: dtype %d is not fp16, bf16 or fp32", who, dtype);
  if (!how) return fail(B200_EINVAL, "%s: null settings", who);
  // (an index runs past the row's end by up to a step of all threads before it is looked at: that has to fit in 31 bits)
  if (rows < 0 || V <= 0 || V >= (1LL << 31) - 65536) return fail(B200_EINVAL, "%s: bad sizes %lld x %lld", who, (long long)rows, (long long)V);
  if (rows == 0) return B200_OK;
  const unsigned size = dtype == B200_F32 ? 4 : 2;
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & (size - 1))) return fail(B200_EINVAL, "%s: logits must be non-null and aligned to their type", who);
  if (stride < V && rows > 1) return fail(B200_EINVAL, "%s: rows overlap", who);
  if (!uniform || !token) return fail(B200_EINVAL, "%s: null random numbers or tokens", who);
  if (rows > 0x7fffffffLL) return fail(B200_EINVAL, "%s: too many rows", who);
  int rc = ensure_device();
  if (rc) return rc;
  SampleParams p = {logits, static_cast<const float*>(uniform), static_cast<int*>(token), static_cast<float*>(logprob),
                    static_cast<const float*>(how->temperatures), static_cast<const int*>(how->top_ks), static_cast<const float*>(how->top_ps),
                    static_cast<const float*>(how->min_ps), stride, rows, (int)V, how->temperature, how->top_p, how->min_p, how->top_k};
  // CTAs of a row: a cluster meets three to seven times, 2000 clocks each.  us for one row of 32000 with 1, 2, 4, 8 CTAs: no filter 13.3, 10.9, 8.2,
  // 7.3; top_k 50 13.6, 12.6, 11.4, 12.3; top_p 0.9 27.7, 23.0, 18.9, 18.6.  64 such rows, top_p 0.9: 28.1, 23.5, 26.5, 48.5.  So each CTA gets 8000 entries
  // at least, and the launch no more CTAs than there are SMs.  With longer rows the passes count for more than the meetings, and two CTAs share an SM:
  // 64 rows of 128000 with 1, 2, 4 CTAs (the rule takes 4): no filter 45.9, 26.7, 23.2; top_k 50 27.4, 20.2, 22.4; top_p 0.9 81, 50, 50;
  // 100 of them with 1, 2, 4 (the rule takes 2): 46, 40, 36; 27, 30, 35; 81, 79, 74.
  int c = 1;
  while (V / (2 * c) >= 8000 && c < kMaxCluster && rows * c * 2 <= sm_count() * (V >= 65536 ? 2 : 1)) c *= 2;
  const bool many = c == 1 && rows > 2 * sm_count();
  auto launch = [&](auto kern, int threads) {
    const int64_t y = rows < 32768 ? rows : 32768;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c, (unsigned)y, (unsigned)((rows + y - 1) / y));
    cfg.blockDim = dim3((unsigned)threads);
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
  auto by_rows = [&](auto type) {
    using T = decltype(type);
    return many ? launch(sample_tokens_kernel<T, kMany>, kMany) : launch(sample_tokens_kernel<T, kFew>, kFew);
  };
  return dtype == B200_F16 ? by_rows(__half()) : dtype == B200_BF16 ? by_rows(__nv_bfloat16()) : by_rows(float());
}
