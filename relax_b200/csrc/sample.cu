// A token of every row of logits, drawn with a given random number: temperature, top-k, top-p, min-p.
//
// In the order (logit downwards, index upwards) what stays is a beginning: of top_k entries, of the fewest whose weights reach top_p of those
// of the top_k, of those with min_p of the largest one's weight.  So all that is wanted of the row is one place in that order, a border:
// the key (value, index) of the last entry that stays.  Then the token is the first one that stays whose sum of weights, in the order of the index,
// is above the random number times the whole.
//
// Which token it is hangs on comparisons of sums: with weights in 32 bits one row in eight of 32000 entries would have a border within the rounding
// of its sum.  Weights and sums are fp64: w = exp2(t), t = (x - max) log2(e) / T, by Tang's method: t = n / 64 + r, a table of 2^(j / 64)
// and Taylor's polynomial of degree 4 of e^(r ln 2) (|r| <= 1 / 128, so its rest is 3.9e-14 of the weight).  The GPU has half as many fp64 units as
// fp32 ones; ten operations an entry are a third of what its special functions would take for as many fp32 weights with a correction.
//
// Passes over the row (a CTA of 512 threads, few rows over a cluster; all passes but the first out of L2):
//   1  the maximum
//   2  with top_k or top_p: how many entries lie in each of 4096 bins of width T / 128 below the maximum
//   3  top_k: the bin with the border is known; its entries are put in order.  top_p: the counts times the bins' weights tell the bin but
//      for an error in the fourth digit; the exact sum above that bin and its neighbours, and their entries in order, find the border or say
//      on which side it lies.  Where a bin holds more entries than the list (nearly equal logits) the border is found by bisection of the keys.
//   4  the sum of what stays, a segment a warp; then the segment in which the random number falls, a vector a thread
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 4096;
constexpr float kBinsPerNat = 128.f;
constexpr int kList = 1536;                     // entries of the bins around a border
constexpr int kTable = 64;                      // 2^(j / 64)
constexpr double kLn2 = 0.6931471805599453094, kLog2e = 1.4426950408889634074;

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

// A row as vectors of 16 bytes on their own grid: its first element is element `lead` of vector 0.  What lies outside the row is -inf,
// an excluded entry.
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
  __device__ __forceinline__ void load(int j, float (&f)[N]) const {
    const int at = first(j);
    if (at >= 0 && at + N <= V) {
      const uint4 v = __ldg(vectors + j);
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
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = at + i >= 0 && at + i < V ? to_float(x[at + i]) : -INFINITY;
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_tokens_kernel(const SampleParams p) {
  constexpr int N = Vec<T>::N;
  __shared__ double sm_table[kTable];
  __shared__ int sm_bins[kBins];
  __shared__ __align__(16) u64 sm_list[kList];
  __shared__ __align__(16) u64 sm_own[kList];   // this CTA's part of the list; then the list's weights in order
  double* sm_order = reinterpret_cast<double*>(sm_own);
  __shared__ double sm_warp[kWarps], sm_sum;    // of warps, of the CTA
  __shared__ int sm_warp_n[kWarps], sm_count;
  __shared__ float sm_max;
  __shared__ int sm_index;
  __shared__ u64 sm_found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = gridDim.x, rank = blockIdx.x;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (tid < kTable) sm_table[tid] = exp2((double)tid / kTable);
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  if (row >= p.rows) return;                    // (whole clusters)
  auto meet = [&]() {                           // all threads of the row
    if (ranks > 1) {
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
  // sums over all threads of the row, in an order of their own: the same bits everywhere
  auto row_sum = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sm_warp[warp] = v;
    __syncthreads();
    double s = 0.;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sm_warp[w];
    if (ranks > 1) {
      if (tid == 0) sm_sum = s;
      meet();
      s = 0.;
      for (int r = 0; r < ranks; ++r) s += *remote(&sm_sum, r);
      meet();
    } else {
      __syncthreads();
    }
    return s;
  };

  const Row<T> x(static_cast<const T*>(p.logits) + row * p.stride, p.V);
  const int per = (x.count + ranks - 1) / ranks, begin = min(rank * per, x.count), end = min(begin + per, x.count);

  // ---- 1: the maximum, NaN where there is one --------------------------------------------------------------------------------------
  float m = -INFINITY;
#pragma unroll 4
  for (int j = begin + tid; j < end; j += kThreads) {
    float f[N];
    x.load(j, f);
#pragma unroll
    for (int i = 0; i < N; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(f[i]));
  }
  auto join = [](float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
    return a;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = join(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sm_warp[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = join(m, (float)sm_warp[w]);
  if (ranks > 1) {
    if (tid == 0) sm_max = m;
    meet();
    for (int r = 0; r < ranks; ++r) m = join(m, *remote(&sm_max, r));
  }
  __syncthreads();
  const bool writes = rank == 0 && tid == 0;
  float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
  if (!(m < INFINITY) || m == -INFINITY) {      // a NaN, an infinity, nothing that is allowed
    if (writes) {
      p.token[row] = -1;
      if (p.logprob) p.logprob[row] = m == -INFINITY ? -INFINITY : NAN;
    }
    meet();                                     // (nobody reads sm_max of a CTA that is gone)
    return;
  }
  const int want_k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float want_p = p.top_ps ? p.top_ps[row] : p.top_p, want_min = p.min_ps ? p.min_ps[row] : p.min_p;
  if (!(temperature > 0.f) || want_p <= 0.f || want_k == 1) {             // the first of the largest
    int at = 0x7fffffff;
    for (int j = begin + tid; j < end; j += kThreads) {
      float f[N];
      x.load(j, f);
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (f[i] == m) at = min(at, x.first(j) + i);
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) sm_warp_n[warp] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) at = min(at, sm_warp_n[w]);
    if (tid == 0) sm_index = at;
    meet();
    if (writes) {
      for (int r = 1; r < ranks; ++r) at = min(at, *remote(&sm_index, r));
      p.token[row] = at;
      if (p.logprob) p.logprob[row] = 0.f;
    }
    meet();
    return;
  }

  const double top = m, per_t = 1. / (double)temperature, scale = kLog2e * per_t;
  // 2^((x - max) scale); 0 below 2^-1000
  auto weight = [&](float v) {
    const double t = ((double)v - top) * (scale * kTable);
    constexpr double kMagic = 6755399441055744.;         // 1.5 * 2^52: its sum with a number has the nearest whole one in its low bits
    const double shifted = t + kMagic;
    const int n = __double2loint(shifted);
    const double r = (t - (shifted - kMagic)) * (kLn2 / kTable);
    double w = fma(r, 1. / 24., 1. / 6.);
    w = fma(w, r, 0.5);
    w = fma(w, r, 1.);
    w = fma(w, r, 1.) * sm_table[n & (kTable - 1)];
    w = __hiloint2double(__double2hiint(w) + (n >> 6) * (1 << 20), __double2loint(w));
    return t >= -1000. * kTable ? w : 0.;
  };
  const bool has_k = want_k > 0 && want_k < p.V, has_p = want_p < 1.f;
  u64 border = 0;                               // the smallest entry that stays
  if (want_min > 0.f) {                         // w >= min_p: a value, rounded up to the next fp32 number
    const double low = want_min < 1.f ? top + (double)temperature * log((double)want_min) : top;
    border = (u64)key_of(__double2float_ru(low)) << 32;
  }

  if (has_k || has_p) {
    // ---- 2: how many entries lie how far below the maximum -----------------------------------------------------------------------
    const float bins_per = fminf(kBinsPerNat / temperature, 1e30f);
    // (grows as a value falls, and so does every rounding of it)
    auto bin_of = [&](float v) { return min((int)fminf((m - v) * bins_per, (float)kBins), kBins - 1); };
    for (int i = tid; i < kBins; i += kThreads) sm_bins[i] = 0;
    __syncthreads();
#pragma unroll 2
    for (int j = begin + tid; j < end; j += kThreads) {
      float f[N];
      x.load(j, f);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (f[i] > -INFINITY) atomicAdd(&sm_bins[bin_of(f[i])], 1);
    }
    meet();
    // a thread has kBins / kThreads neighbouring bins of the whole row
    constexpr int kMine = kBins / kThreads;
    int mine[kMine], sum = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      mine[i] = 0;
      for (int r = 0; r < ranks; ++r) mine[i] += *remote(&sm_bins[tid * kMine + i], r);
      sum += mine[i];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sm_warp_n[warp] = upto;
    __syncthreads();
    int before = upto - sum, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sm_warp_n[w];
      all += sm_warp_n[w];
    }
    __syncthreads();

    // The entries of bins [from, to] that are not below `least`, of the whole row, in sm_list; false: more than it holds.
    int listed = 0;
    auto collect = [&](int from, int to, u64 least, int expected) {
      if (expected > kList) return false;
      if (tid == 0) sm_count = 0;
      __syncthreads();
      u64* own = ranks > 1 ? sm_own : sm_list;
      for (int j = begin + tid; j < end; j += kThreads) {
        float f[N];
        x.load(j, f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int bin = f[i] > -INFINITY ? bin_of(f[i]) : kBins;
          if (bin >= from && bin <= to) {
            const u64 e = entry_of(f[i], x.first(j) + i);
            if (e >= least) own[atomicAdd(&sm_count, 1)] = e;
          }
        }
      }
      meet();
      if (ranks > 1) {
        listed = 0;
        for (int r = 0; r < ranks; ++r) {
          const int n = *remote(&sm_count, r);
          const u64* other = remote(sm_own, r);
          for (int i = tid; i < n; i += kThreads) sm_list[listed + i] = other[i];
          listed += n;
        }
        meet();
      } else {
        listed = sm_count;
        __syncthreads();
      }
      return true;
    };
    // Place of an entry of the list in its order.
    auto place_of = [&](u64 e) {
      int n = 0;
      for (int i = 0; i < listed; ++i) n += sm_list[i] > e;
      return n;
    };
    // The largest entry e for which what(entries >= e), a sum over the row, reaches `goal`: by bisection, for rows that fit no list.
    auto bisect = [&](u64 least, double goal, auto what) {
      u64 lo = least, hi = ~0ull;               // what(>= lo) reaches it, what(>= hi) does not
      while (hi - lo > 1) {
        const u64 mid = lo + (hi - lo) / 2;
        double s = 0.;
        for (int j = begin + tid; j < end; j += kThreads) {
          float f[N];
          x.load(j, f);
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (f[i] > -INFINITY && entry_of(f[i], x.first(j) + i) >= mid) s += what(f[i]);
        }
        if (row_sum(s) >= goal) lo = mid; else hi = mid;
      }
      return lo;
    };

    u64 border_k = 0;
    if (has_k && want_k < all) {
      // ---- 3, top_k: the bin in which the k-th entry lies ---------------------------------------------------------------------------
      int n = before;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (n < want_k && n + mine[i] >= want_k) {
          sm_index = tid * kMine + i;
          sm_warp_n[0] = n;
          sm_warp_n[1] = mine[i];
        }
        n += mine[i];
      }
      __syncthreads();
      const int bin = sm_index, above = sm_warp_n[0], members = sm_warp_n[1];
      __syncthreads();
      if (collect(bin, bin, 0, members)) {
        for (int i = tid; i < listed; i += kThreads)
          if (place_of(sm_list[i]) == want_k - above - 1) sm_found = sm_list[i];
        __syncthreads();
        border_k = sm_found;
        __syncthreads();
      } else {
        border_k = bisect(0, (double)want_k, [](float) { return 1.; });
      }
    }
    u64 border_p = 0;
    if (has_p) {
      // ---- 3, top_p: where the counts times the bins' weights reach it -----------------------------------------------------------------
      const int most = has_k ? min(want_k, all) : all;
      double mass = 0.;
      {
        int n = before;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int c = min(mine[i], max(most - n, 0));
          mass += c * (double)exp2f(-((float)(tid * kMine + i) + 0.5f) * (1.4426950f / kBinsPerNat));
          n += mine[i];
        }
      }
      double to = mass;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, to, o);
        if (lane >= o) to += v;
      }
      if (lane == 31) sm_warp[warp] = to;
      if (tid == 0) sm_index = kBins - 1;
      __syncthreads();
      double goal = 0., below = to - mass;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) below += sm_warp[w];
        goal += sm_warp[w];
      }
      goal *= (double)want_p;
      if (below < goal && below + mass >= goal) {
        int n = before;
        double s = below;
        int at = tid * kMine + kMine - 1;
        for (int i = kMine - 1; i >= 0; --i) {  // (the first bin whose sum reaches it)
          s = below;
          n = before;
          for (int q = 0; q <= i; ++q) {
            int c = 0;
#pragma unroll
            for (int z = 0; z < kMine; ++z)
              if (z == q) c = mine[z];
            s += min(c, max(most - n, 0)) * (double)exp2f(-((float)(tid * kMine + q) + 0.5f) * (1.4426950f / kBinsPerNat));
            n += c;
          }
          if (s >= goal) at = tid * kMine + i;
        }
        sm_index = at;
      }
      __syncthreads();
      int bin = sm_index;
      __syncthreads();
      bool found = false;
      for (int attempt = 0; attempt < 16 && !found; ++attempt) {
        const int from = max(bin - 1, 0), last = min(bin + 1, kBins - 1);
        // how many entries the three bins have
        if (tid == 0) sm_count = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (tid * kMine + i >= from && tid * kMine + i <= last) atomicAdd(&sm_count, mine[i]);
        __syncthreads();
        const int members = sm_count;
        __syncthreads();
        if (!collect(from, last, border_k, members)) break;
        // the exact sums: of everything that top_k leaves, of what lies above these bins
        double s = 0., a = 0.;
        for (int j = begin + tid; j < end; j += kThreads) {
          float f[N];
          x.load(j, f);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (!(f[i] > -INFINITY) || entry_of(f[i], x.first(j) + i) < border_k) continue;
            const double w = weight(f[i]);
            s += w;
            if (bin_of(f[i]) < from) a += w;
          }
        }
        const double whole = row_sum(s), above = row_sum(a), need = (double)want_p * whole;
        if (above >= need && from > 0) {        // it lies further up
          bin = max(from - 1, 0);
          continue;
        }
        // the list in order, its sums
        for (int i = tid; i < listed; i += kThreads) {
          const u64 e = sm_list[i];
          const uint32_t k = (uint32_t)(e >> 32);
          sm_order[place_of(e)] = weight(__uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k));
        }
        __syncthreads();
        constexpr int kEach = kList / kThreads;
        double w[kEach], all_w = 0.;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          w[i] = tid * kEach + i < listed ? sm_order[tid * kEach + i] : 0.;
          all_w += w[i];
        }
        double run = all_w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += v;
        }
        if (lane == 31) sm_warp[warp] = run;
        if (tid == 0) sm_index = -1;
        __syncthreads();
        double at = above + (run - all_w), total = above;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) {
          if (q < warp) at += sm_warp[q];
          total += sm_warp[q];
        }
        // the first place whose sum reaches what is wanted (sums only grow, so it is one thread's)
        int here = -1;
        double s_at = at;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const double next = s_at + w[i];
          if (here < 0 && tid * kEach + i < listed && next >= need) here = tid * kEach + i;
          s_at = next;
        }
        if (here >= 0) atomicMin(reinterpret_cast<unsigned*>(&sm_index), (unsigned)here);
        __syncthreads();
        const int place = sm_index;
        __syncthreads();
        if (place < 0) {
          if (last == kBins - 1) {              // the sums differ in their last bits: everything stays
            found = true;
            break;
          }
          bin = min(last + 1, kBins - 1);
          continue;
        }
        for (int i = tid; i < listed; i += kThreads)
          if (place_of(sm_list[i]) == place) sm_found = sm_list[i];
        __syncthreads();
        border_p = sm_found;
        __syncthreads();
        found = true;
      }
      if (!found) {
        double s = 0.;
        for (int j = begin + tid; j < end; j += kThreads) {
          float f[N];
          x.load(j, f);
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (f[i] > -INFINITY && entry_of(f[i], x.first(j) + i) >= border_k) s += weight(f[i]);
        }
        const double need = (double)want_p * row_sum(s);
        border_p = bisect(border_k, need, weight);
      }
    }
    border = max(border, max(border_k, border_p));
  }

  // ---- 4: the sum of what stays, and where the random number falls in it -------------------------------------------------------------
  auto stays = [&](float v, int index) { return v > -INFINITY && entry_of(v, index) >= border; };
  const int share = (per + kWarps - 1) / kWarps;
  const int from = min(begin + warp * share, end), to = min(from + share, end);
  double s = 0.;
#pragma unroll 2
  for (int j = from + lane; j < to; j += 32) {
    float f[N];
    x.load(j, f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (stays(f[i], x.first(j) + i)) s += weight(f[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sm_warp[warp] = s;
  __syncthreads();
  double own = 0.;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) own += sm_warp[w];
  if (tid == 0) sm_sum = own;
  meet();
  double whole = 0., before = 0.;
  int holder = -1, last = 0;                    // the CTA in which it falls; the last one with anything that stays
  for (int r = 0; r < ranks; ++r) whole += r == rank ? own : *remote(&sm_sum, r);
  const float u = p.uniform[row];
  const double goal = u > 0.f ? fmin((double)u, 1.) * whole : 0.;
  double run = 0.;
  for (int r = 0; r < ranks; ++r) {
    const double v = r == rank ? own : *remote(&sm_sum, r);
    if (v > 0.) last = r;
    if (holder < 0 && run + v > goal) {
      holder = r;
      before = run;
    }
    run += v;
  }
  if (holder < 0) {                             // u = 1, or the sums' last bits
    holder = last;
    before = -1.;
  }
  meet();                                       // (nobody reads sm_sum of a CTA that is gone)
  if (rank != holder) return;
  int segment = -1, last_segment = 0;
  double at = before;
  for (int w = 0; w < kWarps; ++w) {
    const double v = sm_warp[w];
    if (v > 0.) last_segment = w;
    if (segment < 0 && before >= 0. && at + v > goal) segment = w;
    if (segment < 0) at += v;
  }
  const bool at_end = segment < 0;              // the last entry that stays
  if (at_end) segment = last_segment;
  const int first = min(begin + segment * share, end), behind = min(first + share, end);
  if (tid == 0) {
    sm_index = 0x7fffffff;
    sm_count = -1;
  }
  __syncthreads();
  // 512 vectors at a time, in order
  for (int base = first; base < behind; base += kThreads) {
    const int j = base + tid;
    float f[N];
    double w[N], mine = 0.;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0.;
    if (j < behind) {
      x.load(j, f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (stays(f[i], x.first(j) + i)) w[i] = weight(f[i]);
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
    if (p.logprob) p.logprob[row] = token >= 0 ? (float)(((double)to_float(x.x[token]) - top) * per_t - log(whole)) : NAN;
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
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= sm_count() && V / (2 * c) >= 2048) c *= 2;
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
  return dtype == B200_F16 ? launch(sample_tokens_kernel<__half>)
       : dtype == B200_BF16 ? launch(sample_tokens_kernel<__nv_bfloat16>) : launch(sample_tokens_kernel<float>);
}
