// Pages and rows of a call, on the device: which pages the sequences get and give back, where every new token goes.
//
// One prefix sum over the sequences decides everything: of new tokens (the rows of the call), of pages taken, of pages given back.  Every
// CTA makes it for itself in shared memory (a few thousand numbers out of L2), then all of them write a share of the sequences, pages and rows,
// each found by a search in the sums: nothing that is written is read again.  A page taken is the free list's entry at a known place, or,
// where that place is one just given back, the entry of the sequence that gave it.  Where the results are the arguments' own memory, the CTAs are
// one cluster, which meets between the last read of a length and the first write; otherwise there are as many as the rows want.
//
// What bounds it: latency, a launch and a chain of loads, scans and searches: 64 sequences 5.6 us; 301 with 61000 rows 6, on one
// cluster of 8 CTAs 17.
#include <cuda_runtime.h>

#include <algorithm>

#include "internal.h"
#include "sm100_ptx.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxBatch = 8192;                 // sums and lengths of the sequences in shared memory: 16 bytes each
constexpr int kMaxCluster = 8;

struct PlanParams {
  int* table;
  int64_t table_stride;
  const int* lengths;
  const int* counts;
  int* free_pages;
  const int* free_count;
  int* lengths_out;
  int* starts;
  int* positions;
  long long* slots;
  int* free_count_out;
  int* status;
  int batch, pool, page_log2, rows, cluster;
  int max_tokens;
};

struct Sums {
  int64_t rows;
  int64_t taken, back;
  __device__ __forceinline__ Sums operator+(const Sums& o) const { return {rows + o.rows, taken + o.taken, back + o.back}; }
};
__device__ __forceinline__ int pages_of(int64_t tokens, int log2) { return (int)((tokens + (1 << log2) - 1) >> log2); }

__global__ void __launch_bounds__(kThreads)
paged_plan_kernel(const PlanParams p) {
  extern __shared__ int sm[];
  int* sm_row = sm;                             // [batch + 1] each: rows, pages taken, pages given back before a sequence
  int* sm_taken = sm_row + p.batch + 1;
  int* sm_back = sm_taken + p.batch + 1;
  int* sm_length = sm_back + p.batch + 1;       // [batch]
  __shared__ Sums sm_sum[kWarps];
  __shared__ int sm_bad[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = gridDim.x, rank = blockIdx.x;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int count = *p.free_count;

  Sums carry = {0, 0, 0};
  bool bad = false;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    Sums mine = {0, 0, 0};
    if (b < p.batch) {
      const int64_t length = p.lengths[b], n = p.counts[b], to = length + n;
      const bool fits = length >= 0 && length <= p.max_tokens && to >= 0 && to <= p.max_tokens;
      bad |= !fits;
      const int have = fits ? pages_of(length, p.page_log2) : 0, want = fits ? pages_of(to, p.page_log2) : 0;
      mine = {fits ? max(n, (int64_t)0) : 0, max(want - have, 0), max(have - want, 0)};
      sm_length[b] = (int)length;
    }
    Sums upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Sums v = {__shfl_up_sync(0xffffffffu, upto.rows, o), __shfl_up_sync(0xffffffffu, upto.taken, o), __shfl_up_sync(0xffffffffu, upto.back, o)};
      if (lane >= o) upto = upto + v;
    }
    if (lane == 31) sm_sum[warp] = upto;
    __syncthreads();
    Sums before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before = before + sm_sum[w];
      all = all + sm_sum[w];
    }
    if (b < p.batch) {                          // (sums that leave 31 bits are refused below, whatever the low bits say)
      sm_row[b] = (int)(before.rows + upto.rows - mine.rows);
      sm_taken[b] = (int)(before.taken + upto.taken - mine.taken);
      sm_back[b] = (int)(before.back + upto.back - mine.back);
    }
    carry = all;
    __syncthreads();
  }
  if (tid == 0) {
    sm_row[p.batch] = (int)carry.rows;
    sm_taken[p.batch] = (int)carry.taken;
    sm_back[p.batch] = (int)carry.back;
  }
  const unsigned any = __ballot_sync(0xffffffffu, bad);
  if (lane == 0) sm_bad[warp] = any != 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) bad |= sm_bad[w] != 0;
  int status = 0;
  if (bad) status = -1;
  else if (carry.rows > p.rows) status = -2;
  else if (count < 0 || count + carry.back > p.pool) status = -3;
  else if (carry.taken > count + carry.back) status = (int)(carry.taken - count - carry.back);
  const bool done = status == 0;
  // everybody has read the lengths and the count of free pages
  if (p.cluster) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }

  const int thread = rank * kThreads + tid, threads = ranks * kThreads;
  // the last sequence of those [0, batch) whose sum is not above `at`
  auto find = [&](const int* sums, int at) {
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
  };
  // page `i` of those given back: that of a sequence behind what it keeps
  auto given = [&](int i) {
    const int b = find(sm_back, i);
    const int all = sm_back[b + 1] - sm_back[b];
    return p.table[b * p.table_stride + pages_of(sm_length[b], p.page_log2) - all + (i - sm_back[b])];
  };
  const int left = count + (int)carry.back;
  auto taken = [&](int i) {
    const int at = left - 1 - i;
    return at < count ? p.free_pages[at] : given(at - count);
  };
  if (thread == 0) {
    *p.status = status;
    *p.free_count_out = done ? left - (int)carry.taken : count;
  }
  for (int b = thread; b <= p.batch; b += threads) {
    p.starts[b] = done ? sm_row[b] : 0;
    if (b == p.batch) continue;
    int n = 0;
    if (done) n = p.counts[b];
    p.lengths_out[b] = sm_length[b] + n;
  }
  for (int r = thread; r < p.rows; r += threads) {
    int position = -1;
    long long slot = -1;
    if (done && r < (int)carry.rows) {
      const int b = find(sm_row, r);
      position = sm_length[b] + (r - sm_row[b]);
      const int index = position >> p.page_log2, have = pages_of(sm_length[b], p.page_log2);
      const int page = index < have ? p.table[b * p.table_stride + index] : taken(sm_taken[b] + index - have);
      slot = ((long long)page << p.page_log2) + (position & ((1 << p.page_log2) - 1));
    }
    p.positions[r] = position;
    p.slots[r] = slot;
  }
  if (!done) return;
  for (int i = thread; i < (int)carry.taken; i += threads) {
    const int b = find(sm_taken, i);
    p.table[b * p.table_stride + pages_of(sm_length[b], p.page_log2) + (i - sm_taken[b])] = taken(i);
  }
  for (int i = thread; i < (int)carry.back; i += threads) p.free_pages[count + i] = given(i);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_paged_plan(const B200PagedPlan* a, void* stream) {
  const char* who = "paged_plan";
  if (!a) return fail(B200_EINVAL, "%s: null argument descriptor", who);
  if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128)
    return fail(B200_EINVAL, "%s: page_size is 16, 32, 64 or 128, got %d", who, a->page_size);
  if (a->batch < 0 || a->batch > kMaxBatch) return fail(B200_EINVAL, "%s: 0 to %d sequences, got %d", who, kMaxBatch, a->batch);
  if (a->table_width <= 0 || (int64_t)a->table_width * a->page_size > 0x3fffffffLL)
    return fail(B200_EINVAL, "%s: a row of the page table holds 1 to 2^30 tokens", who);
  if (a->table_stride < a->table_width && a->batch > 1) return fail(B200_EINVAL, "%s: rows of the page table overlap", who);
  if (a->pages <= 0 || a->pages > 0x7fffffffLL) return fail(B200_EINVAL, "%s: room for 1 to 2^31 - 1 free pages, got %lld", who, (long long)a->pages);
  if (a->rows < 0 || a->rows > (1 << 26)) return fail(B200_EINVAL, "%s: at most 2^26 rows, got %lld", who, (long long)a->rows);
  if (a->max_tokens < 0) return fail(B200_EINVAL, "%s: negative max_tokens", who);
  if (!a->free_count || !a->free_count_out || !a->status || !a->starts) return fail(B200_EINVAL, "%s: null count, status or starts", who);
  if (a->batch > 0 && (!a->page_table || !a->lengths || !a->counts || !a->lengths_out || !a->free_pages))
    return fail(B200_EINVAL, "%s: null table, lengths, counts or free list", who);
  if (a->rows > 0 && (!a->positions || !a->slots)) return fail(B200_EINVAL, "%s: null positions or slots", who);
  int rc = ensure_device();
  if (rc) return rc;
  PlanParams p = {};
  p.table = static_cast<int*>(a->page_table);
  p.table_stride = a->table_stride;
  p.lengths = static_cast<const int*>(a->lengths);
  p.counts = static_cast<const int*>(a->counts);
  p.free_pages = static_cast<int*>(a->free_pages);
  p.free_count = static_cast<const int*>(a->free_count);
  p.lengths_out = static_cast<int*>(a->lengths_out);
  p.starts = static_cast<int*>(a->starts);
  p.positions = static_cast<int*>(a->positions);
  p.slots = static_cast<long long*>(a->slots);
  p.free_count_out = static_cast<int*>(a->free_count_out);
  p.status = static_cast<int*>(a->status);
  p.batch = a->batch;
  p.pool = (int)a->pages;
  p.page_log2 = a->page_size == 16 ? 4 : a->page_size == 32 ? 5 : a->page_size == 64 ? 6 : 7;
  p.rows = (int)a->rows;
  p.max_tokens = a->table_width * a->page_size;
  if (a->max_tokens > 0 && a->max_tokens < p.max_tokens) p.max_tokens = (int)a->max_tokens;
  const size_t smem = (size_t)(4 * a->batch + 3) * sizeof(int);
  static SmemLimit limit;
  if ((rc = raise_smem_limit(limit, reinterpret_cast<const void*>(paged_plan_kernel), smem, who))) return rc;
  // CTAs: a thread for two rows; one alone needs no cluster.
  const bool own = a->lengths_out == a->lengths || a->free_count_out == a->free_count;
  const int c = (int)std::max<int64_t>(std::min<int64_t>((p.rows + 2 * kThreads - 1) / (2 * kThreads), own ? kMaxCluster : sm_count()), 1);
  p.cluster = own && c > 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster ? (unsigned)c : 1u;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = options().gemv_pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_plan_kernel, p);
  if (e != cudaSuccess) return fail(B200_ELAUNCH, "%s launch: %s", who, cudaGetErrorString(e));
  count_launch();
  return B200_OK;
}
