// Rotary positions for q and k, and the append of k and v to the pages of the key-value cache: for every token of the call, pairs (a, b)
// of a head become (a cos - b sin, b cos + a sin), fp32, rounded once.
//
// A block takes one token; a thread one pair of 8-value chunks (chunk c and c + rotary / 2 in the half layout, two neighbouring chunks in
// the interleaved one) of the head's rotated part, whose 8 cosines and sines it keeps while it goes over the heads, or one chunk that is
// only copied (the rest of a q or k head, v).  16 bytes a load and a store.
#include "paged_common.cuh"

namespace b200 {

namespace {

// Threads of a block; heads and copies that a thread has under way at a time.  7.9k tokens of 48 heads, 209 MB, us: 64 x 2 45.8, 128 x 1 43.1,
// 128 x 2 40.4 (5.2 TB/s; a copy of as much 32), 128 x 3 54, 192 x 2 57, 256 x 2 51.7, 512 x 2 120; 64 tokens 3.0 with 128 x 2, 2.7 with 256 x 2.
constexpr int kThreads = 128, kBatch = 2;

struct AppendParams {
  PagedParams c;
  const void* qkv;
  void* q_out;
  const float* cos_t;
  const float* sin_t;
  const int* positions;
  int64_t qkv_stride, table_rows;
  int heads, rotary;
};

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kThreads)
paged_append_kernel(const AppendParams p) {
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int kv = p.c.kv_heads, page = 1 << p.c.page_log2;
  const int row = blockIdx.x;
  const T* in = static_cast<const T*>(p.qkv) + (int64_t)row * p.qkv_stride;
  T* q = static_cast<T*>(p.q_out) + (int64_t)row * p.heads * D;
  const int half = p.rotary / 2;
  const int pairs = p.rotary / 16;              // chunk pairs of a head's rotated part
  const int c = threadIdx.x % pairs, first = threadIdx.x / pairs, step = kThreads / pairs;
  const int o0 = kInterleaved ? 16 * c : 8 * c, o1 = kInterleaved ? o0 + 8 : half + 8 * c;
  const int kept = (D - p.rotary) / 8;          // chunks of a q or k head that are not turned
  const int turned = first < step ? p.heads + kv : 0, values = kv * (D / 8), copies = values + kept * (p.heads + kv);
  T *kp = nullptr, *vp = nullptr;
  bool placed = false, known = false;
  float cs[8], sn[8];
  // The values are asked for before it is known where they go: that takes a chain of loads of its own.
  int head0 = first, copy0 = threadIdx.x;
  do {
    uint4 x[kBatch], y[kBatch], z[kBatch];
    int from[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int head = head0 + k * step, i = copy0 + k * kThreads;
      if (head < turned) {
        x[k] = *reinterpret_cast<const uint4*>(in + head * D + o0);
        y[k] = *reinterpret_cast<const uint4*>(in + head * D + o1);
      }
      from[k] = -1;
      if (i < values) {
        from[k] = (p.heads + kv) * D + i * 8;
      } else if (i < copies) {
        const int j = i - values, h = j / kept;
        from[k] = h * D + p.rotary + (j - h * kept) * 8;
      }
      if (from[k] >= 0) z[k] = *reinterpret_cast<const uint4*>(in + from[k]);
    }
    if (!known) {
      known = true;
      // the sequence of this row: the last one that starts at or before it
      int b = row;
      if (p.c.starts) {
        int lo = 0, hi = p.c.batch;             // starts[lo] <= row < starts[hi]
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (p.c.starts[mid] <= row) lo = mid; else hi = mid;
        }
        b = lo;
      }
      const Sequence s = sequence_of(p.c, b);
      const int place = row - s.first, position = s.length - s.rows + place;
      placed = position >= 0 && place >= 0 && place < s.rows;
      if (!placed) break;
      const int64_t id = page_of(p.c, b, position >> p.c.page_log2);
      const int64_t slot = (int64_t)(position & (page - 1)) * D;
      kp = static_cast<T*>(p.c.k) + id * p.c.k_stride + slot;
      vp = static_cast<T*>(p.c.v) + id * p.c.v_stride + slot;
      if (turned) {
        int64_t at = p.positions ? p.positions[row] : position;
        at = at < 0 ? 0 : at >= p.table_rows ? p.table_rows - 1 : at;
        const float4* cp = reinterpret_cast<const float4*>(p.cos_t + at * half + c * 8);
        const float4* sp = reinterpret_cast<const float4*>(p.sin_t + at * half + c * 8);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 u = cp[j], w = sp[j];
          cs[4 * j] = u.x; cs[4 * j + 1] = u.y; cs[4 * j + 2] = u.z; cs[4 * j + 3] = u.w;
          sn[4 * j] = w.x; sn[4 * j + 1] = w.y; sn[4 * j + 2] = w.z; sn[4 * j + 3] = w.w;
        }
      }
    }
    const int64_t head_step = (int64_t)page * D;
    // where element `e` of the row goes
    auto target = [&](int e) {
      const int h = e / D, o = e - h * D;
      return h < p.heads ? q + e : h < p.heads + kv ? kp + (h - p.heads) * head_step + o : vp + (h - p.heads - kv) * head_step + o;
    };
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int head = head0 + k * step;
      if (from[k] >= 0) *reinterpret_cast<uint4*>(target(from[k])) = z[k];
      if (head >= turned) continue;
      T* dst = target(head * D);
      const uint32_t xw[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, yw[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
      uint32_t xo[4], yo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = unpack2(T(), xw[j]), w = unpack2(T(), yw[j]);
        if (kInterleaved) {                     // a word is a pair: x holds pairs 0..3 of the eight, y 4..7
          xo[j] = pack2(T(), u.x * cs[j] - u.y * sn[j], u.y * cs[j] + u.x * sn[j]);
          yo[j] = pack2(T(), w.x * cs[4 + j] - w.y * sn[4 + j], w.y * cs[4 + j] + w.x * sn[4 + j]);
        } else {
          xo[j] = pack2(T(), u.x * cs[2 * j] - w.x * sn[2 * j], u.y * cs[2 * j + 1] - w.y * sn[2 * j + 1]);
          yo[j] = pack2(T(), w.x * cs[2 * j] + u.x * sn[2 * j], w.y * cs[2 * j + 1] + u.y * sn[2 * j + 1]);
        }
      }
      *reinterpret_cast<uint4*>(dst + o0) = make_uint4(xo[0], xo[1], xo[2], xo[3]);
      *reinterpret_cast<uint4*>(dst + o1) = make_uint4(yo[0], yo[1], yo[2], yo[3]);
    }
    head0 += kBatch * step;
    copy0 += kBatch * kThreads;
  } while (head0 < turned || copy0 < copies);
  if (!placed)
    for (int i = threadIdx.x; i < p.heads * D / 8; i += kThreads) reinterpret_cast<uint4*>(q)[i] = make_uint4(0, 0, 0, 0);
}

}  // namespace

int paged_params(const char* who, const B200PagedCache* c, PagedParams* out) {
  if (!c) return fail(B200_EINVAL, "%s: null cache descriptor", who);
  if (c->dtype != B200_F16 && c->dtype != B200_BF16) return fail(B200_EINVAL, "%s: dtype %d is neither fp16 nor bf16", who, c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(B200_EINVAL, "%s: head_dim is 64 or 128, got %d", who, c->head_dim);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(B200_EINVAL, "%s: page_size is 16, 32, 64 or 128, got %d", who, c->page_size);
  if (c->kv_heads <= 0 || c->kv_heads > 4096) return fail(B200_EINVAL, "%s: kv_heads in 1..4096, got %d", who, c->kv_heads);
  if (c->batch < 0 || c->tokens < 0 || c->table_width < 0 || c->max_query < 0) return fail(B200_EINVAL, "%s: negative size", who);
  if (c->batch > (1 << 20) || c->tokens > (1 << 26)) return fail(B200_EINVAL, "%s: at most 2^20 sequences and 2^26 rows", who);
  if (!c->starts && c->tokens != c->batch)
    return fail(B200_EINVAL, "%s: %lld rows of %d sequences need starts", who, (long long)c->tokens, c->batch);
  if (c->tokens > 0 && c->batch > 0) {
    if (c->pages <= 0 || c->pages > 0x7fffffffLL) return fail(B200_EINVAL, "%s: pages in 1..2^31-1, got %lld", who, (long long)c->pages);
    if (c->table_width == 0 || (int64_t)c->table_width * c->page_size > 0x3fffffffLL)
      return fail(B200_EINVAL, "%s: a row of the page table holds 1 to 2^30 tokens", who);
    const int64_t whole = (int64_t)c->kv_heads * c->page_size * c->head_dim;
    if (c->k_page_stride < whole || c->v_page_stride < whole || c->k_page_stride % 8 || c->v_page_stride % 8)
      return fail(B200_EINVAL, "%s: page strides are multiples of 8 and at least a page (%lld)", who, (long long)whole);
    if (!c->k_pages || !c->v_pages || !aligned16(c->k_pages) || !aligned16(c->v_pages))
      return fail(B200_EINVAL, "%s: the pages must be non-null and 16-byte aligned", who);
    if (!c->page_table || !c->lengths) return fail(B200_EINVAL, "%s: null page table or lengths", who);
    if (c->table_stride < c->table_width) return fail(B200_EINVAL, "%s: rows of the page table overlap", who);
  }
  out->k = c->k_pages;
  out->v = c->v_pages;
  out->k_stride = c->k_page_stride;
  out->v_stride = c->v_page_stride;
  out->table = static_cast<const int*>(c->page_table);
  out->lengths = static_cast<const int*>(c->lengths);
  out->starts = static_cast<const int*>(c->starts);
  out->table_stride = c->table_stride;
  out->tokens = c->tokens;
  out->batch = c->batch;
  out->table_width = c->table_width;
  out->pages = (int)c->pages;
  out->kv_heads = c->kv_heads;
  out->page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  return B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_paged_rope_append(const B200PagedCache* cache, const void* qkv, int64_t qkv_stride, int32_t heads, const void* cos_t,
                                      const void* sin_t, int64_t table_rows, int32_t rotary, int32_t interleaved, const void* positions,
                                      void* q_out, void* stream) {
  const char* who = "paged_rope_append";
  AppendParams p = {};
  int rc = paged_params(who, cache, &p.c);
  if (rc) return rc;
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
    return interleaved ? launch(paged_append_kernel<T, D, true>) : launch(paged_append_kernel<T, D, false>);
  };
  auto by_dim = [&](auto type) {
    return cache->head_dim == 128 ? by_layout(type, std::integral_constant<int, 128>()) : by_layout(type, std::integral_constant<int, 64>());
  };
  return cache->dtype == B200_F16 ? by_dim(__half()) : by_dim(__nv_bfloat16());
}
