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

// Launch parameters of a checked descriptor; `who` names the entry point in messages.
int paged_params(const char* who, const B200PagedCache* c, PagedParams* out);

}  // namespace b200
