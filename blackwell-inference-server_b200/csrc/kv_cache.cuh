// The paged int8 KV cache's layout, shared by the kernels that write, read, move and attend to it.
//
//   k, v             int8 codes [layers][pages][heads][page][d]
//   k_scale, v_scale fp32       [layers][pages][heads][page]     value = code * scale
//   table            int32 [b][table_ld]: slot s of sequence b is row s % page of page table[b][s / page]
//
// A (page, head) block is page * d consecutive bytes.  A slot past the table's columns, or one whose
// table entry is no page of the cache, does not exist: it is not written, reads as zero and is not
// attended to.  Offsets are 64-bit throughout: a long cache passes 2^31 bytes.
#pragma once

#include "common.cuh"

namespace bw {

constexpr int kKvMaxDim = 256;   // largest head dimension
constexpr int kTreeMaxNodes = 64;  // nodes of a draft tree: one bit each in a 64-bit mask

struct KvCache {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  int64_t pages;
  int heads, page, d;
  int shift;  // page = 1 << shift, or -1
  const int* table;
  int64_t table_ld;
  int table_cols;
};

// Row index (into [pages][heads][page]) of head 0 of a slot, -1 if the slot does not exist.
__device__ __forceinline__ int64_t kv_row(const KvCache& c, int64_t b, int64_t slot) {
  if (slot < 0) return -1;
  const int64_t pi = c.shift >= 0 ? slot >> c.shift : slot / c.page;
  if (pi >= c.table_cols) return -1;
  const int64_t pg = c.table[b * c.table_ld + pi];
  if (pg < 0 || pg >= c.pages) return -1;
  return pg * c.heads * c.page + (slot - pi * c.page);
}

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

inline int page_shift(int page) {
  for (int s = 0; s < 31; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// Argument check shared by the entry points that take a cache.
int check_kv_cache(const KvCache& c, int64_t b, const char* op);

}  // namespace bw
