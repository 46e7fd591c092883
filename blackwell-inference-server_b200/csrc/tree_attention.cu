// Attention of a tree of drafted tokens over a paged int8 KV cache.
//
//   o_i = sum_j w_ij vs_j V_j / sum_j w_ij,   w_ij = exp(scale * ks_j * (q_i . K_j))
// over the slots j < ctx of node i's sequence and the slots ctx + n of the nodes n that i's mask
// names.  One pass over the keys with the running maximum of the scores and the running sum of the
// weights; a row that sees nothing (or only scores of -inf) gives zeros.
#include <stdio.h>

#include "kv_cache.cuh"

namespace bw {

struct AttnArgs {
  const void* q;  // [b, t, hq, d], strides in elements
  int64_t q_sb, q_st, q_sh;
  void* o;        // contiguous
  KvCache c;
  const int* ctx;                   // [b]
  const unsigned long long* mask;   // [b, t] or null: node i sees nodes 0 .. i
  const int* counts;                // [b] nodes of a sequence, or null: all t
  int64_t b;
  int t, hq;
  float scale_log2;                 // softmax scale times log2(e)
};

__device__ __forceinline__ unsigned long long low_bits(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// The nodes that node i of sequence b sees.
__device__ __forceinline__ unsigned long long node_mask(const AttnArgs& a, int64_t b, int i, int nodes) {
  const unsigned long long m = a.mask != nullptr ? a.mask[b * a.t + i] : low_bits(i + 1);
  return m & low_bits(nodes);
}

constexpr int kRowWarps = 4;

// Any head dimension and page size: one CTA per (sequence, node, query head); a warp takes every
// fourth key, lane = head dimension modulo 32.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) attn_rows_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ float sm[kRowWarps], sl[kRowWarps], so[kRowWarps][kKvMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x, i = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int d = a.c.d;
  const int hk = h / (a.hq / a.c.heads);
  int nodes = a.counts != nullptr ? a.counts[b] : a.t;
  nodes = nodes < 0 ? 0 : (nodes < a.t ? nodes : a.t);
  const int64_t ctx = a.ctx[b] > 0 ? a.ctx[b] : 0;
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + i * a.q_st + h * a.q_sh;
  float qv[kKvMaxDim / 32], o[kKvMaxDim / 32];
#pragma unroll
  for (int e = 0; e < kKvMaxDim / 32; ++e) {
    qv[e] = lane + 32 * e < d ? to_f32(q[lane + 32 * e]) * a.scale_log2 : 0.f;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const unsigned long long bits = node_mask(a, b, i, nodes);
  const int64_t keys = i < nodes ? ctx + nodes : 0;
  for (int64_t j = warp; j < keys; j += kRowWarps) {
    if (j >= ctx && !((bits >> (j - ctx)) & 1)) continue;
    const int64_t row0 = kv_row(a.c, b, j);
    if (row0 < 0) continue;
    const int64_t row = row0 + static_cast<int64_t>(hk) * a.c.page;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kKvMaxDim / 32; ++e)
      if (lane + 32 * e < d) s += qv[e] * static_cast<float>(a.c.k[row * d + lane + 32 * e]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.c.ks[row];
    if (s == -INFINITY) continue;
    if (s > m) {
      const float f = exp2f(m - s);
      m = s;
      l *= f;
#pragma unroll
      for (int e = 0; e < kKvMaxDim / 32; ++e) o[e] *= f;
    }
    const float p = exp2f(s - m);
    l += p;
    const float pv = p * a.c.vs[row];
#pragma unroll
    for (int e = 0; e < kKvMaxDim / 32; ++e)
      if (lane + 32 * e < d) o[e] += pv * static_cast<float>(a.c.v[row * d + lane + 32 * e]);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < kKvMaxDim / 32; ++e)
    if (lane + 32 * e < d) so[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float top = sm[0];
  for (int w = 1; w < kRowWarps; ++w) top = fmaxf(top, sm[w]);
  float sum = 0.f, f[kRowWarps];
  for (int w = 0; w < kRowWarps; ++w) {
    f[w] = sm[w] == -INFINITY && !(sl[w] != sl[w]) ? 0.f : exp2f(sm[w] - top);
    sum += f[w] * sl[w];
  }
  T* out = static_cast<T*>(a.o) + ((b * a.t + i) * a.hq + h) * d;
  for (int e = threadIdx.x; e < d; e += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < kRowWarps; ++w) x += f[w] != 0.f ? f[w] * so[w][e] : 0.f;
    out[e] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
  }
}

}  // namespace bw

extern "C" size_t bw_tree_attention_int8_workspace_size(int64_t b, int64_t t, int64_t hq, int64_t hk, int64_t d) {
  (void)b, (void)t, (void)hq, (void)hk, (void)d;
  return 0;
}

extern "C" size_t bw_tree_attention_int8_workspace_zeroed_bytes(int64_t b, int64_t t, int64_t hq, int64_t hk,
                                                                int64_t d) {
  (void)b, (void)t, (void)hq, (void)hk, (void)d;
  return 0;
}

extern "C" int bw_tree_attention_int8(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, void* out,
                                      const int8_t* cache_k, const int8_t* cache_v, const float* k_scale,
                                      const float* v_scale, int64_t pages, int64_t heads, int64_t page, int64_t d,
                                      const int32_t* table, int64_t table_ld, int64_t table_cols,
                                      const int32_t* ctx_lens, const uint64_t* mask, const int32_t* counts, int64_t b,
                                      int64_t t, int64_t hq, float softmax_scale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  using namespace bw;
  (void)workspace, (void)workspace_bytes;
  AttnArgs a = {};
  a.c.k = const_cast<int8_t*>(cache_k);
  a.c.v = const_cast<int8_t*>(cache_v);
  a.c.ks = const_cast<float*>(k_scale);
  a.c.vs = const_cast<float*>(v_scale);
  a.c.pages = pages;
  a.c.heads = heads > 0 && heads <= 65535 ? static_cast<int>(heads) : 0;
  a.c.page = page > 0 && page <= (1 << 24) ? static_cast<int>(page) : 0;
  a.c.d = d > 0 && d <= kKvMaxDim ? static_cast<int>(d) : 0;
  a.c.table = table;
  a.c.table_ld = table_ld;
  a.c.table_cols = table_cols >= 0 && table_cols <= INT32_MAX ? static_cast<int>(table_cols) : -1;
  if (int s = check_kv_cache(a.c, b, "tree_attention_int8")) return s;
  if (dtype != BW_DTYPE_F16 && dtype != BW_DTYPE_BF16)
    return fail(BW_ERR_INVALID_ARGUMENT, "tree_attention_int8: q must be fp16 or bf16 (dtype %d)", dtype);
  if (b < 0 || b > 65535 || t < 0 || t > kTreeMaxNodes)
    return fail(BW_ERR_INVALID_ARGUMENT, "tree_attention_int8: need 0 <= b < 65536 and 0 <= t <= %d", kTreeMaxNodes);
  if (hq < 1 || hq > 65535 || hq % a.c.heads != 0)
    return fail(BW_ERR_INVALID_ARGUMENT, "tree_attention_int8: query heads must be a multiple of the cache's heads");
  if (q_sb < 0 || q_st < 0 || q_sh < 0) return fail(BW_ERR_INVALID_ARGUMENT, "tree_attention_int8: negative stride");
  if (b == 0 || t == 0) return BW_OK;
  if (!q || !out || !ctx_lens) return fail(BW_ERR_INVALID_ARGUMENT, "tree_attention_int8: null pointer");
  if (int s = require_sm100()) return s;
  a.q = q;
  a.q_sb = q_sb;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.o = out;
  a.ctx = ctx_lens;
  a.mask = reinterpret_cast<const unsigned long long*>(mask);
  a.counts = counts;
  a.b = b;
  a.t = static_cast<int>(t);
  a.hq = static_cast<int>(hq);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(hq), static_cast<unsigned>(t), static_cast<unsigned>(b));
  if (dtype == BW_DTYPE_BF16) attn_rows_kernel<__nv_bfloat16><<<grid, 32 * kRowWarps, 0, st>>>(a);
  else attn_rows_kernel<__half><<<grid, 32 * kRowWarps, 0, st>>>(a);
  return check_launch("attn_rows_kernel");
}
