// Causal attention over whole prompts, packed one behind the other, grouped query heads.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = exp(scale q_i . k_j)   within a sequence
//
// Sequences.  offsets[0 .. b] lie on the device, so the host knows neither lengths nor how many blocks of P rows a
// sequence has.  With the rows before the first and behind the last sequence as two more segments (of zeros), segment
// i's blocks are numbered from offset_i / P + i on (whole division): ceil(length / P) of them always fit before the
// next segment's, at most one number a segment is left without a block, and n / P + b + 2 numbers are enough for all.
// Offsets are clamped to [0, n]: where they descend, results are undefined but nothing outside is read or written.
#include <stdio.h>

#include <mutex>

#include "kv_cache.cuh"

namespace bw {

struct PromptArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // strides of a token and a head
  void* o;                                     // [n, hq, d] contiguous
  const int* offsets;                          // [b + 1]
  int64_t n;
  int b, hq, hk, d;
  float scale_log2;
};

// A block of at most P rows of one segment: rows [row0, row1), its sequence's first row, and whether it is a sequence's.
struct PromptBlock {
  int64_t first, row0, row1;
  bool real;
};
__device__ __forceinline__ int64_t prompt_edge(const PromptArgs& a, int i) {  // segment i's first row
  if (i == 0) return 0;
  if (i == a.b + 2) return a.n;
  const int64_t e = a.offsets[i - 1];
  return e < 0 ? 0 : (e < a.n ? e : a.n);
}
// Block number `slot`; the last blocks of a sequence, which see most keys, come first.
template <int P>
__device__ __forceinline__ bool prompt_block(const PromptArgs& a, int64_t slot, PromptBlock& blk) {
  int lo = 0, hi = a.b + 1;  // the last segment whose numbers start at `slot` or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prompt_edge(a, mid) / P + mid <= slot) lo = mid;
    else hi = mid - 1;
  }
  const int64_t e0 = prompt_edge(a, lo), e1 = prompt_edge(a, lo + 1);
  const int64_t blocks = e1 > e0 ? (e1 - e0 + P - 1) / P : 0;
  const int64_t i = slot - (e0 / P + lo);
  if (i >= blocks) return false;
  blk.first = e0;
  blk.row0 = e0 + (blocks - 1 - i) * P;
  blk.row1 = blk.row0 + P < e1 ? blk.row0 + P : e1;
  blk.real = lo >= 1 && lo <= a.b;
  return true;
}

// ---------------------------------------------------------------------------
// any head dimension up to 256, any strides: a CTA has 16 queries of one head, its four warps four each, and 32 keys
// at a time in shared memory (lane = key for the scores, lane = element for the output)
// ---------------------------------------------------------------------------
constexpr int kRowsQ = 16, kRowsK = 32;

template <typename T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const PromptArgs a) {
  extern __shared__ float smem_f[];
  const int d = a.d, ld = d + 1;  // rows of keys start in different banks
  float* sq = smem_f;             // [16][d]
  float* sk = sq + kRowsQ * d;    // [32][d + 1]
  float* sv = sk + kRowsK * ld;   // [32][d]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  PromptBlock blk;
  if (!prompt_block<kRowsQ>(a, blockIdx.x, blk)) return;
  const int rows = static_cast<int>(blk.row1 - blk.row0);
  const int h = blockIdx.y, hk = h / (a.hq / a.hk);
  T* out = static_cast<T*>(a.o);
  if (!blk.real) {
    for (int e = threadIdx.x; e < rows * d; e += 128)
      out[((blk.row0 + e / d) * a.hq + h) * d + e % d] = from_f32<T>(0.f);
    return;
  }
  const T* q = static_cast<const T*>(a.q) + h * a.q_sh;
  const T* k = static_cast<const T*>(a.k) + hk * a.k_sh;
  const T* v = static_cast<const T*>(a.v) + hk * a.v_sh;
  for (int e = threadIdx.x; e < rows * d; e += 128)
    sq[e] = to_f32(q[(blk.row0 + e / d) * a.q_st + e % d]) * a.scale_log2;
  float o[4][kKvMaxDim / 32], m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kKvMaxDim / 32; ++i) o[r][i] = 0.f;
  }
  for (int64_t j0 = blk.first; j0 < blk.row1; j0 += kRowsK) {
    const int keys = static_cast<int>(blk.row1 - j0 < kRowsK ? blk.row1 - j0 : kRowsK);
    __syncthreads();
    for (int e = threadIdx.x; e < keys * d; e += 128) {
      const int j = e / d, c = e - j * d;
      sk[j * ld + c] = to_f32(k[(j0 + j) * a.k_st + c]);
      sv[j * d + c] = to_f32(v[(j0 + j) * a.v_st + c]);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = warp * 4 + r;
      if (row >= rows) continue;
      // keys of this tile that the query sees, one at least in a sequence's first tile
      const int64_t past = blk.row0 + row - j0 + 1;
      const int see = static_cast<int>(past < keys ? past : keys);
      if (see <= 0) continue;
      float s = -INFINITY;
      if (lane < see) {
        s = 0.f;
        for (int c = 0; c < d; ++c) s += sq[row * d + c] * sk[lane * ld + c];
      }
      float top = s;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(top, m[r]);
      const float base = top == -INFINITY ? 0.f : top;  // (scores of -inf alone: no weight)
      const float f = exp2f(m[r] - base), p = lane < see ? exp2f(s - base) : 0.f;
      m[r] = top;
      l[r] = l[r] * f + p;  // the lane's keys
#pragma unroll
      for (int i = 0; i < kKvMaxDim / 32; ++i) o[r][i] *= f;
      for (int j = 0; j < see; ++j) {
        const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
        for (int i = 0; i < kKvMaxDim / 32; ++i)
          if (lane + 32 * i < d) o[r][i] += pj * sv[j * d + lane + 32 * i];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = warp * 4 + r;
    if (row >= rows) continue;
    float sum = l[r];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < kKvMaxDim / 32; ++i)
      if (lane + 32 * i < d) out[((blk.row0 + row) * a.hq + h) * d + lane + 32 * i] = from_f32<T>(o[r][i] * inv);
  }
}

template <typename T>
static int launch_rows(const PromptArgs& a, cudaStream_t st) {
  const int smem = (kRowsQ * a.d + kRowsK * (2 * a.d + 1)) * static_cast<int>(sizeof(float));
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return check_cuda(e, "cudaGetDevice");
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(prompt_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (kRowsQ * kKvMaxDim + kRowsK * (2 * kKvMaxDim + 1)) * static_cast<int>(sizeof(float)));
  });
  if (int s = check_cuda(attr_err[dev], "cudaFuncSetAttribute(prompt_rows_kernel)")) return s;
  const dim3 grid(static_cast<unsigned>(a.n / kRowsQ + a.b + 2), static_cast<unsigned>(a.hq));
  prompt_rows_kernel<T><<<grid, 128, smem, st>>>(a);
  return check_launch("prompt_rows_kernel");
}

}  // namespace bw

extern "C" int bw_prompt_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                                   const void* v, int64_t v_st, int64_t v_sh, int dtype, void* out,
                                   const int32_t* offsets, int64_t b, int64_t n, int64_t hq, int64_t hk, int64_t d,
                                   float softmax_scale, void* stream) {
  using namespace bw;
  if (dtype != BW_DTYPE_F16 && dtype != BW_DTYPE_BF16)
    return fail(BW_ERR_INVALID_ARGUMENT, "prompt_attention: inputs must be fp16 or bf16 (dtype %d)", dtype);
  if (b < 0 || n < 0 || b > INT32_MAX / 4 || n > INT32_MAX / 4)
    return fail(BW_ERR_INVALID_ARGUMENT, "prompt_attention: need 0 <= b, n < 2^29");
  if (hk < 1 || hq < 1 || hq > 65535 || hq % hk != 0)
    return fail(BW_ERR_INVALID_ARGUMENT, "prompt_attention: query heads must be a multiple of the key heads, at most 65535");
  if (d < 1 || d > kKvMaxDim) return fail(BW_ERR_INVALID_ARGUMENT, "prompt_attention: need 1 <= d <= %d", kKvMaxDim);
  if (q_st < 0 || q_sh < 0 || k_st < 0 || k_sh < 0 || v_st < 0 || v_sh < 0)
    return fail(BW_ERR_INVALID_ARGUMENT, "prompt_attention: negative stride");
  if (n == 0) return BW_OK;
  if (!q || !k || !v || !out || !offsets) return fail(BW_ERR_INVALID_ARGUMENT, "prompt_attention: null pointer");
  if (int s = require_sm100()) return s;
  PromptArgs a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.k_st = k_st;
  a.k_sh = k_sh;
  a.v_st = v_st;
  a.v_sh = v_sh;
  a.o = out;
  a.offsets = offsets;
  a.n = n;
  a.b = static_cast<int>(b);
  a.hq = static_cast<int>(hq);
  a.hk = static_cast<int>(hk);
  a.d = static_cast<int>(d);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == BW_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(a, st) : launch_rows<__half>(a, st);
}
