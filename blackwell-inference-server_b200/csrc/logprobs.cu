// Log probabilities of given tokens, the entropy, and the most likely alternatives, in one pass over the logits.
//
// With m = max x, S = sum exp(x - m), T = sum (x - m) exp(x - m) over a row x of logits:
//   log p(i) = x_i - m - ln S,   H = -sum p ln p = ln S - T / S   (both terms of H are >= 0: nothing cancels).
// A thread keeps m, S and T (in powers of two) of what it has seen and rescales S and T where m moves; the joins
// are made in one order, so results do not depend on timing.
//
// The alternatives cost the pass nothing but where each thread's maximum is.  A thread sees every 512th group of
// eight logits; the k largest logits (by value, then by lowest index: a total order) lie in the k threads whose
// maxima are largest by (value, group), for if one lay elsewhere, k maxima would come before it.  So the k best
// threads are found (a sort of 32 in each warp, merges of sorted lists), and only their groups are read again,
// one 512th of the row each, from L2: k lists of some 300 logits, of which those before the k-th maximum are candidates.
#include <type_traits>

#include "common.cuh"

namespace bw {

constexpr int kLpThreads = 512;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpTop = 32;  // alternatives at most: a list is a warp's

struct LogprobArgs {
  const void* x;        // [rows, v], row stride ld
  int64_t ld;
  const int64_t* tok;   // [rows]
  float* logp;          // [rows]
  float* entropy;       // [rows]
  float* top_logp;      // [rows, top]
  int64_t* top_tok;     // [rows, top]
  int v, top;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNoWeight = -200.f;  // a power of two that is 0, finite: 0 times it is 0

// What a part of a row comes to.  m = -inf: nothing seen but -inf.
struct LpSums {
  float m, s, t;
};
__device__ __forceinline__ LpSums lp_join(const LpSums& a, const LpSums& b) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf((a.m - m) * kLog2e, kNoWeight), db = fmaxf((b.m - m) * kLog2e, kNoWeight);
  const float fa = exp2_approx(da), fb = exp2_approx(db);
  return {m, fa * a.s + fb * b.s, fa * (a.t + da * a.s) + fb * (b.t + db * b.s)};
}

// Keys order like (value, lowest index): -0 is 0.
__device__ __forceinline__ uint32_t lp_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t u) {
  return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ unsigned long long lp_key(float x, uint32_t index) {
  return (static_cast<unsigned long long>(lp_order(x)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ unsigned long long lp_max(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long lp_min(unsigned long long a, unsigned long long b) { return a > b ? b : a; }

// A warp's 32 keys in descending order: a bitonic network (Batcher 1968).
__device__ __forceinline__ unsigned long long lp_sort(unsigned long long x, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, j);
      x = ((lane & j) == 0) == ((lane & k) == 0) ? lp_max(x, y) : lp_min(x, y);
    }
  }
  return x;
}
// The 32 largest of two descending lists, descending; b in reverse.
__device__ __forceinline__ unsigned long long lp_merge(unsigned long long a, unsigned long long b_reversed, int lane) {
  unsigned long long x = lp_max(a, b_reversed);
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, j);
    x = (lane & j) == 0 ? lp_max(x, y) : lp_min(x, y);
  }
  return x;
}
// The 32 largest of the warps' descending lists into lists[0], by all threads.
__device__ __forceinline__ void lp_merge_warps(unsigned long long (*lists)[32], unsigned long long mine, int warp, int lane) {
  lists[warp][lane] = mine;
  __syncthreads();
#pragma unroll
  for (int n = kLpWarps / 2; n > 0; n >>= 1) {
    if (warp < n) lists[warp][lane] = mine = lp_merge(mine, lists[warp + n][31 - lane], lane);
    __syncthreads();
  }
}

// Eight logits of a group that lies in the row and on 16-byte boundaries.
template <typename T>
struct LpRaw {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ LpRaw<T> lp_fetch(const T* group) {
  LpRaw<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(group) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void lp_unpack(const LpRaw<T>& r, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
}
__device__ __forceinline__ float lp_to_f32(float x) { return x; }
__device__ __forceinline__ float lp_to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float lp_to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// One CTA a row.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int U = 8 / sizeof(T);  // groups of a thread on their way
  __shared__ unsigned long long lists[kLpWarps][32];
  __shared__ LpSums part[kLpWarps];
  __shared__ LpSums whole;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Groups lie on 32-byte (16-bit types: 16-byte) boundaries of memory: index i of group c is 8 c - shift + i.
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T) & 7);
  const int groups = static_cast<int>((static_cast<int64_t>(a.v) + shift + 7) >> 3);
  const int whole_lo = shift ? 1 : 0, whole_hi = static_cast<int>((static_cast<int64_t>(a.v) + shift) >> 3);
  auto at = [&](int c) { return x + (static_cast<int64_t>(c) * 8 - shift); };
  auto load = [&](int c, float(&f)[8]) {
    if (c >= whole_lo && c < whole_hi) {
      lp_unpack<T>(lp_fetch<T>(at(c)), f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t i = static_cast<int64_t>(c) * 8 - shift + e;
        f[e] = i >= 0 && i < a.v ? lp_to_f32(x[i]) : -INFINITY;
      }
    }
  };
  const int64_t tok = tid == 0 ? a.tok[row] : -1;
  const bool given = tok >= 0 && tok < a.v;
  const float x_tok = given ? lp_to_f32(x[tok]) : 0.f;

  LpSums sum = {-INFINITY, 0.f, 0.f};
  int best = tid;  // the first group with the thread's maximum
  auto take = [&](int c, const float(&f)[8]) {
    float top = fmaxf(f[0], f[1]);
#pragma unroll
    for (int e = 2; e < 8; ++e) top = fmaxf(top, f[e]);
    if (top > sum.m) {
      const float d = fmaxf((sum.m - top) * kLog2e, kNoWeight), w = exp2_approx(d);
      sum.t = w * (sum.t + d * sum.s);
      sum.s *= w;
      sum.m = top;
      best = c;
    }
    const float m = sum.m == -INFINITY ? 0.f : sum.m;  // (-inf alone weighs nothing)
    const float2 m2 = make_float2(-m, -m), c2 = make_float2(kLog2e, kLog2e);
    float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      // the difference first: times log2 e a 16-bit type's lowest value would pass the range
      const float2 z = __fmul2_rn(__fadd2_rn(make_float2(f[e], f[e + 1]), m2), c2);
      const float2 w = make_float2(exp2_approx(z.x), exp2_approx(z.y));
      s = __fadd2_rn(s, w);
      t = __ffma2_rn(w, make_float2(fmaxf(z.x, kNoWeight), fmaxf(z.y, kNoWeight)), t);
    }
    sum.s += s.x + s.y;
    sum.t += t.x + t.y;
  };
  {
    float f[8];
    if (tid == 0 && shift) {
      load(0, f);
      take(0, f);
    }
    int c = tid < whole_lo ? tid + kLpThreads : tid;
    for (; c < whole_hi; c += U * kLpThreads) {
      LpRaw<T> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * kLpThreads < whole_hi) raw[u] = lp_fetch<T>(at(c + u * kLpThreads));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * kLpThreads < whole_hi) {
          lp_unpack<T>(raw[u], f);
          take(c + u * kLpThreads, f);
        }
      }
    }
    const int last = groups - 1;  // a group that the row ends in
    if (last >= whole_hi && (last > 0 || !shift) && tid == last % kLpThreads) {
      load(last, f);
      take(last, f);
    }
  }
  const unsigned long long mine = tid < groups ? lp_key(sum.m, best) : 0ull;  // 0: a thread without groups
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSums other;
    other.m = __shfl_xor_sync(0xffffffffu, sum.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, sum.s, o);
    other.t = __shfl_xor_sync(0xffffffffu, sum.t, o);
    sum = lane & o ? lp_join(other, sum) : lp_join(sum, other);
  }
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    LpSums all = part[0];
#pragma unroll
    for (int w = 1; w < kLpWarps; ++w) all = lp_join(all, part[w]);
    whole = all;
    const float log_s = log2f(all.s) * kLn2;
    const bool bad = !(all.s <= 3.402823466e38f), none = all.m == -INFINITY;
    a.logp[row] = !given ? 0.f : (bad ? NAN : (none ? -INFINITY : (x_tok - all.m) - log_s));
    a.entropy[row] = bad ? NAN : (none ? 0.f : log_s - all.t / all.s * kLn2);
  }
  if (a.top == 0) return;
  lp_merge_warps(lists, lp_sort(mine, lane), warp, lane);
  const unsigned long long limit = lists[0][a.top - 1];  // the k-th maximum: what comes behind it is not among the k
  unsigned long long list = 0ull;                        // the warp's best so far, descending
  unsigned long long first[2];                           // this warp's threads to read again: the warp-th and so on
  static_assert(kLpTop <= 2 * kLpWarps, "two a warp");
#pragma unroll
  for (int k = 0; k < 2; ++k) first[k] = warp + k * kLpWarps < a.top ? lists[0][warp + k * kLpWarps] : 0ull;
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    if (first[k] == 0ull) break;
    const int column = static_cast<int>((0xffffffffu - static_cast<uint32_t>(first[k])) % kLpThreads);
    for (int c0 = column; c0 < groups; c0 += 32 * kLpThreads) {
      const int c = c0 + lane * kLpThreads;
      float f[8];
      if (c < groups) load(c, f);
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const int64_t i = static_cast<int64_t>(c) * 8 - shift + e;
        unsigned long long key = 0ull;
        if (c < groups && i >= 0 && i < a.v) {
          float v = f[0];
#pragma unroll
          for (int j = 1; j < 8; ++j) v = e == j ? f[j] : v;
          if (lp_key(v, c) >= limit) key = lp_key(v, static_cast<uint32_t>(i));
        }
        unsigned todo = __ballot_sync(0xffffffffu, key > __shfl_sync(0xffffffffu, list, 31));
        while (todo) {
          const unsigned long long in = __shfl_sync(0xffffffffu, key, __ffs(todo) - 1);
          todo &= todo - 1;
          const int place = __popc(__ballot_sync(0xffffffffu, list > in));
          const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
          if (lane >= place) list = lane == place ? in : up;
        }
      }
    }
  }
  lp_merge_warps(lists, list, warp, lane);
  if (tid < a.top) {
    const unsigned long long key = lists[0][tid];
    const LpSums all = whole;
    const bool bad = !(all.s <= 3.402823466e38f);
    const float log_s = log2f(all.s) * kLn2;
    const float v = lp_value(static_cast<uint32_t>(key >> 32));
    a.top_logp[row * a.top + tid] = bad ? NAN : (v == -INFINITY ? -INFINITY : (v - all.m) - log_s);
    a.top_tok[row * a.top + tid] = bad ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
  }
}

template <typename T>
static int launch_logprobs(const LogprobArgs& a, int64_t rows, cudaStream_t st) {
  token_logprobs_kernel<T><<<static_cast<unsigned>(rows), kLpThreads, 0, st>>>(a);
  return check_launch("token_logprobs_kernel");
}

}  // namespace bw

extern "C" int bw_token_logprobs(const void* logits, int dtype, int64_t ld, const int64_t* tokens, int64_t rows, int64_t v,
                                 int64_t top, float* logprobs, float* entropy, float* top_logprobs, int64_t* top_tokens,
                                 void* stream) {
  using namespace bw;
  if (dtype != BW_DTYPE_F16 && dtype != BW_DTYPE_BF16 && dtype != BW_DTYPE_F32)
    return fail(BW_ERR_INVALID_ARGUMENT, "token_logprobs: logits must be fp16, bf16 or fp32 (dtype %d)", dtype);
  if (rows < 0 || rows > INT32_MAX || v < 1 || v > INT32_MAX - 16)
    return fail(BW_ERR_INVALID_ARGUMENT, "token_logprobs: need 0 <= rows < 2^31 and 1 <= v < 2^31 - 16");
  if (ld < 0) return fail(BW_ERR_INVALID_ARGUMENT, "token_logprobs: negative row stride");
  if (top < 0 || top > kLpTop || top > v)
    return fail(BW_ERR_INVALID_ARGUMENT, "token_logprobs: need 0 <= top <= %d and top <= v", kLpTop);
  if (rows == 0) return BW_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
    return fail(BW_ERR_INVALID_ARGUMENT, "token_logprobs: null pointer");
  if (int s = require_sm100()) return s;
  LogprobArgs a = {logits, ld, tokens, logprobs, entropy, top_logprobs, top_tokens, static_cast<int>(v),
                   static_cast<int>(top)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == BW_DTYPE_F32) return launch_logprobs<float>(a, rows, st);
  return dtype == BW_DTYPE_BF16 ? launch_logprobs<__nv_bfloat16>(a, rows, st) : launch_logprobs<__half>(a, rows, st);
}
