// Verification of a tree of drafted tokens against the target's probabilities, from given random
// numbers, so that the tokens that come out are distributed as the target alone would draw them.
//
// At node c (the root first) with w = p_c and Z = 1, the children x_1, x_2, .. are tried in index
// order: child i is taken if u_i q(x_i) Z < w(x_i); else
//   w <- max(w - Z q_c, 0)   (no draft distribution: w(x_i) <- 0, as for q one at x_i),  Z <- sum w.
// The walk ends at a node none of whose children is taken; its token is argmax_v w(v) / e(v) with
// e exponential: an exponential race draws v with probability w(v) / Z and needs neither Z nor a
// cumulative sum.  Ties go to the lowest token; an empty residual falls back to p_c.
//
// Every product, difference and quotient is rounded separately in fp32 (no contraction); only Z
// depends on a summation order, and only from a second sibling on.
#include <stdio.h>

#include "kv_cache.cuh"

namespace bw {

constexpr int kVerifyThreads = 1024;

struct VerifyArgs {
  const float* p;        // [b, t, v]
  const float* q;        // [b, t, v] or null
  const int64_t* tok;    // [b, t]
  const int* parents;    // [b, t]
  const float* u;        // [b, t]
  const float* e;        // [b, v]
  int* n_out;            // [b]
  int* path;             // [b, t]
  int64_t* out;          // [b, t]
  int64_t v;
  int t;
};

// w(x) after the rejections so far at a node: with a draft distribution the recurrence over the
// normalisers z[0 .. r), without one 0 for a rejected token.
__device__ __forceinline__ float residual(float p, float q, const float* z, int r) {
  float w = p;
  for (int i = 0; i < r; ++i) w = fmaxf(__fsub_rn(w, __fmul_rn(z[i], q)), 0.f);
  return w;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_tree_kernel(const VerifyArgs a) {
  __shared__ int parent[kTreeMaxNodes];
  __shared__ int64_t tok[kTreeMaxNodes];
  __shared__ int64_t dropped[kTreeMaxNodes];
  __shared__ float z[kTreeMaxNodes + 1];
  __shared__ float red[32];
  __shared__ float best_s[32];
  __shared__ int64_t best_i[32];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < a.t) {
    parent[tid] = a.parents[b * a.t + tid];
    tok[tid] = a.tok[b * a.t + tid];
  }
  __syncthreads();
  int cur = 0, taken = 0, r = 0;
  if (tid == 0) z[0] = 1.f;
  __syncthreads();
  for (int i = 1; i < a.t; ++i) {
    if (parent[i] != cur) continue;
    const int64_t x = tok[i];
    bool take = false;
    if (x >= 0 && x < a.v) {
      const int64_t at = (b * a.t + cur) * a.v + x;
      float w = a.p[at], q = 1.f;
      if (a.q != nullptr) {
        q = a.q[at];
        w = residual(w, q, z, r);
      } else {
        for (int j = 0; j < r; ++j)
          if (dropped[j] == x) w = 0.f;
      }
      take = __fmul_rn(__fmul_rn(a.u[b * a.t + i], q), z[r]) < w;
    }
    __syncthreads();  // z and dropped are read before they change
    if (take) {
      if (tid == 0) a.path[b * a.t + taken] = i;
      if (tid == 0) a.out[b * a.t + taken] = x;
      cur = i;
      ++taken;
      r = 0;
      continue;
    }
    if (tid == 0) dropped[r] = x;
    __syncthreads();
    float sum = 0.f;
    const float* p = a.p + (b * a.t + cur) * a.v;
    const float* q = a.q != nullptr ? a.q + (b * a.t + cur) * a.v : nullptr;
    for (int64_t v = tid; v < a.v; v += kVerifyThreads) {
      float w = p[v];
      if (q != nullptr) {
        w = residual(w, q[v], z, r + 1);
      } else {
        for (int j = 0; j <= r; ++j)
          if (dropped[j] == v) w = 0.f;
      }
      sum += w;
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      float s = 0.f;
      for (int k = 0; k < 32; ++k) s += red[k];
      z[r + 1] = s;
    }
    ++r;
    __syncthreads();
  }
  // the token at the end of the walk
  const float* p = a.p + (b * a.t + cur) * a.v;
  const float* q = a.q != nullptr ? a.q + (b * a.t + cur) * a.v : nullptr;
  for (int pass = 0; pass < 2; ++pass) {  // second pass: the residual was empty
    float bs = -1.f;
    int64_t bi = 0;
    for (int64_t v = tid; v < a.v; v += kVerifyThreads) {
      float w = p[v];
      if (pass == 0) {
        if (q != nullptr) {
          w = residual(w, q[v], z, r);
        } else {
          for (int j = 0; j < r; ++j)
            if (dropped[j] == v) w = 0.f;
        }
      }
      if (w > 0.f) {
        const float s = __fdiv_rn(w, a.e[b * a.v + v]);
        if (s > bs) {
          bs = s;
          bi = v;
        }
      }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const float s = __shfl_xor_sync(0xffffffffu, bs, o);
      const int64_t i = __shfl_xor_sync(0xffffffffu, bi, o);
      if (s > bs || (s == bs && i < bi)) {
        bs = s;
        bi = i;
      }
    }
    if (lane == 0) {
      best_s[warp] = bs;
      best_i[warp] = bi;
    }
    __syncthreads();
    bs = best_s[0];
    bi = best_i[0];
    for (int k = 1; k < 32; ++k)
      if (best_s[k] > bs || (best_s[k] == bs && best_i[k] < bi)) {
        bs = best_s[k];
        bi = best_i[k];
      }
    __syncthreads();
    if (bs >= 0.f || pass == 1) {
      if (tid == 0) {
        a.n_out[b] = taken;
        a.out[b * a.t + taken] = bi;
        a.path[b * a.t + taken] = -1;
      }
      for (int i = taken + 1 + tid; i < a.t; i += kVerifyThreads) {
        a.path[b * a.t + i] = -1;
        a.out[b * a.t + i] = -1;
      }
      break;
    }
  }
}

}  // namespace bw

extern "C" int bw_verify_tree(const float* target, const float* draft, const int64_t* tokens, const int32_t* parents,
                              const float* accept_u, const float* sample_e, int64_t b, int64_t t, int64_t v,
                              int32_t* n_accepted, int32_t* path, int64_t* out_tokens, void* stream) {
  using namespace bw;
  if (b < 0 || b > INT32_MAX || t < 0 || t > kTreeMaxNodes || v < 1 || v > INT32_MAX)
    return fail(BW_ERR_INVALID_ARGUMENT, "verify_tree: need b >= 0, 0 <= t <= %d and v >= 1", kTreeMaxNodes);
  if (b == 0 || t == 0) return BW_OK;
  if (!target || !tokens || !parents || !accept_u || !sample_e || !n_accepted || !path || !out_tokens)
    return fail(BW_ERR_INVALID_ARGUMENT, "verify_tree: null pointer");
  if (int s = require_sm100()) return s;
  VerifyArgs a = {target, draft, tokens, parents, accept_u, sample_e, n_accepted, path, out_tokens, v,
                  static_cast<int>(t)};
  verify_tree_kernel<<<static_cast<unsigned>(b), kVerifyThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return check_launch("verify_tree_kernel");
}
