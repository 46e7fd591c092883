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
constexpr int kVerifyCluster = 8;

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

// One value of each CTA of the cluster into all of them, in the CTAs' order; `slot`s are not reused before
// every CTA has passed another exchange.
template <typename V>
__device__ __forceinline__ void cluster_share(V (*slot)[kVerifyCluster], V v, int rank) {
  if (threadIdx.x < kVerifyCluster) {
    const uint32_t at = mapa_shared(smem_u32(&(*slot)[rank]), threadIdx.x);
    if constexpr (sizeof(V) == 8)
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
    else
      asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(__float_as_uint(v)) : "memory");
  }
  cluster_sync_all();
}

// One cluster per sequence, a CTA each eighth of the vocabulary.  Every CTA walks the tree on its own: the
// probabilities of all drafted tokens at their parents are gathered at once, so a walk without a rejected
// sibling before another one reads nothing more, and only then is Z summed over the row (cluster-wide, in
// one order).  The token at the end takes one pass over the row's p, q and e: bound by their bytes where
// sequences are many, by three dependent reads (tree, gather, row) where they are few.
// Scores are positive floats, whose bits order like them; with the token's complement below, the maximum of
// the 64-bit keys is the best score at its lowest token.
template <bool DRAFT, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads) verify_tree_kernel(const VerifyArgs a) {
  __shared__ int parent[kTreeMaxNodes];
  __shared__ int64_t tok[kTreeMaxNodes];
  __shared__ int64_t dropped[kTreeMaxNodes];
  __shared__ float pv[kTreeMaxNodes], qv[kTreeMaxNodes], uv[kTreeMaxNodes];
  __shared__ float z[kTreeMaxNodes + 1];
  __shared__ float red[kVerifyThreads / 32];
  __shared__ unsigned long long redk[kVerifyThreads / 32];
  __shared__ float sums[2][kVerifyCluster];
  __shared__ unsigned long long keys[2][kVerifyCluster];
  __shared__ int walk[4];  // node, rejections, accepted nodes, next child to try (t: the walk has ended)
  const int rank = static_cast<int>(cluster_ctarank());
  const int64_t b = blockIdx.x / kVerifyCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int threads = blockDim.x;
  if (tid < a.t) {
    const int p = a.parents[b * a.t + tid];
    const int64_t x = a.tok[b * a.t + tid];
    parent[tid] = p;
    tok[tid] = x;
    uv[tid] = a.u[b * a.t + tid];
    const bool in = tid > 0 && p >= 0 && p < tid && x >= 0 && x < a.v;
    const int64_t at = in ? (b * a.t + p) * a.v + x : 0;
    pv[tid] = in ? a.p[at] : 0.f;
    if (!in) uv[tid] = INFINITY;  // a token that is none is never taken
    qv[tid] = in && DRAFT ? a.q[at] : 1.f;
    z[0] = 1.f;
  }
  if (tid < 4) walk[tid] = tid == 3 ? 1 : 0;
  // this CTA's part of a row, whole groups of four
  const int64_t per = ((a.v + kVerifyCluster - 1) / kVerifyCluster + 3) / 4 * 4;
  const int64_t v0 = min(per * rank, a.v), v1 = min(v0 + per, a.v);
  __syncthreads();
  // What is left of four consecutive tokens' weights after the first r rejections.
  auto rest = [&](float4& w, const float4& qw, int64_t v, int r) {
    if (DRAFT) {
      w = make_float4(residual(w.x, qw.x, z, r), residual(w.y, qw.y, z, r), residual(w.z, qw.z, z, r),
                      residual(w.w, qw.w, z, r));
    } else {
      for (int j = 0; j < r; ++j) {
        const int64_t off = dropped[j] - v;
        if (off == 0) w.x = 0.f;
        if (VEC && off == 1) w.y = 0.f;
        if (VEC && off == 2) w.z = 0.f;
        if (VEC && off == 3) w.w = 0.f;
      }
    }
  };
  int phase = 0;
#pragma unroll 1
  for (;;) {
    // walk until it ends or a normaliser is missing
    if (tid == 0) {
      int cur = walk[0], r = walk[1], taken = walk[2], i = walk[3];
      bool sum = false;
      for (; i < a.t && !sum; ++i) {
        if (parent[i] != cur) continue;
        const int64_t x = tok[i];
        float w = pv[i];
        if (DRAFT) {
          w = residual(w, qv[i], z, r);
        } else {
          for (int j = 0; j < r; ++j)
            if (dropped[j] == x) w = 0.f;
        }
        if (__fmul_rn(__fmul_rn(uv[i], qv[i]), z[r]) < w) {
          if (rank == 0) {
            a.path[b * a.t + taken] = i;
            a.out[b * a.t + taken] = x;
          }
          ++taken;
          cur = i;
          r = 0;
          continue;
        }
        dropped[r++] = x;
        for (int k = i + 1; k < a.t && !sum; ++k) sum = parent[k] == cur;  // another sibling needs Z
      }
      walk[0] = cur;
      walk[1] = r;
      walk[2] = taken;
      walk[3] = sum ? i : kTreeMaxNodes;
    }
    __syncthreads();
    if (walk[3] >= kTreeMaxNodes) break;
    const int cur = walk[0], r = walk[1];
    const float* p = a.p + (b * a.t + cur) * a.v;
    const float* q = DRAFT ? a.q + (b * a.t + cur) * a.v : nullptr;
    float sum = 0.f;
    if constexpr (VEC) {
#pragma unroll 4
      for (int64_t v = v0 + tid * 4; v < v1; v += threads * 4) {
        float4 w = __ldg(reinterpret_cast<const float4*>(p + v));
        const float4 qw = DRAFT ? __ldg(reinterpret_cast<const float4*>(q + v)) : make_float4(0.f, 0.f, 0.f, 0.f);
        rest(w, qw, v, r);
        sum += (w.x + w.y) + (w.z + w.w);
      }
    } else {
#pragma unroll 4
      for (int64_t v = v0 + tid; v < v1; v += threads) {
        float4 w = make_float4(__ldg(p + v), 0.f, 0.f, 0.f);
        rest(w, make_float4(DRAFT ? __ldg(q + v) : 0.f, 0.f, 0.f, 0.f), v, r);
        sum += w.x;
      }
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    sum = 0.f;
    for (int k = 0; k < threads / 32; ++k) sum += red[k];
    cluster_share(&sums[phase & 1], sum, rank);
    if (tid == 0) {
      float s = 0.f;
      for (int k = 0; k < kVerifyCluster; ++k) s += sums[phase & 1][k];
      z[r] = s;
    }
    ++phase;
    __syncthreads();
  }
  const int cur = walk[0], r = walk[1], taken = walk[2];
  const float* p = a.p + (b * a.t + cur) * a.v;
  const float* q = DRAFT ? a.q + (b * a.t + cur) * a.v : nullptr;
  const float* e = a.e + b * a.v;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // second pass: the residual was empty
    unsigned long long best = 0;  // no candidate
    auto score = [&](float w, float ew, int64_t v) {
      if (w > 0.f) {
        const float s = __fdiv_rn(w, ew);
        const unsigned long long key =
            (static_cast<unsigned long long>(__float_as_uint(s)) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
        if (s >= 0.f && key > best) best = key;
      }
    };
    const int rr = pass == 0 ? r : 0;
    if constexpr (VEC) {
#pragma unroll 4
      for (int64_t v = v0 + tid * 4; v < v1; v += threads * 4) {
        float4 w = __ldg(reinterpret_cast<const float4*>(p + v));
        const float4 ew = __ldg(reinterpret_cast<const float4*>(e + v));
        const float4 qw = DRAFT && rr > 0 ? __ldg(reinterpret_cast<const float4*>(q + v)) : make_float4(0.f, 0.f, 0.f, 0.f);
        rest(w, qw, v, rr);
        score(w.x, ew.x, v);
        score(w.y, ew.y, v + 1);
        score(w.z, ew.z, v + 2);
        score(w.w, ew.w, v + 3);
      }
    } else {
#pragma unroll 4
      for (int64_t v = v0 + tid; v < v1; v += threads) {
        float4 w = make_float4(__ldg(p + v), 0.f, 0.f, 0.f);
        const float ew = __ldg(e + v);
        rest(w, make_float4(DRAFT && rr > 0 ? __ldg(q + v) : 0.f, 0.f, 0.f, 0.f), v, rr);
        score(w.x, ew, v);
      }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) redk[warp] = best;
    __syncthreads();
    best = 0;
    for (int k = 0; k < threads / 32; ++k) best = redk[k] > best ? redk[k] : best;
    cluster_share(&keys[pass], best, rank);
    best = 0;
    for (int k = 0; k < kVerifyCluster; ++k) best = keys[pass][k] > best ? keys[pass][k] : best;
    if (best == 0 && pass == 0) continue;
    if (rank == 0) {
      if (tid == 0) {
        a.n_out[b] = taken;
        a.out[b * a.t + taken] = best == 0 ? 0 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(best));
        a.path[b * a.t + taken] = -1;
      }
      for (int i = taken + 1 + tid; i < a.t; i += threads) {
        a.path[b * a.t + i] = -1;
        a.out[b * a.t + i] = -1;
      }
    }
    break;
  }
  cluster_sync_all();  // no CTA leaves while another may still write its shared memory
}

template <bool DRAFT, bool VEC>
static int launch_verify(const VerifyArgs& a, int64_t b, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(b * kVerifyCluster));
  // one CTA an SM while there is an SM for each, two smaller ones where there are more
  cfg.blockDim = dim3(b * kVerifyCluster <= num_sms() ? kVerifyThreads : kVerifyThreads / 2);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kVerifyCluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, verify_tree_kernel<DRAFT, VEC>, a), "cudaLaunchKernelEx(verify_tree_kernel)");
}

}  // namespace bw

extern "C" int bw_verify_tree(const float* target, const float* draft, const int64_t* tokens, const int32_t* parents,
                              const float* accept_u, const float* sample_e, int64_t b, int64_t t, int64_t v,
                              int32_t* n_accepted, int32_t* path, int64_t* out_tokens, void* stream) {
  using namespace bw;
  if (b < 0 || b > INT32_MAX / kVerifyCluster || t < 0 || t > kTreeMaxNodes || v < 1 || v > INT32_MAX)
    return fail(BW_ERR_INVALID_ARGUMENT, "verify_tree: need b >= 0, 0 <= t <= %d and v >= 1", kTreeMaxNodes);
  if (b == 0 || t == 0) return BW_OK;
  if (!target || !tokens || !parents || !accept_u || !sample_e || !n_accepted || !path || !out_tokens)
    return fail(BW_ERR_INVALID_ARGUMENT, "verify_tree: null pointer");
  if (int s = require_sm100()) return s;
  VerifyArgs a = {target, draft, tokens, parents, accept_u, sample_e, n_accepted, path, out_tokens, v,
                  static_cast<int>(t)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // rows of 16-byte groups: every row starts on one
  const bool vec = v % 4 == 0 && (reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft) |
                                  reinterpret_cast<uintptr_t>(sample_e)) % 16 == 0;
  if (draft != nullptr) return vec ? launch_verify<true, true>(a, b, st) : launch_verify<true, false>(a, b, st);
  return vec ? launch_verify<false, true>(a, b, st) : launch_verify<false, false>(a, b, st);
}
