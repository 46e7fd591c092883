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
// depends on a summation order, and only from a second sibling on.  That order is the same for every
// number of sequences and of CTAs, so a sequence's tokens do not depend on its batch.
#include <stdio.h>

#include <mutex>

#include "kv_cache.cuh"

namespace bw {

constexpr int kVerifyThreads = 512;
constexpr int kVerifyStages = 3;  // steps of a row that a thread has on their way
constexpr int kVerifySmem = kVerifyStages * 3 * kVerifyThreads * 16;
constexpr int kVerifyCluster = 16;  // CTAs of a cluster at most

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
  int ctas;              // of a cluster
};

// w(x) after the rejections so far at a node: with a draft distribution the recurrence over the
// normalisers z[0 .. r), without one 0 for a rejected token.
__device__ __forceinline__ float residual(float p, float q, const float* z, int r) {
  float w = p;
  for (int i = 0; i < r; ++i) w = fmaxf(__fsub_rn(w, __fmul_rn(z[i], q)), 0.f);
  return w;
}

__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// Within 2^-23 of 1 / x for the x that are trusted below.
__device__ __forceinline__ float approx_inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kTrustLow = 0x1p-60f, kTrustHigh = 0x1p60f;

// By one warp: a value into slot `index` of all CTAs of the cluster, which have it after the next
// cluster_sync_all; slots are not reused before every CTA has passed another one.
template <typename V>
__device__ __forceinline__ void cluster_share(V (*slot)[kVerifyCluster], V v, int index, int ctas) {
  if ((threadIdx.x & 31) < ctas) {
    const uint32_t at = mapa_shared(smem_u32(&(*slot)[index]), threadIdx.x & 31);
    if constexpr (sizeof(V) == 8)
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
    else
      asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(__float_as_uint(v)) : "memory");
  }
}

__device__ __forceinline__ float sum4(const float4& v) { return (v.x + v.y) + (v.z + v.w); }
__device__ __forceinline__ float sum16(const float* x) {
  const float4* v = reinterpret_cast<const float4*>(x);
  return (sum4(v[0]) + sum4(v[1])) + (sum4(v[2]) + sum4(v[3]));
}

// One cluster per sequence.  A row is cut into sixteen parts whatever the cluster's size, a warp's step to each
// in turn (so that all end together); a CTA has one part, or two neighbouring ones, whose sums it keeps apart:
// the order of a sum is then the same in both (2 % of the time below).  Every CTA walks the tree on its own:
// the probabilities of all drafted tokens at their parents are gathered at once, so a walk without a rejected
// sibling before another one reads nothing more, and only then is Z summed over the row, cluster-wide.  The
// token at the end takes one pass over the row's p, q and e.
// Few sequences are bound by three dependent reads (tree, gather, row), many by the bytes of the passes that
// the unluckiest walk makes one after another.  One sequence, a chain of 5 over 151936 tokens: 7.3 us with
// sixteen CTAs, 9.6 with eight (launch, gather and cluster barriers alone: 4.8).  32 sequences, trees of 16
// without draft probabilities: 23 us, of which the last pass 11 (39 MB) and the sums of Z 8.
// Scores are positive floats, whose bits order like them; with the token's complement below, the maximum of
// the 64-bit keys is the best score at its lowest token.
template <bool DRAFT, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_tree_kernel(const VerifyArgs a) {
  extern __shared__ float4 stages[];  // [kVerifyStages][p, q, e][thread]
  __shared__ int parent[kTreeMaxNodes];
  __shared__ int64_t tok[kTreeMaxNodes];
  __shared__ int64_t dropped[kTreeMaxNodes];
  __shared__ float pv[kTreeMaxNodes], qv[kTreeMaxNodes], uv[kTreeMaxNodes];
  __shared__ float z[kTreeMaxNodes + 1];
  __shared__ __align__(16) float red[2][kVerifyThreads / 32];
  __shared__ unsigned long long redk[kVerifyThreads / 32];
  __shared__ __align__(16) float sums[2][kVerifyCluster];
  static_assert(kVerifyThreads / 32 == 16 && kVerifyCluster == 16, "sum16");
  __shared__ unsigned long long keys[2][kVerifyCluster];
  __shared__ int walk[4];  // node, rejections, accepted nodes, next child to try (t: the walk has ended)
  const int rank = static_cast<int>(cluster_ctarank());
  const int ctas = a.ctas;
  const int64_t b = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int threads = blockDim.x;
  const int two = ctas < kVerifyCluster;  // parts of this CTA, less one
  cluster_arrive();
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
  // the first group of four tokens (the first token) of this thread, and the steps to the next ones: from an even
  // one and from an odd one, as they go through the CTA's parts in turn
  constexpr int kWidth = VEC ? 4 : 1;
  const int v0 = ((warp * kVerifyCluster + (rank << two)) * 32 + lane) * kWidth;
  const int even = (two ? 32 : threads * kVerifyCluster) * kWidth;
  const int odd = (threads * kVerifyCluster - (two ? 32 : 0)) * kWidth;
  __syncthreads();
  cluster_wait();  // every CTA runs (the wait lies behind the gather): its shared memory may be written
  // What is left of four consecutive tokens' weights after the first r rejections.
  auto rest = [&](float4& w, const float4& qw, int64_t v, int r) {
    if (DRAFT) {
      for (int i = 0; i < r; ++i) {  // (residual, of four)
        const float zi = z[i];
        w.x = fmaxf(__fsub_rn(w.x, __fmul_rn(zi, qw.x)), 0.f);
        w.y = fmaxf(__fsub_rn(w.y, __fmul_rn(zi, qw.y)), 0.f);
        w.z = fmaxf(__fsub_rn(w.z, __fmul_rn(zi, qw.z)), 0.f);
        w.w = fmaxf(__fsub_rn(w.w, __fmul_rn(zi, qw.w)), 0.f);
      }
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
  // f(four tokens of p, of q and of e, or zeros where a row is not given; the first of them; which of the
  // CTA's parts) over this thread's tokens, in order.  Each thread copies its own groups to shared memory,
  // kVerifyStages steps ahead (in registers they would be too few to cover the latency); rows that are no groups
  // of four go one by one.
  auto each = [&](const float* pr, const float* qr, const float* er, auto f) {
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (VEC) {
      int64_t ahead = v0;
      auto fetch = [&](int k, int stage) {
        const int64_t v = ahead;
        ahead += (k & 1) ? odd : even;
        if (v < a.v) {
          float4* to = stages + stage * 3 * threads + tid;
          copy16_async(to, pr + v);
          if (qr != nullptr) copy16_async(to + threads, qr + v);
          if (er != nullptr) copy16_async(to + 2 * threads, er + v);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll 1
      for (int k = 0; k < kVerifyStages; ++k) fetch(k, k);
      int stage = 0;
#pragma unroll 1
      for (int64_t v = v0, k = 0; v < a.v; v += (k++ & 1) ? odd : even) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kVerifyStages - 1) : "memory");
        const float4* from = stages + stage * 3 * threads + tid;
        const float4 w = from[0];
        const float4 qw = qr != nullptr ? from[threads] : none;
        const float4 ew = er != nullptr ? from[2 * threads] : none;
        f(w, qw, ew, v, k & two);
        fetch(k + kVerifyStages, stage);
        stage = stage + 1 == kVerifyStages ? 0 : stage + 1;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
#pragma unroll 2
      for (int64_t v = v0, k = 0; v < a.v; v += (k++ & 1) ? odd : even) {
        const float4 qw = make_float4(qr != nullptr ? __ldg(qr + v) : 0.f, 0.f, 0.f, 0.f);
        const float4 ew = make_float4(er != nullptr ? __ldg(er + v) : 0.f, 0.f, 0.f, 0.f);
        f(make_float4(__ldg(pr + v), 0.f, 0.f, 0.f), qw, ew, v, k & two);
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
    float sum[2] = {0.f, 0.f};
    each(p, q, nullptr, [&](float4 w, const float4& qw, const float4&, int64_t v, int part) {
      rest(w, qw, v, r);
      const float s = (w.x + w.y) + (w.z + w.w);
      if (part) sum[1] += s;
      else sum[0] += s;
    });
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      for (int o = 16; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      if (lane == 0) red[i][warp] = sum[i];
    }
    __syncthreads();
    if (warp <= two) cluster_share(&sums[phase & 1], sum16(red[warp]), (rank << two) + warp, ctas);
    cluster_sync_all();
    if (tid == 0) z[r] = sum16(sums[phase & 1]);
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
    auto scores = [&](auto f) {  // f(w, e, token)
      each(p, rr > 0 ? q : nullptr, e, [&](float4 w, const float4& qw, const float4& ew, int64_t v, int) {
        rest(w, qw, v, rr);
        f(w.x, ew.x, static_cast<int>(v));
        if (VEC) {
          f(w.y, ew.y, static_cast<int>(v) + 1);
          f(w.z, ew.z, static_cast<int>(v) + 2);
          f(w.w, ew.w, static_cast<int>(v) + 3);
        }
      });
    };
    // First w times an approximate 1 / e (together within 2^-22), of which a thread keeps the best and the
    // second best; then the rounded quotient of what comes within 2^-20 of the CTA's best, usually one
    // token.  A thread whose second best does, and every thread where the approximation's error is not
    // known (e or the best score outside [2^-60, 2^60]), goes through its part again with rounded
    // quotients.
    float top = 0.f, second = 0.f, top_w = 0.f, top_e = 1.f, e_min = 1.f, e_max = 1.f;
    int top_v = 0;
    scores([&](float w, float ew, int v) {
      const float s = w * approx_inverse(ew);
      e_min = fminf(e_min, ew);
      e_max = fmaxf(e_max, ew);
      second = fmaxf(second, fminf(top, s));
      if (s > top) {
        top = s;
        top_w = w;
        top_e = ew;
        top_v = v;
      }
    });
    float most = top;
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) red[0][warp] = most;
    const bool unsure = __syncthreads_or(!(e_min >= kTrustLow && e_max <= kTrustHigh));
    for (int k = 0; k < threads / 32; ++k) most = fmaxf(most, red[0][k]);
    const float near = most * (1.f - 0x1p-20f);
    if (unsure || !(most >= kTrustLow && most <= kTrustHigh) || second >= near)
      scores(score);
    else if (top >= near)
      score(top_w, top_e, top_v);
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) redk[warp] = best;
    __syncthreads();
    best = 0;
    for (int k = 0; k < threads / 32; ++k) best = redk[k] > best ? redk[k] : best;
    if (warp == 0) cluster_share(&keys[pass], best, rank, ctas);
    cluster_sync_all();
    best = 0;
    for (int k = 0; k < ctas; ++k) best = keys[pass][k] > best ? keys[pass][k] : best;
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
static int launch_verify(VerifyArgs a, int64_t b, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.dynamicSmemBytes = VEC ? kVerifySmem : 0;
  auto shape = [&](int ctas) {
    a.ctas = ctas;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    cfg.gridDim = dim3(static_cast<unsigned>(b * ctas));
  };
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  static bool wide[64];
  int dev = 0;
  if (cudaError_t err = cudaGetDevice(&dev)) return check_cuda(err, "cudaGetDevice");
  dev &= 63;
  std::call_once(once[dev], [&] {
    auto kernel = verify_tree_kernel<DRAFT, VEC>;
    attr_err[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kVerifySmem);
    shape(kVerifyCluster);
    int fit = 0;
    wide[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) == cudaSuccess && fit > 0;
    if (!wide[dev]) cudaGetLastError();
  });
  if (int s = check_cuda(attr_err[dev], "cudaFuncSetAttribute(verify_tree_kernel)")) return s;
  // Few sequences: sixteen CTAs each, where the device can place such a cluster; else two CTAs an SM.
  shape(wide[dev] && b * kVerifyCluster <= num_sms() ? kVerifyCluster : 8);
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
                  static_cast<int>(t), 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // rows of 16-byte groups: every row starts on one
  const bool vec = v % 4 == 0 && (reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft) |
                                  reinterpret_cast<uintptr_t>(sample_e)) % 16 == 0;
  if (draft != nullptr) return vec ? launch_verify<true, true>(a, b, st) : launch_verify<true, false>(a, b, st);
  return vec ? launch_verify<false, true>(a, b, st) : launch_verify<false, false>(a, b, st);
}
