// Log probabilities of given tokens, the entropy, and the most likely alternatives, in one pass over the logits.
//
// With m = max x, S = sum exp(x - m), T = sum (x - m) exp(x - m) over a row x of logits:
//   log p(i) = x_i - m - ln S,   H = -sum p ln p = ln S - T / S   (both terms of H are >= 0: nothing cancels).
// A thread keeps m, S and T (in powers of two) of what it has seen and rescales S and T where m moves.  A row is
// cut into four parts, one group of eight logits a thread to each in turn; a cluster of one, two or four CTAs has a
// row, and a thread's sums of the four parts are joined first, then the threads': the order of a sum is the same
// for every cluster and every number of rows, so a row's results depend on neither.  Nor do they on where in memory the
// row starts: groups go by the logits' numbers, and a row that starts on no 16-byte boundary (every second row of an odd
// vocabulary and more) is still read by wide loads: fp32 groups by the widest that their place allows, 16-bit ones in
// 16-byte pieces, two for a group.
//
// The alternatives cost the pass itself nothing but where each thread's maximum is; their search behind it, with
// none of the next row's logits on their way, costs 9 us with one and 57 with twenty of 2047 rows of 151936, which
// take 124 without.  A thread sees every 256th group of its CTA's; the k largest logits (by value, then by lowest
// index: a total order) lie in the k threads whose maxima are largest by (value, group), for if one lay elsewhere,
// k maxima would come before it.  So the k best threads are found (a sort of 32 in each warp, merges of sorted
// lists), and only their groups are read again, one 256th of the CTA's each, from L2: lists of some 300 logits, of
// which those before the k-th maximum are candidates.
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace bw {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpTop = 32;  // alternatives at most: a list is a warp's
constexpr int kLpParts = 4;

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

// Eight logits of a group.
template <typename T>
struct LpRaw {
  uint4 w[sizeof(T) / 2];
};
// fp32, `Q` words behind a 16-byte boundary.
template <int Q>
__device__ __forceinline__ LpRaw<float> lp_words(const float* p) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
  auto two = [&](int i) { return __ldg(reinterpret_cast<const uint2*>(u + i)); };
  auto four = [&](int i) { return __ldg(reinterpret_cast<const uint4*>(u + i)); };
  if constexpr (Q == 0) {
    return {{four(0), four(4)}};
  } else if constexpr (Q == 1) {
    const uint32_t a = __ldg(u), d = __ldg(u + 7);
    const uint2 b = two(1);
    const uint4 c = four(3);
    return {{make_uint4(a, b.x, b.y, c.x), make_uint4(c.y, c.z, c.w, d)}};
  } else if constexpr (Q == 2) {
    const uint2 a = two(0), c = two(6);
    const uint4 b = four(2);
    return {{make_uint4(a.x, a.y, b.x, b.y), make_uint4(b.z, b.w, c.x, c.y)}};
  } else {
    const uint32_t a = __ldg(u), d = __ldg(u + 7);
    const uint4 b = four(1);
    const uint2 c = two(5);
    return {{make_uint4(a, b.x, b.y, b.z), make_uint4(b.w, c.x, c.y, d)}};
  }
}
// 16-bit, from the five words that they lie in: from the first's lower half on, or its upper (__byte_perm's selectors).
__device__ __forceinline__ uint4 lp_halves(const uint32_t (&x)[5], uint32_t halves) {
  return make_uint4(__byte_perm(x[0], x[1], halves), __byte_perm(x[1], x[2], halves), __byte_perm(x[2], x[3], halves),
                    __byte_perm(x[3], x[4], halves));
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

__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void lp_send(uint32_t addr, const LpSums& x) {
  st_shared_cluster_f32(addr, x.m);
  st_shared_cluster_f32(addr + 4, x.s);
  st_shared_cluster_f32(addr + 8, x.t);
}

// Steps of four groups that a thread has on their way in shared memory, and CTAs of an SM.  16-bit logits: three, 198 KB an SM,
// which registers have no room for (2047 rows of 151936: 125 us, from registers 141); CTAs of a cluster hold the others' sums,
// too, and an SM three of them.  fp32 logits have 128 bytes a thread in a step as it is, from registers (2047 rows of
// 50256: 86 us; through shared memory, rows of 50257, 112 us).
template <typename T>
struct LpRing {
  static constexpr int STAGES = sizeof(T) == 4 ? 0 : 3, CTAS = sizeof(T) == 4 ? 3 : 4;
  static constexpr int ROW = 33;  // pieces of a warp's 32 groups: one more, into which the last one's logits may reach
  static constexpr int BYTES = STAGES * kLpParts * kLpWarps * ROW * 16;
};

// A cluster of kLpParts / OWN CTAs a row.
template <typename T, int OWN>
__global__ void __launch_bounds__(kLpThreads, LpRing<T>::CTAS) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int U = kLpParts / OWN;  // groups of a part in a step
  constexpr int STAGES = LpRing<T>::STAGES;
  extern __shared__ uint4 ring[];    // [stage][group of a step][warp][LpRing::ROW]
  __shared__ unsigned long long lists[kLpWarps][32];
  __shared__ unsigned long long firsts[32];              // the k best threads
  __shared__ unsigned long long from[kLpParts][32];      // at rank 0: the CTAs' lists
  __shared__ LpSums sent[kLpParts][kLpThreads];          //            their threads' sums
  __shared__ float tops[kLpWarps];
  __shared__ float2 part[kLpWarps];
  constexpr int ctas = kLpParts / OWN, own = OWN;  // CTAs of the row, parts of this one
  const int rank = ctas > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  if (ctas > 1) cluster_arrive();
  const int64_t row = blockIdx.x / ctas;
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Group c has the logits 8 c to 8 c + 7 and is thread c % 256's of part c / 256 % 4.  The row starts `shift` logits behind a
  // 16-byte boundary.  Where a 16-bit one does, group c lies in the pieces c and c + 1 from that boundary on: pieces 1 .. hi - 1
  // lie in the row as a whole, and so do all of the groups lo .. whole - 1.  Groups before and behind those are read one by one.
  constexpr int PIECE = 16 / sizeof(T);
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (PIECE - 1);
  const bool apart = sizeof(T) == 2 && shift != 0;
  const int word = sizeof(T) == 4 ? shift : shift >> 1;  // that a group starts in, behind a boundary
  const uint32_t halves = shift & 1 ? 0x5432 : 0x3210;
  const uint4* piece = reinterpret_cast<const uint4*>(x - shift);
  const int groups = static_cast<int>((static_cast<int64_t>(a.v) + 7) >> 3);
  const int hi = static_cast<int>((static_cast<int64_t>(a.v) + shift) >> 3);
  const int lo = apart ? 1 : 0, whole = apart ? hi - 1 : a.v >> 3;  // (may be -1)
  auto load = [&](int c, float(&f)[8]) {
    if (c >= lo && c < whole && (sizeof(T) == 2 || shift == 0)) {
      LpRaw<T> raw;
      if constexpr (sizeof(T) == 4) {
        raw = lp_words<0>(x + static_cast<int64_t>(c) * 8);
      } else if (!apart) {
        raw.w[0] = __ldg(piece + c);
      } else {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(piece + c) + word;
        uint32_t y[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) y[i] = __ldg(from + i);
        raw.w[0] = lp_halves(y, halves);
      }
      lp_unpack<T>(raw, f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t i = static_cast<int64_t>(c) * 8 + e;
        f[e] = i < a.v ? lp_to_f32(x[i]) : -INFINITY;
      }
    }
  };
  const int64_t tok = tid == 0 && rank == 0 ? a.tok[row] : -1;
  const bool given = tok >= 0 && tok < a.v;
  const float x_tok = given ? lp_to_f32(x[tok]) : 0.f;

  LpSums sum[OWN];                              // of the parts
#pragma unroll
  for (int p = 0; p < OWN; ++p) sum[p] = {-INFINITY, 0.f, 0.f};
  float most = -INFINITY;                       // the thread's maximum, and the first of its groups that has it
  int best = rank * own * kLpThreads + tid;
  auto take = [&](int c, const float(&f)[8], LpSums& sum) {
    const float top = fmaxf(max3(max3(f[0], f[1], f[2]), f[3], f[4]), max3(f[5], f[6], f[7]));
    if (top > sum.m) {
      const float d = fmaxf((sum.m - top) * kLog2e, kNoWeight), w = exp2_approx(d);
      sum.t = w * (sum.t + d * sum.s);
      sum.s *= w;
      sum.m = top;
      if (top > most || (top == most && c < best)) {
        most = top;
        best = c;
      }
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
    // four groups at a time, whatever the cluster: of one part, two or four
    constexpr int step = kLpParts * kLpThreads;
    const int c0 = rank * own * kLpThreads + tid;
    auto place = [&](int n) { return n % OWN * kLpThreads + n / OWN * step; };
    float f[8];
    // Copies of the pass, for 2047 rows of 50257 in us (in brackets with groups that go by the boundaries): fp32, one for each
    // word that a row may start at 89 (87.5), two and selections 97; 16-bit, one for rows on a boundary and one for those between
    // 68 (63), selections in place of shared memory's words 73, one for each word, more code than its cache holds, 76.
    auto pass = [&](auto start, auto between) {
      constexpr int Q = decltype(start)::value;
      constexpr bool APART = decltype(between)::value;
      if constexpr (LpRing<T>::STAGES == 0) {
        for (int k = 0; c0 + k < whole; k += U * step) {
          LpRaw<T> raw[kLpParts];
#pragma unroll
          for (int n = 0; n < kLpParts; ++n) {
            const int c = c0 + k + place(n);
            if (c < whole) raw[n] = lp_words<Q>(x + static_cast<int64_t>(c) * 8);
          }
#pragma unroll
          for (int n = 0; n < kLpParts; ++n) {
            const int c = c0 + k + place(n);
            if (c < whole) {
              lp_unpack<T>(raw[n], f);
              take(c, f, sum[n % OWN]);
            }
          }
        }
      } else {
        // Each lane copies its own groups' pieces to shared memory, three steps of four ahead.  APART: a lane reads its neighbour's
        // piece, too (the last one's neighbour is an additional piece of its own), so a warp's lanes go on together.
        constexpr int ROW = APART ? LpRing<T>::ROW : 32, GROUP = kLpWarps * ROW;
        uint4* mine = ring + warp * ROW + lane;
        const int begin = APART ? c0 - lane : c0;
        auto fetch = [&](int k, int stage) {
#pragma unroll
          for (int n = 0; n < kLpParts; ++n) {
            const int c = c0 + k + place(n);
            uint4* to = mine + (stage * kLpParts + n) * GROUP;
            if ((!APART || c > 0) && c < hi) copy16_async(to, piece + c);
            if (APART && lane == 31 && c + 1 < hi) copy16_async(to + 1, piece + c + 1);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < STAGES; ++i) fetch(i * U * step, i);
        if (APART && c0 == 0) {
          load(0, f);
          take(0, f, sum[0]);
        }
        int stage = 0;
        for (int k = 0; begin + k < whole; k += U * step) {
          asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
          if (APART) __syncwarp();  // the neighbour's, too
#pragma unroll
          for (int n = 0; n < kLpParts; ++n) {
            const int c = c0 + k + place(n);
            if ((!APART || c > 0) && c < whole) {
              const uint4* from = mine + (stage * kLpParts + n) * GROUP;
              LpRaw<T> raw;
              if constexpr (APART) {
                uint32_t y[5];
#pragma unroll
                for (int i = 0; i < 5; ++i) y[i] = reinterpret_cast<const uint32_t*>(from)[word + i];
                raw.w[0] = lp_halves(y, halves);
              } else {
                raw.w[0] = from[0];
              }
              lp_unpack<T>(raw, f);
              take(c, f, sum[n % OWN]);
            }
          }
          if (APART) __syncwarp();  // read by both
          fetch(k + STAGES * U * step, stage);
          stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      }
    };
    using std::integral_constant;
    if constexpr (sizeof(T) == 4) {
      if (word == 0) pass(integral_constant<int, 0>{}, std::false_type{});
      else if (word == 1) pass(integral_constant<int, 1>{}, std::false_type{});
      else if (word == 2) pass(integral_constant<int, 2>{}, std::false_type{});
      else pass(integral_constant<int, 3>{}, std::false_type{});
    } else if (apart) {
      pass(integral_constant<int, 0>{}, std::true_type{});
    } else {
      pass(integral_constant<int, 0>{}, std::false_type{});
    }
    // the groups that the row ends in: two at most (fp32: one), each its thread's last
    if constexpr (sizeof(T) == 4) {
      for (int c = whole; c < groups; ++c) {
#pragma unroll
        for (int p = 0; p < OWN; ++p)
          if (c0 + p * kLpThreads == c % step) {
            load(c, f);
            take(c, f, sum[p]);
          }
      }
    } else {
      const int end = max(whole, lo);
#pragma unroll
      for (int p = 0; p < OWN; ++p) {
        const int c = end + ((c0 + p * kLpThreads - end) & (step - 1));
        if (c < groups) {
          load(c, f);
          take(c, f, sum[p]);
        }
      }
    }
  }
  LpSums all = sum[0];  // (0 + 1) + (2 + 3), or what the CTA has of it
  if constexpr (OWN >= 2) all = lp_join(sum[0], sum[1]);
  if constexpr (OWN == 4) all = lp_join(all, lp_join(sum[2], sum[3]));
  const bool any = rank * own * kLpThreads + tid < groups;  // the thread has a group
  unsigned long long mine = any ? lp_key(most, best) : 0ull;
  if (ctas > 1) {
    cluster_wait();  // every CTA runs: its shared memory may be written
    if (rank != 0) lp_send(mapa_shared(smem_u32(&sent[rank][tid]), 0), all);
  }
  // the k best threads of the CTA, then the CTA's k best
  unsigned long long list = 0ull;  // the warp's best so far, descending
  if (a.top > 0) {
    unsigned long long limit;  // the k-th maximum: what comes behind it is not among the k
    if (a.top == 1) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mine = lp_max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
      if (lane == 0) lists[warp][0] = mine;
      __syncthreads();
      limit = lists[lane % kLpWarps][0];
#pragma unroll
      for (int o = kLpWarps / 2; o > 0; o >>= 1) limit = lp_max(limit, __shfl_xor_sync(0xffffffffu, limit, o));
      if (tid == 0) firsts[0] = limit;
    } else {
      lp_merge_warps(lists, lp_sort(mine, lane), warp, lane);
      limit = lists[0][a.top - 1];
      if (warp == 0) firsts[lane] = lists[0][lane];
    }
    __syncthreads();
    // The k threads' groups, `each` of one at most, one a lane.  They are few: most lanes find nothing before the limit.
    const int each = (groups + kLpParts * kLpThreads - 1) / (kLpParts * kLpThreads) * own;
    for (int q0 = warp * 32; q0 < a.top * each; q0 += kLpThreads) {
      const int k = (q0 + lane) / each, j = q0 + lane - k * each;
      const unsigned long long first = k < a.top ? firsts[k] : 0ull;
      const int column = static_cast<int>((0xffffffffu - static_cast<uint32_t>(first)) % kLpThreads);
      const int c = (j / own * kLpParts + rank * own + j % own) * kLpThreads + column;
      float f[8];
      bool has = false;
      if (first != 0ull && c < groups) {
        if constexpr (sizeof(T) == 4) {
          // (the widest loads here, too: 600 rows of 50257, top 20, 47 us for 50 one by one; inside `load`, where the
          // row's last group would have them as well, registers spill)
          const T* from = x + static_cast<int64_t>(c) * 8;
          if (c >= whole) load(c, f);
          else if (word == 0) lp_unpack<T>(lp_words<0>(from), f);
          else if (word == 1) lp_unpack<T>(lp_words<1>(from), f);
          else if (word == 2) lp_unpack<T>(lp_words<2>(from), f);
          else lp_unpack<T>(lp_words<3>(from), f);
        } else {
          load(c, f);
        }
        has = lp_key(fmaxf(max3(max3(f[0], f[1], f[2]), f[3], f[4]), max3(f[5], f[6], f[7])), c) >= limit;
      }
      if (!__any_sync(0xffffffffu, has)) continue;
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const int64_t i = static_cast<int64_t>(c) * 8 + e;
        unsigned long long key = 0ull;
        if (has && i < a.v) {
          float v = f[0];
#pragma unroll
          for (int n = 1; n < 8; ++n) v = e == n ? f[n] : v;
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
    lp_merge_warps(lists, list, warp, lane);  // (at top 1, any warp may have the one)
    if (warp == 0) list = lists[0][lane];
    if (ctas > 1 && rank != 0 && warp == 0) {
      const uint32_t to = mapa_shared(smem_u32(&from[rank][lane]), 0);
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(to), "l"(list) : "memory");
    }
  }
  if (ctas > 1) {
    cluster_sync_all();  // (no CTA is written to after this)
    if (rank != 0) return;
    all = ctas == 2 ? lp_join(all, sent[1][tid]) : lp_join(lp_join(all, sent[1][tid]), lp_join(sent[2][tid], sent[3][tid]));
  }
  // the maximum of all threads, then their sums relative to it
  float top = all.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  top = tops[lane % kLpWarps];
#pragma unroll
  for (int o = kLpWarps / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  {
    const float d = fmaxf((all.m - top) * kLog2e, kNoWeight), w = exp2_approx(d);
    all.t = w * (all.t + d * all.s);
    all.s *= w;
    all.m = top;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all.s += __shfl_xor_sync(0xffffffffu, all.s, o);
    all.t += __shfl_xor_sync(0xffffffffu, all.t, o);
  }
  if (lane == 0) part[warp] = make_float2(all.s, all.t);
  __syncthreads();
  if (warp != 0) return;
  all.s = part[lane % kLpWarps].x;
  all.t = part[lane % kLpWarps].y;
#pragma unroll
  for (int o = kLpWarps / 2; o > 0; o >>= 1) {
    all.s += __shfl_xor_sync(0xffffffffu, all.s, o);
    all.t += __shfl_xor_sync(0xffffffffu, all.t, o);
  }
  const float log_s = log2f(all.s) * kLn2;
  const bool bad = !(all.s <= 3.402823466e38f), none = all.m == -INFINITY;
  if (tid == 0) {
    a.logp[row] = !given ? 0.f : (bad ? NAN : (none ? -INFINITY : (x_tok - all.m) - log_s));
    a.entropy[row] = bad ? NAN : (none ? 0.f : log_s - all.t / all.s * kLn2);
  }
  if (a.top == 0) return;
  for (int r = 1; r < ctas; ++r) list = lp_merge(list, from[r][31 - lane], lane);
  if (lane < a.top) {
    const float v = lp_value(static_cast<uint32_t>(list >> 32));
    a.top_logp[row * a.top + lane] = bad ? NAN : (v == -INFINITY ? -INFINITY : (v - all.m) - log_s);
    a.top_tok[row * a.top + lane] = bad ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(list));
  }
}

template <typename T, int OWN>
static int launch_logprobs_own(const LogprobArgs& a, int64_t rows, cudaStream_t st) {
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return check_cuda(e, "cudaGetDevice");
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(token_logprobs_kernel<T, OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         LpRing<T>::BYTES);
  });
  if (int s = check_cuda(attr_err[dev], "cudaFuncSetAttribute(token_logprobs_kernel)")) return s;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kLpParts / OWN;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3(static_cast<unsigned>(rows * (kLpParts / OWN)));
  cfg.blockDim = dim3(kLpThreads);
  cfg.dynamicSmemBytes = LpRing<T>::BYTES;
  return check_cuda(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, OWN>, a), "cudaLaunchKernelEx(token_logprobs_kernel)");
}

template <typename T>
static int launch_logprobs(const LogprobArgs& a, int64_t rows, cudaStream_t st) {
  // Long rows, and few: clusters.  A CTA costs some 5 us whatever its part of the row, the cluster's exchange 1, and one that
  // waits for a place all of that again, so the more CTAs an SM has, the longer the rows must be.  Us with one, two and four CTAs
  // a row: 8 rows of 8000 (bf16, top 5) 6.3, 7.0 and 7.2, of 32000 9.0, 8.5 and 7.8; 80 of 32000 9.4, 9.7 and 11.4; 64 of 50257
  // (fp32, top 8) 14.0, 11.4 and 10.6; 90 14.5, 12.5 and 12.6; 90 of 128256 (bf16, top 5) 21.8, 17.6 and 15.4, 111 22.3, 18.3 and
  // 22.7, 222 27.5, 23.2 and 35.5, 240 27.5, 33.3 and 37.2.
  int ctas = 1;
  if (a.v >= 16384 && rows * 4 * 25000 <= static_cast<int64_t>(num_sms()) * (a.v < 62500 ? a.v : 62500)) ctas = 4;
  else if (a.v >= 32768 && rows * 2 <= 3 * num_sms()) ctas = 2;
  if (ctas == 4) return launch_logprobs_own<T, 1>(a, rows, st);
  return ctas == 2 ? launch_logprobs_own<T, 2>(a, rows, st) : launch_logprobs_own<T, 4>(a, rows, st);
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
