// Attention of a tree of drafted tokens over a paged int8 KV cache.
//
//   o_i = sum_j w_ij vs_j V_j / sum_j w_ij,   w_ij = exp(scale * ks_j * (q_i . K_j))
// over the slots j < ctx of node i's sequence and the slots ctx + n of the nodes n that i's mask
// names.  One pass over the keys with the running maximum of the scores and the running sum of the
// weights; a row that sees nothing (or only scores of -inf) gives zeros.
#include <stdio.h>

#include <mutex>
#include <type_traits>

#define BW_WHOLE_PROGRAM
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

// ---------------------------------------------------------------------------
// tensor-core kernel (head dimensions 64 and 128)
//
// A tile is 128 slots of one sequence and key head; the R query rows of a CTA are the (node, query
// head of the group) pairs that read that head.  Both products put the 128-row side on the cache, so
// one query row costs the tensor core no more than sixteen:
//   S^T [128 slots x R]  = K [128 x D] (TMEM, dequantised) . Q^T (shared memory)
//   O^T [D x 2R]        += V^T [D x 128] (shared memory, dequantised) . [P_hi | P_lo] [128 x 2R]
// Codes are exact in 16 bits, so the products see the cache's values without a rounding; the scales
// ks_j and vs_j multiply the scores and the weights in fp32.  A weight w vs_j goes in as the sum of
// two bf16 numbers (hi = bf16(x), lo = bf16(x - hi), 2^-17 of x left out): fp16 would be one number
// but cannot hold w vs_j for every scale, one bf16 alone loses 2^-9.
//
// Softmax: one thread holds one slot's scores, so the exponentials need no exchange; what is shared is
// each row's reference m.  m moves only when a score exceeds it by more than 8 (in powers of two): the
// warps vote while they work out the weights, and only if one has such a score are the row maxima taken
// over the 128 slots, the sums l and the accumulators rescaled.  Weights stay under 2^8, sums and
// accumulators are fp32.
//
// Work: the (sequence, key head, tile) units, laid end to end, are split evenly over the CTAs, so
// ragged lengths balance; with more rows than R, neighbouring CTAs take the row blocks of one range
// at the same time, and the second reads the cache from L2.  A (sequence, head) cut by a range end
// is joined by its last CTA (a ticket) from the pieces in the workspace, in range order, so results
// do not depend on timing.
//
// One CTA per SM, five warpgroups.  Warps 0 and 3: TMA of K and of V (one box per page), scales, each
// segment's Q and row masks; warp 0 also watches the time for all waits.  Warps 1 and 2 issue K.Q and V.P.
// 4-7 dequantise K into TMEM (thread = slot), 8-11 V into shared memory, 12-15 and 16-19 are the two softmax
// groups.
//
// What bounds it (one B200, D = 128, bf16, long contexts): with 16 rows the two dequantisers' issue slots,
// 1.05 us a tile of 32 KB in every SM, 4.7 TB/s (fp16, whose conversion has five instructions for four codes
// where bf16 has nine: 0.87 us, 5.7 TB/s); with 64 rows the softmax groups, 1.55 us a tile, 400 TFLOP/s;
// with short contexts a segment's start and end, under 3 us together.  One token over 1k slots: 12 us, of
// which 1 from launch to the first barrier, 2 to the first tile, 1.5 from scores to weights, 1.4 the ticket
// (timed one by one; the rest was not).
// Measured and not kept: 64 rows in alternate tiles, whose scores are then fetched twice (a sixth slower on a
// tree of 64 nodes over 128k slots); row blocks of equal height (690 us for 618 there: branches between the
// columns cost more than the columns); a segment's end put off into the next one's first tiles (125 us for
// 116 on 64 x 4k).
// ---------------------------------------------------------------------------
constexpr int kTile = 128;
constexpr int kAttnThreads = 20 * 32;
// Registers of a thread of the five warpgroups after setmaxnreg: their sum is five times the 96 that
// a thread of 640 has at launch.
constexpr int kRegsIssue = 72, kRegsK = 80, kRegsV = 72, kRegsSoft = 128;
static_assert(kRegsIssue + kRegsK + kRegsV + 2 * kRegsSoft == 5 * 96, "register split");
constexpr int kScaleStages = 4;   // tiles whose scales are on their way or in use
constexpr float kLowest = -3.0e38f;  // a row's reference before any score: finite, so differences are
constexpr int kAttnMaxBatch = 512;  // sequences of one launch (their unit ranges lie in shared memory)
// Tickets, two per CTA, in a prefix of one size for every shape: calls of different shapes share a workspace
// whose prefix is zeroed once.  A grid that it cannot hold (more than 32768 rows) takes attn_rows_kernel.
constexpr size_t kAttnCounterBytes = 4096;
constexpr int kAttnMaxGrid = kAttnCounterBytes / (2 * sizeof(int));
enum AttnSite : int { kSiteAtTma = 401, kSiteAtDrain = 402, kSiteAtDone = 403, kSiteAtFinal = 404, kSiteAtVote = 405 };

template <int D, int R>
struct ACfg {
  // The two softmax groups take alternate tiles with all rows, each with its own references, sums and
  // accumulators, joined at a segment's end (few rows: a tile's softmax is a chain of latencies), or
  // half the rows of every tile (many rows: throughput, and registers for half of them).
  static constexpr bool ALT = R <= 32;
  static constexpr int RC = ALT ? R : R / 2;           // rows of a softmax group
  static constexpr int RH = R / 2;                     // rows of a group at a segment's end
  static constexpr int GW = ALT ? 4 : 8;               // softmax warps of a tile
  static constexpr int KV = kTile * D;                 // bytes of one K or V tile of codes
  static constexpr int VB = (D / 64) * kTile * 128;    // a V tile in bf16
  static constexpr int ZB = D == 64 ? kTile * 128 : 0; // zeros: the rows 64 .. 127 of V^T
  static constexpr int PB = (2 * R + 63) / 64 * kTile * 128;
  static constexpr int QB = R * D * 2;
  static constexpr int NQ = R == 64 ? 1 : 2;           // Q buffers
  static constexpr int OFF_VB = 0;
  static constexpr int OFF_Z = OFF_VB + 2 * VB;
  static constexpr int OFF_P = OFF_Z + ZB;
  static constexpr int OFF_Q = OFF_P + 2 * PB;
  static constexpr int OFF_RING = OFF_Q + NQ * QB;
  static constexpr int SCALES = kScaleStages * (2 * kTile * 4 + 16);
  static constexpr int CTRL = 640 + SCALES + 2 * 4 * 32 * 4 * 2 + 2 * 4 * 32 * 4 + 4 * 64 * 4 + (2 * 256 + 32) * 4 + 2 * 64 * 8 + 64 * 4 +
                              (kAttnMaxBatch + 1) * 4 + 64;
  static constexpr int ROOM = 227 * 1024 - 1024 - OFF_RING - CTRL;
  static constexpr int ST = ROOM / (2 * KV) < 6 ? ROOM / (2 * KV) : 6;  // stages of a K and a V tile
  static constexpr int OFF_CTRL = OFF_RING + 2 * ST * KV;
  static constexpr int SMEM = OFF_CTRL + CTRL + 1024;
  static constexpr int A_COLS = D / 2;                 // TMEM columns of a K tile
  static constexpr int S_COL = 2 * A_COLS;
  static constexpr int O_COL = S_COL + 2 * R;
  static constexpr int COLS = O_COL + (ALT ? 4 : 2) * R <= 256 ? 256 : 512;
  static_assert(ST >= 2, "at least two stages");
  static_assert(QB % 1024 == 0 && KV % 1024 == 0, "swizzled tiles are 1024-byte aligned");
};

struct TileArgs {
  AttnArgs a;
  int64_t b0;      // first sequence of this launch
  int nb;          // its sequences
  int rts;         // row blocks
  int groups;      // CTAs per row block
  int qvec;        // q rows are 16-byte aligned
  float* pieces;   // [grid][2][R][D] fp32 accumulators, then [R] m, [R] l each
  int* counters;   // [grid][2]
  int* status;     // where a wait that runs out is recorded, and its limit
  const long long* limit;
};

// The units of one CTA's range, one (sequence, head) segment after another.
struct AttnSeg {
  int b, h;        // sequence of this launch, key head
  int kt0, n_kt;   // first tile, tiles
  int tiles;       // tiles of the whole (sequence, head)
  int u0;          // its first unit
  int slot;        // 0: the range's first segment
};
struct AttnWalk {
  int x, end, b;
  bool first;
  __device__ __forceinline__ AttnWalk(const int* pre, int nb, int x0, int x1) : x(x0), end(x1), first(true) {
    int lo = 0, hi = nb - 1;  // the last b with pre[b] <= x
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
  }
  __device__ __forceinline__ bool next(const int* pre, int heads, AttnSeg& s) {
    if (x >= end) return false;
    while (pre[b + 1] <= x) ++b;
    s.b = b;
    s.tiles = (pre[b + 1] - pre[b]) / heads;
    const int rel = x - pre[b];
    s.h = rel / s.tiles;
    s.kt0 = rel - s.h * s.tiles;
    s.u0 = x - s.kt0;
    s.n_kt = min(s.tiles - s.kt0, end - x);
    s.slot = first ? 0 : 1;
    first = false;
    x += s.n_kt;
    return true;
  }
};

// `units` units over `groups` CTAs (units >= groups): the first `rem` have one more than the others.
struct AttnSplit {
  int each, rem;
  __device__ __forceinline__ AttnSplit(int units, int groups) : each(units / groups), rem(units - each * groups) {}
  __device__ __forceinline__ int start(int c) const { return c * each + min(c, rem); }
  __device__ __forceinline__ int owner(int x) const {  // the CTA that holds unit x
    const int wide = rem * (each + 1);
    return x < wide ? x / (each + 1) : rem + (x - wide) / each;
  }
};

__device__ __forceinline__ int seq_nodes(const AttnArgs& a, int64_t b) {
  const int n = a.counts != nullptr ? a.counts[b] : a.t;
  return n < 0 ? 0 : (n < a.t ? n : a.t);
}
__device__ __forceinline__ int64_t seq_ctx(const AttnArgs& a, int64_t b) { return a.ctx[b] > 0 ? a.ctx[b] : 0; }

// v less two bf16 numbers, one instruction each (a multiply-add of bf16 factors and an fp32 addend).
__device__ __forceinline__ float2 sub_bf16x2(const float2& v, uint32_t h) {
  float2 y;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tfma.rn.f32.bf16 %0, a, %5, %3;\n\tfma.rn.f32.bf16 %1, b, %5, %4;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "r"(h), "f"(v.x), "f"(v.y), "h"(static_cast<unsigned short>(0xBF80)));  // -1
  return y;
}
// 1 / sum of a row's weights; 0 where it saw nothing.
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : __frcp_rn(sum); }

// 16 bytes global -> shared without registers; zeros, and nothing read, if !have.
__device__ __forceinline__ void cp_async16_zfill(void* dst, const void* src, bool have) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(have ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ void fence_acq_rel_gpu() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }
// One arrival on `bar` when this thread's copies so far are complete.
__device__ __forceinline__ void cp_async_arrive_noinc(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Four codes -> two bf16x2 words, exactly, with half of the work on the FMA pipe (the integer pipe, at half
// its rate, bounds the dequantisers).  u = code + 128 in the low byte of 0x4300 reads as v = 128 + u for
// u < 128 and 2 u above, where the byte's top bit falls into the exponent.  d = v - 256 is the code there and
// twice the code here, so code = d - relu(d / 2); every value fits bf16's 8 bits.
__device__ __forceinline__ void codes4_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  uint32_t v[2];
  asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(v[0]) : "r"(u), "r"(0x43434343u));
  asm("prmt.b32 %0, %1, %2, 0x5342;" : "=r"(v[1]) : "r"(u), "r"(0x43434343u));
  uint32_t q[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t r, d;
    asm("fma.rn.relu.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v[i]), "r"(0x3F003F00u), "r"(0xC300C300u));  // 0.5 v - 128
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v[i]), "r"(0x3F803F80u), "r"(0xC380C380u));       // v - 256
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(q[i]) : "r"(r), "r"(0xBF80BF80u), "r"(d));                 // d - r
  }
  lo = q[0];
  hi = q[1];
}

// 16 codes -> 16 fp16 or bf16 values.
template <bool BF16>
__device__ __forceinline__ void codes16(const uint4& v, uint32_t* o) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) codes4_bf16(w[i], o[2 * i], o[2 * i + 1]);
    else i8x4_to_f16x4(w[i], o[2 * i], o[2 * i + 1]);
  }
}

// Maximum or sum over a warp of each of N per-thread values: value c ends in the lanes
// [c * 32 / N, (c + 1) * 32 / N).
template <int N, bool MAX>
__device__ __forceinline__ float warp_columns(float (&v)[N], int lane) {
  int o = 16;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = up ? v[i] : v[i + n / 2];
      const float keep = up ? v[i + n / 2] : v[i];
      const float got = __shfl_xor_sync(0xffffffffu, send, o);
      v[i] = MAX ? fmaxf(keep, got) : keep + got;
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) {
    const float got = __shfl_xor_sync(0xffffffffu, v[0], o);
    v[0] = MAX ? fmaxf(v[0], got) : v[0] + got;
  }
  return v[0];
}

template <int D, int R, typename T>
__global__ void __launch_bounds__(kAttnThreads, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ TileArgs ta) {
  using C = ACfg<D, R>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int RC = C::RC;
  constexpr int RH = C::RH;
  constexpr int ST = C::ST;
  const AttnArgs& a = ta.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sVB = smem + C::OFF_VB;
  uint8_t* sP = smem + C::OFF_P;
  uint8_t* sQ = smem + C::OFF_Q;
  uint8_t* sK = smem + C::OFF_RING;
  uint8_t* sV = sK + ST * C::KV;
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + C::OFF_CTRL);
  uint64_t* kempty = kfull + ST;
  uint64_t* vfull = kempty + ST;
  uint64_t* vempty = vfull + ST;
  uint64_t* afull = vempty + ST;      // 2: K dequantised in TMEM
  uint64_t* vbfull = afull + 2;       // 2: V dequantised
  uint64_t* sfull = vbfull + 2;       // 2: scores (and the K tile is read)
  uint64_t* pfull = sfull + 2;        // 2: weights (and the scores are read)
  uint64_t* pempty = pfull + 2;       //    read, as is the V tile, and added to the accumulator
  uint64_t* qfull = pempty + 2;       // 2: Q and the row masks of a segment
  uint64_t* qempty = qfull + 2;
  uint64_t* scfull = qempty + 2;      // scales of a tile
  uint64_t* scempty = scfull + kScaleStages;
  uint64_t* final_bar = scempty + kScaleStages;  // 2
  uint64_t* done = final_bar + 2;                // the softmax warps have no more to do
  uint64_t* voted = done + 1;                    // 2: a group's four warps have voted on a tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(voted + 2);
  WaitControl* ctl = reinterpret_cast<WaitControl*>(voted + 3);
  volatile int* votes = reinterpret_cast<volatile int*>(voted + 6);  // [2 groups][2 parities]
  float* sScale = reinterpret_cast<float*>(smem + C::OFF_CTRL + 640);  // [stages][2][128]: ks, vs
  uint32_t* sPages = reinterpret_cast<uint32_t*>(sScale + kScaleStages * 2 * kTile);  // [stages]: pages that exist
  float* wred = reinterpret_cast<float*>(smem + C::OFF_CTRL + 640 + C::SCALES);  // [2 groups][2][4 warps][32]
  float* refs = wred + 2 * 2 * 4 * 32;                               // [2 groups][4][32]: m, its factor, sums, -m
  float* fin = refs + 2 * 4 * 32;                                    // [4][64]: m, sum, factors of the two streams
  float* ftab = fin + 4 * 64;                                        // [2 groups][2][128], 32 zeros
  unsigned long long* rmask = reinterpret_cast<unsigned long long*>(ftab + 2 * 256 + 32);  // [2][64]
  int* rows = reinterpret_cast<int*>(rmask + 2 * 64);                // [64] node | query head of the group << 16
  int* pre = rows + 64;                                              // [nb + 1] first unit of a sequence
  int* cut = pre + kAttnMaxBatch + 1;                                // [NQ][2] first and last CTA of a segment's whole
  static_assert((4 * 6 + 25 + 2 * kScaleStages) * 8 + 8 + sizeof(WaitControl) + 16 <= 640 && sizeof(WaitControl) == 24,
                "barriers");

  const int warp = warp_uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int grp = a.hq / a.c.heads;  // query heads of a key head
  const int heads = a.c.heads;
  const uint32_t never = static_cast<uint32_t>(a.t) >> 31;  // 0

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&kfull[s], 1);
      mbar_init(&kempty[s], 4);
      mbar_init(&vfull[s], 1);
      mbar_init(&vempty[s], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&afull[i], 4);
      mbar_init(&vbfull[i], 4);
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], C::GW);
      mbar_init(&pempty[i], 1);
      mbar_init(&qfull[i], 1);
      mbar_init(&qempty[i], 9);  // the last K.Q of the segment, and the softmax warps
      mbar_init(&final_bar[i], 1);
    }
    mbar_init(done, 8);
    mbar_init(&voted[0], 4);
    mbar_init(&voted[1], 4);
    for (int i = 0; i < 4; ++i) votes[i] = 0;
    for (int i = 0; i < kScaleStages; ++i) {
      mbar_init(&scfull[i], 33);  // each lane's copies, and the page word
      mbar_init(&scempty[i], C::GW);
    }
    ctl->abort = 0;
    for (int i = 0; i < 32; ++i) ftab[2 * 256 + i] = 0.f;
    ctl->status = ta.status;
    ctl->limit = ta.limit;
    fence_mbar_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  if constexpr (C::ZB > 0) {
    for (int i = threadIdx.x; i < C::ZB / 16; i += kAttnThreads)
      reinterpret_cast<uint4*>(smem + C::OFF_Z)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  const int gi = blockIdx.x / ta.rts, rt = blockIdx.x - gi * ta.rts;
  if (threadIdx.x >= 64 && threadIdx.x < 64 + R) {
    const int r = threadIdx.x - 64;
    const int n = (rt * R + r) / grp;
    rows[r] = min(n, 0x7fff) | ((rt * R + r - n * grp) << 16);
  }
  pdl_wait();  // lengths, tables, masks, q and the cache may come from the preceding kernel
  pdl_launch_dependents();
  // units before each sequence; one at least, so that every output row is written
  if (warp == 0) {
    const int64_t room = static_cast<int64_t>(a.c.table_cols) * a.c.page;
    int base = 0;
    for (int i0 = 0; i0 < ta.nb; i0 += 32) {
      int n = 0;
      if (i0 + lane < ta.nb) {
        int64_t keys = seq_ctx(a, ta.b0 + i0 + lane) + seq_nodes(a, ta.b0 + i0 + lane);
        keys = keys < room ? keys : room;
        n = static_cast<int>(keys > 0 ? (keys + kTile - 1) / kTile : 1) * heads;
      }
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int got = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += got;
      }
      if (i0 + lane < ta.nb) pre[i0 + lane] = base + sum - n;
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) pre[ta.nb] = base;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int units = pre[ta.nb];
  const int groups = min(ta.groups, units);
  const AttnSplit range(units, groups);
  const int x0 = gi < groups ? range.start(gi) : 0;
  const int x1 = gi < groups ? range.start(gi + 1) : 0;  // an empty range: nothing to do

  if (warp < 4) setmaxnreg_dec<kRegsIssue>();
  if (warp == 0 || warp == 3) {
    // ------- TMA, one box per page of a tile.  Warp 0: K.  Warp 3: V, the scales, each segment's Q and row masks -------
    const int box = min(a.c.page, kTile);           // rows of a box
    const int per = kTile / box;                    // boxes of a tile
    const int tiles_pp = max(a.c.page / kTile, 1);  // tiles of a page
    const int page_rows = heads * a.c.page;
    const uint64_t pol = ta.rts > 1 ? l2_policy_evict_normal() : l2_policy_evict_first();
    uint8_t* ring = warp == 0 ? sK : sV;
    const CUtensorMap* tm = warp == 0 ? &tm_k : &tm_v;
    uint64_t* full = warp == 0 ? kfull : vfull;
    uint64_t* empty = warp == 0 ? kempty : vempty;
    // Q of a segment (row r = node r / grp, query head r % grp of the group) into its swizzled K-major panels
    auto load_q = [&](int sq, const AttnSeg& q_sg) -> bool {
      const int qb = sq % C::NQ;
      const int64_t b = ta.b0 + q_sg.b;
      if (!mbar_wait_or_abort(&qempty[qb], ((sq / C::NQ) & 1) ^ 1, ctl)) return false;
      const int nodes = seq_nodes(a, b);
#pragma unroll 1
      for (int e0 = 0; e0 < R * (D / 8); e0 += 32 * 4) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = e0 + k * 32 + lane;
          const int r = e / (D / 8), c = e - r * (D / 8);
          const int ng = r < R ? rows[r] : 0x7fff;
          const int n = ng & 0xffff, g = ng >> 16;
          v[k] = make_uint4(0u, 0u, 0u, 0u);
          if (n < a.t) {
            const T* x = static_cast<const T*>(a.q) + b * a.q_sb + n * a.q_st + (q_sg.h * grp + g) * a.q_sh + c * 8;
            if (ta.qvec) {
              v[k] = *reinterpret_cast<const uint4*>(x);
            } else {
              const unsigned short* y = reinterpret_cast<const unsigned short*>(x);
              v[k] = make_uint4(y[0] | (static_cast<uint32_t>(y[1]) << 16), y[2] | (static_cast<uint32_t>(y[3]) << 16),
                                y[4] | (static_cast<uint32_t>(y[5]) << 16), y[6] | (static_cast<uint32_t>(y[7]) << 16));
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = e0 + k * 32 + lane;
          const int r = e / (D / 8), c = e - r * (D / 8);
          if (r < R)
            *reinterpret_cast<uint4*>(sQ + qb * C::QB + (c >> 3) * R * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[k];
        }
      }
      for (int r = lane; r < R; r += 32) {
        const int n = rows[r] & 0xffff;
        rmask[qb * 64 + r] = n < a.t ? node_mask(a, b, n, nodes) : 0ull;
      }
      if (lane == 0 && q_sg.n_kt != q_sg.tiles) {
        cut[qb * 2] = range.owner(q_sg.u0);
        cut[qb * 2 + 1] = range.owner(q_sg.u0 + q_sg.tiles - 1);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&qfull[qb]);
      return true;
    };
    bool ok = true;
    int it = 0, seg = 0;
    AttnWalk wk(pre, ta.nb, x0, x1);
    AttnSeg sg;
#pragma unroll 1
    for (; ok && wk.next(pre, heads, sg); ++seg) {
      const int64_t room = static_cast<int64_t>(a.c.table_cols) * a.c.page;
      const int64_t keys = min(seq_ctx(a, ta.b0 + sg.b) + seq_nodes(a, ta.b0 + sg.b), room);
      const int* table = a.c.table + (ta.b0 + sg.b) * a.c.table_ld;
      // 32 boxes' pages at a time, one a lane, fetched while the boxes before them are loaded
      const int batch = 32 / per;  // tiles
      auto fetch = [&](int i) -> int {
        const int64_t slot = static_cast<int64_t>(sg.kt0 + i) * kTile + lane * box;
        const int pi = tiles_pp > 1 ? (sg.kt0 + i + lane) / tiles_pp : (sg.kt0 + i) * per + lane;
        return slot < keys ? table[pi] : -1;
      };
      int raw = fetch(0), base = -1;
      if (warp == 3 && !load_q(seg, sg)) {
        ok = false;
        break;
      }
#pragma unroll 1
      for (int i = 0; i < sg.n_kt; ++i, ++it) {
        if ((i & (batch - 1)) == 0) {
          base = raw >= 0 && raw < a.c.pages ? raw * page_rows + sg.h * a.c.page : -1;
          if (i + batch < sg.n_kt) raw = fetch(i + batch);
        }
        const int first = (i & (batch - 1)) * per;  // lane of the tile's first box
        const int off = tiles_pp > 1 ? (sg.kt0 + i) % tiles_pp * kTile : 0;
        const int mine = __shfl_sync(0xffffffffu, base, first + (lane & (per - 1)));
        const bool have = lane < per && mine >= 0;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, have)) * box * D;
        const int s = it % ST;
        if (it >= ST) {
          // warp 0 watches the time for all roles
          const uint32_t ph = ((it / ST) & 1) ^ 1;
          ok = warp == 0 ? mbar_wait_at(&empty[s], ph, ctl, kSiteAtTma) : mbar_wait_or_abort(&empty[s], ph, ctl);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[s], bytes);
        __syncwarp();
        if (have) tma_load_2d(ring + s * C::KV + lane * box * D, tm, &full[s], 0, mine + off, pol);
        if (warp == 3) {  // scales, four slots a lane
          const int sc = it % kScaleStages;
          const int at = __shfl_sync(0xffffffffu, base, first + lane * 4 / box);
          const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
          if (it >= kScaleStages) {
            ok = mbar_wait_or_abort(&scempty[sc], ((it / kScaleStages) & 1) ^ 1, ctl);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
              ++it;  // (this tile's V is on its way)
              break;
            }
          }
          const int64_t row = at >= 0 ? at + off + lane * 4 % box : 0;
          float* dst = sScale + sc * 2 * kTile + lane * 4;
          cp_async16_zfill(dst, a.c.ks + row, at >= 0);
          cp_async16_zfill(dst + kTile, a.c.vs + row, at >= 0);
          cp_async_arrive_noinc(&scfull[sc]);
          if (lane == 0) {
            sPages[sc] = there;  // bit l: slots 4 l .. 4 l + 3 exist
            mbar_arrive(&scfull[sc]);
          }
        }
      }
    }
    if (!ok)  // wait (bounded) for the copies still in flight into this CTA's shared memory
      for (int j = (it > ST ? it - ST : 0); j < it; ++j)
        mbar_wait_at(&full[j % ST], (j / ST) & 1, ctl, kSiteAtDrain, false);
    if (warp == 3) cp_async_wait_all();
    // (the other roles' waits run out while warp 0 waits for the softmax warps to be done)
    if (warp == 0 && ok) mbar_wait_at(done, 0, ctl, kSiteAtDone);
  } else if (warp == 1) {
    // ---------------- K . Q ----------------
    constexpr uint32_t idesc = make_idesc_f16(128, R, BF16, false);
    const uint32_t tm = warp_uniform(tmem);
    int it = 0, seg = 0;
    bool ok = true;
    AttnWalk wk(pre, ta.nb, x0, x1);
    AttnSeg sg;
    for (; ok && wk.next(pre, heads, sg); ++seg) {
      const int qb = seg % C::NQ;
      const uint32_t q_base = smem_u32(sQ + qb * C::QB);
      ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&qfull[qb], (seg / C::NQ) & 1, ctl));
      if (!ok) break;
      const int n_kt = warp_uniform(sg.n_kt);
      for (int i = 0; i < n_kt; ++i, ++it) {
        const int t = it & 1;
        const uint32_t ph = (it >> 1) & 1;
        // (once the tile's predecessor is in the accumulator, its scores and weights are read as well: the
        // softmax warps, who see this tile's scores, need not wait for either)
        ok = mbar_wait_or_abort(&afull[t], ph, ctl) && mbar_wait_or_abort(&pempty[t], ph ^ 1, ctl);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)  // panels of 64 elements of the head dimension, 16 a step
            umma_f16_ts(tm + C::S_COL + t * R, tm + t * C::A_COLS + kk * 8,
                        make_sdesc(q_base + (kk >> 2) * R * 128 + (kk & 3) * 32, 16, 1024, kLayoutSW128), idesc, kk > 0);
          umma_commit(&sfull[t]);
          if (i == n_kt - 1) umma_commit(&qempty[qb]);
        }
        __syncwarp();
      }
    }
    if (elect_one()) {
      umma_commit(&final_bar[0]);  // every MMA issued here has completed before TMEM is released
      mbar_wait_at(&final_bar[0], 0, ctl, kSiteAtFinal, false);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------- V . P ----------------
    constexpr uint32_t idesc = make_idesc_f16(128, 2 * R, true, true, true);
    constexpr int first = C::ALT ? 1 : 0;  // the last tile of a segment that starts an accumulator
    const uint32_t tm = warp_uniform(tmem);
    int it = 0;
    bool ok = true;
    AttnWalk wk(pre, ta.nb, x0, x1);
    AttnSeg sg;
    while (ok && wk.next(pre, heads, sg)) {
      const int n_kt = warp_uniform(sg.n_kt);
      for (int i = 0; i < n_kt; ++i, ++it) {
        const int t = it & 1;
        const uint32_t ph = (it >> 1) & 1;
        ok = mbar_wait_or_abort(&vbfull[t], ph, ctl) && mbar_wait_or_abort(&pfull[t], ph, ctl);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t o_tmem = tm + C::O_COL + (C::ALT ? t * 2 * R : 0);
          const uint32_t v_base = smem_u32(sVB + t * C::VB);
          const uint32_t p_base = smem_u32(sP + t * C::PB);
          // the second 64 rows of V^T: the next panel, or zeros
          const uint32_t lbo = D == 128 ? kTile * 128 : smem_u32(smem + C::OFF_Z) - v_base;
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            umma_f16(o_tmem, make_sdesc(v_base + kk * 2048, lbo, 1024, kLayoutSW128),
                     make_sdesc(p_base + kk * 2048, kTile * 128, 1024, kLayoutSW128), idesc, i > first || kk > 0);
          umma_commit(&pempty[t]);
        }
        __syncwarp();
      }
    }
    if (elect_one()) {
      umma_commit(&final_bar[1]);
      mbar_wait_at(&final_bar[1], 0, ctl, kSiteAtFinal, false);
    }
    __syncwarp();
  } else if (warp < 8) {
    // ---------------- K codes -> TMEM (thread = slot) ----------------
    const int q = warp & 3;
    const int row = q * 32 + lane;
    const uint32_t dst = tmem + (static_cast<uint32_t>(q * 32) << 16);
    setmaxnreg_dec<kRegsK>();
    const int total = x1 - x0;
    for (int it = 0; it < total; ++it) {
      const int s = it % ST, t = it & 1;
      if (!mbar_wait_or_abort(&kfull[s], (it / ST) & 1, ctl)) break;
      // D = 128: 128-byte rows, 128-byte swizzle; D = 64: 64-byte rows, 64-byte swizzle (16-byte
      // chunk index exclusive-or bits 7, 8 of the address)
      const uint8_t* src = sK + s * C::KV + row * D;
      const int sw = D == 128 ? (row & 7) : ((row >> 1) & 3);
      if (!mbar_wait_or_abort(&sfull[t], ((it >> 1) & 1) ^ 1, ctl)) break;
      tc_fence_after();
      uint32_t loaded = 0;
#pragma unroll 1
      for (int c = 0; c < D / 16; c += 2) {
        const uint4 r0 = *reinterpret_cast<const uint4*>(src + ((c ^ sw) << 4));
        const uint4 r1 = *reinterpret_cast<const uint4*>(src + (((c + 1) ^ sw) << 4));
        uint32_t o[16];
        codes16<BF16>(r0, o);
        codes16<BF16>(r1, o + 8);
        tmem_st16(dst + t * C::A_COLS + c * 8, o);
        loaded |= r0.w | r1.w;
      }
      mbar_arrive_loaded(&kempty[s], loaded, never, lane);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&afull[t]);
    }
  } else if (warp < 12) {
    setmaxnreg_dec<kRegsV>();
    // ---------------- V codes -> shared memory ----------------
    const int w = warp - 8;
    const int total = x1 - x0;
    {
      for (int it = 0; it < total; ++it) {
        const int s = it % ST, t = it & 1;
        if (!mbar_wait_or_abort(&vfull[s], (it / ST) & 1, ctl)) break;
        if (!mbar_wait_or_abort(&pempty[t], ((it >> 1) & 1) ^ 1, ctl)) break;
        const uint8_t* src = sV + s * C::KV;
        uint8_t* dst = sVB + t * C::VB;
        uint32_t loaded = 0;
        // One 16-byte chunk of codes -> chunks 2 (c % 4), 2 (c % 4) + 1 of a bf16 row of panel c / 4.
        // Two chunks a step, few steps unrolled: five roles share the instruction cache, and with the
        // loops of the dequantisers unrolled in full half of all issue slots waited for it.
        // D = 128: the eight lanes of one shared-memory phase take four chunks of two slots whose
        // numbers differ in bits 0 and 2, so neither the swizzled read (chunks c) nor the write meets a
        // bank twice.
        const int tok8 = D == 128 ? (lane & 4 ? (lane >> 3) ^ 5 : lane >> 3) : lane >> 2;
        const int c4 = lane & 3;
        const int w0 = (((2 * c4) ^ tok8) << 4), w1 = (((2 * c4 + 1) ^ tok8) << 4);
#pragma unroll 2
        for (int k = 0; k < kTile / 32; k += D == 128 ? 1 : 2) {
          uint4 r0, r1;
          uint8_t *d0, *d1;
          if constexpr (D == 128) {  // one slot, both halves of its row
            const int tok = (w + 4 * k) * 8 + tok8;
            r0 = *reinterpret_cast<const uint4*>(src + tok * 128 + ((c4 ^ tok8) << 4));
            r1 = *reinterpret_cast<const uint4*>(src + tok * 128 + (((c4 + 4) ^ tok8) << 4));
            d0 = dst + tok * 128;
            d1 = d0 + kTile * 128;
          } else {  // two slots
            const int tok = k * 32 + w * 8 + tok8;
            r0 = *reinterpret_cast<const uint4*>(src + tok * 64 + ((c4 ^ ((tok8 >> 1) & 3)) << 4));
            r1 = *reinterpret_cast<const uint4*>(src + (tok + 32) * 64 + ((c4 ^ ((tok8 >> 1) & 3)) << 4));
            d0 = dst + tok * 128;
            d1 = d0 + 32 * 128;
          }
          uint32_t o[16];
          codes16<true>(r0, o);
          codes16<true>(r1, o + 8);
          *reinterpret_cast<uint4*>(d0 + w0) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(d0 + w1) = make_uint4(o[4], o[5], o[6], o[7]);
          *reinterpret_cast<uint4*>(d1 + w0) = make_uint4(o[8], o[9], o[10], o[11]);
          *reinterpret_cast<uint4*>(d1 + w1) = make_uint4(o[12], o[13], o[14], o[15]);
          loaded |= r0.w | r1.w;
        }
        mbar_arrive_loaded(&vempty[s], loaded, never, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&vbfull[t]);
      }
    }
  } else {
    // ---------------- softmax: thread = slot for the scores, = head dimension for the output ----------------
    setmaxnreg_inc<kRegsSoft>();
    const int g = (warp - 12) >> 2;    // group: tiles it % 2 == g, or rows [g RC, (g + 1) RC) of every tile
    constexpr int STEP = C::ALT ? 2 : 1;
    const int cb = C::ALT ? 0 : g * RC;            // first row of the group's tiles
    const int o_col = C::O_COL + (C::ALT ? g * 2 * R : cb);  // its accumulator: hi columns; lo: R further
    const int w = warp & 3;
    const int q = w;                   // TMEM lanes of this warp
    const int row = q * 32 + lane;
    const int tid = w * 32 + lane;
    const int bar = 1 + g;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
    float* gmax = wred + g * 2 * 4 * 32;
    float* gsum = gmax + 4 * 32;
    float* mref = refs + g * 4 * 32;
    float* fac = mref + 32;
    float* mneg = mref + 96;  // -m, as the scores' multiply-add takes it
    float* tab = ftab + g * 256;
    const float* zeros = ftab + 2 * 256;
    int it0 = 0, seg = 0;  // it0: the segment's first tile
    uint32_t poll = 0;     // tiles that the group has voted on
    bool ok = true;
    AttnWalk wk(pre, ta.nb, x0, x1);
    AttnSeg sg;
    for (; ok && wk.next(pre, heads, sg); it0 += sg.n_kt, ++seg) {
      const int64_t b = ta.b0 + sg.b;
      const int64_t ctx = seq_ctx(a, b);
      const int nodes = seq_nodes(a, b);
      const int64_t keys = ctx + nodes;
      const int qb = seg % C::NQ;
      const bool got_q = mbar_wait_or_abort(&qfull[qb], (seg / C::NQ) & 1, ctl);
      if (tid < RC) {
        mref[tid] = kLowest;
        mneg[tid] = -kLowest;
      }
      // A group that gives up still meets the other at the segment's end (barrier 3), where both leave.
      if (named_bar_any(bar, 128, !got_q)) ok = false;
      const unsigned long long* masks = rmask + qb * 64 + cb;
      float l[RC];
#pragma unroll
      for (int c = 0; c < RC; ++c) l[c] = 0.f;
      const int i0 = C::ALT ? (it0 ^ g) & 1 : 0;  // the group's first tile of the segment
      for (int i = i0; ok && i < sg.n_kt; i += STEP) {
        const int it = it0 + i;
        const int t = it & 1;
        const uint32_t ph = (it >> 1) & 1;
        const int64_t j0 = static_cast<int64_t>(sg.kt0 + i) * kTile;
        const int left = static_cast<int>(min(keys - j0, static_cast<int64_t>(kTile)));  // slots of the tile
        const int sc = it % kScaleStages;
        bool fine = mbar_wait_or_abort(&sfull[t], ph, ctl);
        tc_fence_after();
        // x = score - reference, in powers of two; -inf where the row does not see the slot.  A vote
        // over the group: does any score exceed its row's reference by more than 8?  The weights are
        // worked out meanwhile; if one does, once more from 0 for the rows' maxima, and again from the
        // new references.
        float x[RC];
        float ks = 0.f, vs = 0.f;
        uint32_t see = 0;  // rows that see a slot that not all see
        bool masked = false;
        int pass = i == i0 ? 1 : 0;  // (a segment's first tile has no reference yet)
        bool got = false;
#pragma unroll 1
        for (;; ++pass) {
          const float* m = pass == 1 ? zeros : mneg;
          const uint32_t s_tmem = lanes + C::S_COL + t * R + cb;
          if constexpr (RC == 32) tmem_ld32(s_tmem, reinterpret_cast<uint32_t(&)[32]>(x));
          else tmem_ld16(s_tmem, reinterpret_cast<uint32_t(&)[16]>(x));
          if (!got) {  // (while the scores are on their way)
            got = true;
            fine = mbar_wait_or_abort(&scfull[sc], (it / kScaleStages) & 1, ctl) && fine;
            ks = sScale[sc * 2 * kTile + row] * a.scale_log2;
            vs = sScale[sc * 2 * kTile + kTile + row];
            const bool there = row < left && ((sPages[sc] >> (row >> 2)) & 1);
            // a node's slot is seen by the rows whose mask names it, a context slot by all
            const int node = row + static_cast<int>(max(j0 - ctx, static_cast<int64_t>(-kTile)));
            masked = !there || node >= 0;
            if (masked && there) {
#pragma unroll 1
              for (int c = 0; c < RC; ++c) see |= static_cast<uint32_t>((masks[c] >> node) & 1) << c;
            }
          }
          tmem_ld_wait();
          const float2 k2 = make_float2(ks, ks);
#pragma unroll
          for (int c = 0; c < RC; c += 4) {
            const float4 r = *reinterpret_cast<const float4*>(m + c);
            const float2 a01 = __ffma2_rn(make_float2(x[c], x[c + 1]), k2, make_float2(r.x, r.y));
            const float2 a23 = __ffma2_rn(make_float2(x[c + 2], x[c + 3]), k2, make_float2(r.z, r.w));
            x[c] = a01.x;
            x[c + 1] = a01.y;
            x[c + 2] = a23.x;
            x[c + 3] = a23.y;
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < RC; ++c)
              if (!((see >> c) & 1)) x[c] = -INFINITY;
          }
          if (pass != 1) {
            if (pass == 0) {
              float top[2] = {x[0], x[1]};
#pragma unroll
              for (int c = 2; c < RC; c += 4) {
                top[0] = max3(top[0], x[c], x[c + 1]);
                if (c + 2 < RC) top[1] = max3(top[1], x[c + 2], x[c + 3]);
              }
              const float most = fmaxf(top[0], top[1]);
              const bool again = __any_sync(0xffffffffu, most > 8.f || !fine);
              if (lane == 0) {
                if (again) votes[g * 2 + (poll & 1)] = 1;
                mbar_arrive(&voted[g]);
              }
            }
#pragma unroll
            for (int c = 0; c < RC / 2; ++c) x[c] = exp2_approx(x[c]);  // (the other half between the conversions)
            if (pass == 2) break;
            // (All four warps vote, also after a wait that ran out, so this one ends.)
            mbar_wait_tries(&voted[g], poll & 1, ctl, kSiteAtVote);
            const bool again = votes[g * 2 + (poll & 1)] != 0;
            ++poll;
            if (!again) break;
            continue;
          }
          const float top = warp_columns<RC, true>(x, lane);
          if (lane % (32 / RC) == 0) gmax[w * 32 + lane / (32 / RC)] = top;
          // (the barrier also takes the group's decision to give up)
          if (named_bar_any(bar, 128, !fine || ctl->abort)) {
            ok = false;
            break;
          }
          if (tid == 0) votes[g * 2 + ((poll - 1) & 1)] = 0;  // all have read it
          if (tid < RC) {
            const float old = mref[tid];
            const float best = fmaxf(fmaxf(fmaxf(gmax[tid], gmax[32 + tid]), fmaxf(gmax[64 + tid], gmax[96 + tid])), old);
            mref[tid] = best;
            mneg[tid] = -best;
            fac[tid] = exp2_approx(old - best);
          }
          // the accumulator is still: its last V . P is complete, the next waits for this tile's weights
          if (i > i0) fine = mbar_wait_or_abort(&pempty[(it - STEP) & 1], ((it - STEP) >> 1) & 1, ctl);
          if (named_bar_any(bar, 128, !fine)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < RC; ++c) l[c] *= fac[c];
          if (i > i0) {
#pragma unroll 1
            for (int c = 0; c < 2 * RC; c += 8) {  // hi, then lo
              const uint32_t at = lanes + o_col + (c < RC ? c : R + c - RC);
              const float* f = fac + c % RC;
              uint32_t o[8];
              tmem_ld8(at, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f[e]);
              tmem_st8(at, o);
            }
            tmem_st_wait();
          }
        }
        if (!ok) break;
        // weights
        uint8_t* prow = sP + t * C::PB + row * 128;
        const uint32_t p_addr = smem_u32(prow) + ((row & 7) << 4);
#pragma unroll
        for (int c0 = 0; c0 < RC; c0 += 8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = c0 + 2 * e;
            const float2 p = c0 < RC / 2 ? make_float2(x[c], x[c + 1]) : make_float2(exp2_approx(x[c]), exp2_approx(x[c + 1]));
            const float2 l2 = __fadd2_rn(make_float2(l[c], l[c + 1]), p);
            l[c] = l2.x;
            l[c + 1] = l2.y;
            const float2 v = __fmul2_rn(p, make_float2(vs, vs));
            const __nv_bfloat162 h = __float22bfloat162_rn(v);
            hi[e] = *reinterpret_cast<const uint32_t*>(&h);
            const float2 left = sub_bf16x2(v, hi[e]);  // exact
            const __nv_bfloat162 r = __float22bfloat162_rn(left);
            lo[e] = *reinterpret_cast<const uint32_t*>(&r);
          }
          const int nh = cb + c0, nl = R + nh;  // columns of P
          st_shared16((p_addr ^ ((nh & 63) << 1)) + (nh >> 6) * kTile * 128, hi);
          st_shared16((p_addr ^ ((nl & 63) << 1)) + (nl >> 6) * kTile * 128, lo);
        }
        // What is not seen adds nothing, whatever its scale (0 times one that is not finite is not 0).
        if (masked && !(fabsf(vs) <= 3.402823466e38f)) {
#pragma unroll 1
          for (int c = 0; c < RC; ++c) {
            if ((see >> c) & 1) continue;
            const int nh = cb + c, nl = R + nh;
            *reinterpret_cast<unsigned short*>(prow + (nh >> 6) * kTile * 128 + ((((nh & 63) >> 3) ^ (row & 7)) << 4) + (nh & 7) * 2) = 0;
            *reinterpret_cast<unsigned short*>(prow + (nl >> 6) * kTile * 128 + ((((nl & 63) >> 3) ^ (row & 7)) << 4) + (nl & 7) * 2) = 0;
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&pfull[t]);
          mbar_arrive(&scempty[sc]);
        }
      }
      const bool split = sg.n_kt != sg.tiles;  // several CTAs share the (sequence, head)
      const int c_first = split ? cut[qb * 2] : 0;
      const int c_last = split ? cut[qb * 2 + 1] : 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&qempty[qb]);  // the masks are read no more
      // ---- the segment's end: sums of the weights, output or piece ----
      const int last = it0 + i0 + (sg.n_kt - 1 - i0) / STEP * STEP;  // the group's last tile
      const bool any = i0 < sg.n_kt;
      {
        const float sum = warp_columns<RC, false>(l, lane);
        if (lane % (32 / RC) == 0) gsum[w * 32 + lane / (32 / RC)] = sum;
      }
      const bool fine = ok && (!any || mbar_wait_or_abort(&pempty[last & 1], (last >> 1) & 1, ctl));
      if (named_bar_any(3, 256, !fine || ctl->abort)) break;
      tc_fence_after();
      const bool mine = row < D;                 // this thread's head dimension
      // From here on a group has the rows [rb, rb + RH): their references and sums, of both streams' where
      // there are two.
      const int rb = g * RH;
      if (tid < RH) {
        const int c = rb + tid;
        // (C::ALT ? both streams' sums over the four warps : the group's)
        const float* sums = wred + 4 * 32 + (C::ALT ? c : g * 2 * 4 * 32 + tid);
        float sum = ((sums[0] + sums[32]) + sums[64]) + sums[96];
        float top = mref[tid], f0 = 1.f;
        if constexpr (C::ALT) {
          const float m0 = refs[c], m1 = refs[4 * 32 + c];
          sums += 2 * 4 * 32;
          const float sum1 = ((sums[0] + sums[32]) + sums[64]) + sums[96];
          top = fmaxf(m0, m1);
          f0 = exp2_approx(m0 - top);
          const float f1 = exp2_approx(m1 - top);
          sum = f0 * sum + f1 * sum1;
          fin[192 + c] = f1;
        }
        fin[c] = top;
        fin[64 + c] = split ? sum : inverse(sum);
        fin[128 + c] = f0;
      }
      named_bar_sync(bar, 128);
      T* out = static_cast<T*>(a.o) + (b * a.t * a.hq + sg.h * grp) * static_cast<int64_t>(D) + row;
      constexpr int PIECE = R * D + 2 * R;
      float* piece = ta.pieces + (static_cast<int64_t>(blockIdx.x) * 2 + sg.slot) * PIECE;
      // piece p of the (sequence, head): CTA c_first + p's first segment, unless it started before
      auto piece_of = [&](int p) {
        const int c = c_first + p;
        const int slot = range.start(c) >= sg.u0 ? 0 : 1;
        return ta.pieces + (static_cast<int64_t>(c * ta.rts + rt) * 2 + slot) * PIECE;
      };
      const int n_p = c_last - c_first + 1;
      // Stage 0, of a (sequence, head) that several CTAs share: accumulator -> piece, and the last of them
      // goes on.  Stage 1: accumulator, or the joined pieces -> output.
#pragma unroll 1
      for (int stage = split ? 0 : 1; stage < 2; ++stage) {
        const bool join = split && stage == 1;
        if (join) {
          constexpr int SUB = 128 / RH;  // threads of one row
          float m = kLowest, sum = 0.f;
#pragma unroll 1
          for (int p = tid / RH; p < n_p; p += SUB) {
            const float* pp = piece_of(p) + R * D + rb + tid % RH;
            const float pm = __ldcg(pp), ps = __ldcg(pp + R);
            const float top = fmaxf(m, pm);
            sum = sum * exp2_approx(m - top) + ps * exp2_approx(pm - top);
            m = top;
          }
          tab[tid] = m;
          tab[128 + tid] = sum;
          named_bar_sync(bar, 128);
          if (tid < RH) {
#pragma unroll 1
            for (int k = 1; k < SUB; ++k) {
              const float pm = tab[tid + k * RH], top = fmaxf(m, pm);
              sum = sum * exp2_approx(m - top) + tab[128 + tid + k * RH] * exp2_approx(pm - top);
              m = top;
            }
            fin[rb + tid] = m;
            fin[64 + rb + tid] = inverse(sum);
          }
          named_bar_sync(bar, 128);
        }
#pragma unroll 1
        for (int c0 = 0; c0 < RH; c0 += 8) {
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = 0.f;
          if (!join) {
            constexpr int NS = C::ALT ? 2 : 1;
            uint32_t hi[NS][8], lo[NS][8];
#pragma unroll
            for (int k = 0; k < NS; ++k) {
              tmem_ld8(lanes + C::O_COL + k * 2 * R + rb + c0, hi[k]);
              tmem_ld8(lanes + C::O_COL + k * 2 * R + R + rb + c0, lo[k]);
            }
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < NS; ++k) {
              // (a stream without a tile has no accumulator)
              if (C::ALT && sg.n_kt == 1 && k != (it0 & 1)) continue;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                o[e] += (__uint_as_float(hi[k][e]) + __uint_as_float(lo[k][e])) * fin[128 + 64 * k + rb + c0 + e];
            }
          } else {
            // four pieces at a time: every thread's values and, by one warp, their factors on the way together
#pragma unroll 1
            for (int p0 = 0; p0 < n_p; p0 += 4) {
              float v[4][8];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float* pp = piece_of(min(p0 + k, n_p - 1)) + (rb + c0) * D + (mine ? row : 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] = __ldcg(pp + e * D);
              }
              if (tid < 32) {
                const int p = p0 + (tid >> 3), e = rb + c0 + (tid & 7);
                tab[tid] = p < n_p ? exp2_approx(__ldcg(piece_of(p) + R * D + e) - fin[e]) : 0.f;
              }
              named_bar_sync(bar, 128);
#pragma unroll
              for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += v[k][e] * tab[k * 8 + e];
              named_bar_sync(bar, 128);
            }
          }
          if (mine) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (stage == 0) {
                piece[(rb + c0 + e) * D + row] = o[e];
              } else {
                const int ng = rows[rb + c0 + e];
                const int n = ng & 0xffff;
                if (n < a.t)
                  out[(n * a.hq + (ng >> 16)) * static_cast<int64_t>(D)] =
                      from_f32<T>(n >= nodes ? 0.f : o[e] * fin[64 + rb + c0 + e]);
              }
            }
          }
        }
        if (!join) {
          tc_fence_before();
          if (C::ALT) named_bar_sync(3, 256);  // both groups have read both accumulators
        }
        if (stage == 0) {
          if (tid < RH) piece[R * D + rb + tid] = fin[rb + tid];
          if (tid < RH) piece[R * D + R + rb + tid] = fin[64 + rb + tid];
          named_bar_sync(bar, 128);
          if (tid == 0) {
            int* cnt = ta.counters + (c_first * ta.rts + rt) * 2 + g;
            fence_acq_rel_gpu();  // the group's stores, seen through the barrier, come before the ticket
            const bool final_one = atomicAdd(cnt, 1) == c_last - c_first;
            if (final_one) {
              fence_acq_rel_gpu();  // and the others' pieces after it
              *cnt = 0;
            }
            gmax[0] = final_one ? 1.f : 0.f;
          }
          named_bar_sync(bar, 128);
          if (gmax[0] == 0.f) break;
        }
      }
    }
    if (lane == 0) mbar_arrive(done);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, C::COLS);
}

// Row blocks: the smallest R that holds all rows, 64 at most.
static int rows_per_cta(int64_t rows) { return rows <= 16 ? 16 : (rows <= 32 ? 32 : 64); }

struct TilePlan {
  int r, rts, groups, grid;
  size_t bytes;
};
static TilePlan tile_plan(int64_t t, int64_t grp, int64_t d) {
  TilePlan p;
  p.r = rows_per_cta(t * grp);
  p.rts = static_cast<int>((t * grp + p.r - 1) / p.r);
  p.groups = num_sms() / p.rts > 1 ? num_sms() / p.rts : 1;
  p.grid = p.groups * p.rts;
  p.bytes = kAttnCounterBytes + static_cast<size_t>(p.grid) * 2 * (p.r * d + 2 * p.r) * sizeof(float);
  return p;
}
// A tile is made of whole pages or lies inside one.
static bool tile_dims(int64_t d, int64_t page) {
  return (d == 64 || d == 128) && page >= 16 && page % 16 == 0 && (kTile % page == 0 || page % kTile == 0);
}

template <int D, int R, typename T>
static int launch_tiles(const AttnArgs& a, const TilePlan& p, void* ws, bool qvec, cudaStream_t st) {
  using C = ACfg<D, R>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return check_cuda(e, "cudaGetDevice");
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(attn_tile_kernel<D, R, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (int s = check_cuda(attr_err[dev], "cudaFuncSetAttribute(attn_tile_kernel)")) return s;
  CUtensorMap tk, tv;
  const uint64_t rows = static_cast<uint64_t>(a.c.pages) * a.c.heads * a.c.page;
  const uint32_t box = a.c.page < kTile ? a.c.page : kTile;
  const CUtensorMapSwizzle swz = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (int s = make_tmap_2d(&tk, a.c.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, rows, D, D, box, D, swz)) return s;
  if (int s = make_tmap_2d(&tv, a.c.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, rows, D, D, box, D, swz)) return s;
  TileArgs ta = {};
  ta.a = a;
  ta.rts = p.rts;
  ta.groups = p.groups;
  ta.qvec = qvec;
  ta.counters = static_cast<int*>(ws);
  if (int s = device_wait_ptrs(&ta.status, &ta.limit)) return s;
  ta.pieces = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kAttnCounterBytes);
  for (int64_t b0 = 0; b0 < a.b; b0 += kAttnMaxBatch) {
    ta.b0 = b0;
    ta.nb = static_cast<int>(a.b - b0 < kAttnMaxBatch ? a.b - b0 : kAttnMaxBatch);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.grid);
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (int s = check_cuda(cudaLaunchKernelEx(&cfg, attn_tile_kernel<D, R, T>, tk, tv, ta),
                           "cudaLaunchKernelEx(attn_tile_kernel)"))
      return s;
  }
  return BW_OK;
}

template <int D, int R>
static int launch_tiles_dt(const AttnArgs& a, const TilePlan& p, void* ws, bool qvec, int dtype, cudaStream_t st) {
  return dtype == BW_DTYPE_BF16 ? launch_tiles<D, R, __nv_bfloat16>(a, p, ws, qvec, st)
                                : launch_tiles<D, R, __half>(a, p, ws, qvec, st);
}
template <int D>
static int launch_tiles_d(const AttnArgs& a, const TilePlan& p, void* ws, bool qvec, int dtype, cudaStream_t st) {
  switch (p.r) {
    case 16: return launch_tiles_dt<D, 16>(a, p, ws, qvec, dtype, st);
    case 32: return launch_tiles_dt<D, 32>(a, p, ws, qvec, dtype, st);
    default: return launch_tiles_dt<D, 64>(a, p, ws, qvec, dtype, st);
  }
}

}  // namespace bw

extern "C" size_t bw_tree_attention_int8_workspace_size(int64_t b, int64_t t, int64_t hq, int64_t heads, int64_t d) {
  if (b <= 0 || t <= 0 || t > bw::kTreeMaxNodes || heads <= 0 || hq < heads || hq > 65535 || (d != 64 && d != 128))
    return 0;
  const bw::TilePlan p = bw::tile_plan(t, hq / heads, d);
  return p.grid <= bw::kAttnMaxGrid ? p.bytes : 0;
}

extern "C" size_t bw_tree_attention_int8_workspace_zeroed_bytes(int64_t b, int64_t t, int64_t hq, int64_t heads,
                                                                int64_t d) {
  return bw_tree_attention_int8_workspace_size(b, t, hq, heads, d) != 0 ? bw::kAttnCounterBytes : 0;
}

extern "C" int bw_tree_attention_int8(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, void* out,
                                      const int8_t* cache_k, const int8_t* cache_v, const float* k_scale,
                                      const float* v_scale, int64_t pages, int64_t heads, int64_t page, int64_t d,
                                      const int32_t* table, int64_t table_ld, int64_t table_cols,
                                      const int32_t* ctx_lens, const uint64_t* mask, const int32_t* counts, int64_t b,
                                      int64_t t, int64_t hq, float softmax_scale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  using namespace bw;
  AttnArgs a = {};
  a.c.k = const_cast<int8_t*>(cache_k);
  a.c.v = const_cast<int8_t*>(cache_v);
  a.c.ks = const_cast<float*>(k_scale);
  a.c.vs = const_cast<float*>(v_scale);
  a.c.pages = pages;
  a.c.heads = heads > 0 && heads <= 65535 ? static_cast<int>(heads) : 0;
  a.c.page = page > 0 && page <= (1 << 24) ? static_cast<int>(page) : 0;
  a.c.shift = page_shift(a.c.page);
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
  // the tensor-core kernel's units are counted in 32 bits, its cache rows addressed in them
  const int64_t units = b * heads * ((table_cols * page + kTile - 1) / kTile + 1);
  const TilePlan p = tile_plan(t, hq / heads, d);
  if (tile_dims(d, page) && p.grid <= kAttnMaxGrid && units < INT32_MAX && pages > 0 && pages * heads * page < INT32_MAX &&
      (reinterpret_cast<uintptr_t>(cache_k) | reinterpret_cast<uintptr_t>(cache_v) |
       reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) % 16 == 0) {
    if (workspace == nullptr || workspace_bytes < p.bytes)
      return fail(BW_ERR_WORKSPACE, "tree_attention_int8: workspace of %zu bytes required, %zu given", p.bytes,
                  workspace_bytes);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
      return fail(BW_ERR_WORKSPACE, "tree_attention_int8: workspace must be 256-byte aligned");
    const bool qvec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_sb % 8 == 0 && q_st % 8 == 0 && q_sh % 8 == 0;
    return d == 128 ? launch_tiles_d<128>(a, p, workspace, qvec, dtype, st)
                    : launch_tiles_d<64>(a, p, workspace, qvec, dtype, st);
  }
  const dim3 grid(static_cast<unsigned>(hq), static_cast<unsigned>(t), static_cast<unsigned>(b));
  if (dtype == BW_DTYPE_BF16) attn_rows_kernel<__nv_bfloat16><<<grid, 32 * kRowWarps, 0, st>>>(a);
  else attn_rows_kernel<__half><<<grid, 32 * kRowWarps, 0, st>>>(a);
  return check_launch("attn_rows_kernel");
}
