// Causal attention over whole prompts, packed one behind the other, grouped query heads.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = exp(scale q_i . k_j)   within a sequence
//
// Sequences.  offsets[0 .. b] lie on the device, so the host knows neither lengths nor how many blocks of P rows a
// sequence has.  With the rows before the first and behind the last sequence as two more segments (of zeros), segment
// i's blocks are numbered from offset_i / P + i on (whole division): ceil(length / P) of them always fit before the
// next segment's, at most one number a segment is left without a block, and n / P + b + 2 numbers are enough for all.
// Offsets are clamped to [0, n]: where they descend, results are undefined but nothing outside is read or written.
//
// Values that are not finite.  An element of v that is infinite or NaN goes to that element of every row that sees it, whatever
// its weight: the rows' element is the sum of such values (infinities of one sign: this infinity).  The formula says so for
// every weight over 0, and all weights are; as a product, a weight that underflows would make it NaN, and whether it
// does would go by the tiles.
#include <stdio.h>

#include <mutex>
#include <type_traits>

#define BW_WHOLE_PROGRAM
#include "kv_cache.cuh"

namespace bw {

struct PromptArgs {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // strides of a token and a head
  void* o;                                     // [n, hq, d] contiguous
  const int* offsets;                          // [b + 1]
  int n, b, hq, hk, d;
  float scale_log2;
};

// A block of at most P rows of one segment: rows [row0, row1), its sequence's first row, and whether it is a sequence's.
struct PromptBlock {
  int first, row0, row1;
  bool real;
};
__device__ __forceinline__ int prompt_edge(const PromptArgs& a, int i) {  // segment i's first row
  if (i == 0) return 0;
  if (i == a.b + 2) return a.n;
  return min(max(a.offsets[i - 1], 0), a.n);
}
// Block number `slot` of P rows, by a whole warp; the last blocks of a sequence, which see most keys, come first.
__device__ __forceinline__ bool prompt_block(const PromptArgs& a, int P, int slot, PromptBlock& blk) {
  // the last segment whose numbers start at `slot` or before: 32 of the segments lo .. hi - 1 at a time
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.b + 2;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, i = lo + lane * step;
    const bool before = i < hi && prompt_edge(a, i) / P + i <= slot;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, before) | 1u);
    hi = min(hi, lo + (last + 1) * step);
    lo += last * step;
  }
  const int e0 = prompt_edge(a, lo), e1 = prompt_edge(a, lo + 1);
  const int blocks = e1 > e0 ? (e1 - e0 + P - 1) / P : 0;
  const int i = slot - (e0 / P + lo);
  if (i >= blocks) return false;
  blk.first = e0;
  blk.row0 = e0 + (blocks - 1 - i) * P;
  blk.row1 = min(blk.row0 + P, e1);
  blk.real = lo >= 1 && lo <= a.b;
  return true;
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

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
  if (!prompt_block(a, kRowsQ, blockIdx.x, blk)) return;
  const int rows = blk.row1 - blk.row0;
  const int h = blockIdx.y, hk = h / (a.hq / a.hk);
  T* out = static_cast<T*>(a.o);
  if (!blk.real) {
    for (int e = threadIdx.x; e < rows * d; e += 128)
      out[(static_cast<int64_t>(blk.row0 + e / d) * a.hq + h) * d + e % d] = from_f32<T>(0.f);
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
  for (int j0 = blk.first; j0 < blk.row1; j0 += kRowsK) {
    const int keys = min(blk.row1 - j0, kRowsK);
    __syncthreads();
    bool bad = false;
    for (int e = threadIdx.x; e < keys * d; e += 128) {
      const int j = e / d, c = e - j * d;
      const float y = to_f32(v[(j0 + j) * a.v_st + c]);
      sk[j * ld + c] = to_f32(k[(j0 + j) * a.k_st + c]);
      sv[j * d + c] = y;
      bad |= !is_finite(y);
    }
    const bool odd = __syncthreads_or(bad);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = warp * 4 + r;
      if (row >= rows) continue;
      // keys of this tile that the query sees, one at least in a sequence's first tile
      const int see = min(blk.row0 + row - j0 + 1, keys);
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
      // (2^-16: sums over as many keys of values near bf16's largest stay finite)
      const float f = exp2f(m[r] - base), p = lane < see ? exp2f(s - base - 16.f) : 0.f;
      m[r] = top;
      l[r] = l[r] * f + p;  // the lane's keys
#pragma unroll
      for (int i = 0; i < kKvMaxDim / 32; ++i) o[r][i] *= fmaxf(f, 1.17549435e-38f);  // (an infinity stays one)
      for (int j = 0; j < see; ++j) {
        const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
        for (int i = 0; i < kKvMaxDim / 32; ++i)
          if (lane + 32 * i < d) {
            const float y = sv[j * d + lane + 32 * i];
            if (odd && !is_finite(y)) o[r][i] += y;
            else o[r][i] += pj * y;
          }
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
    const float inv = sum == 0.f ? 1.f : 1.f / sum;  // (scores of -inf alone: 0, or what is not finite)
#pragma unroll
    for (int i = 0; i < kKvMaxDim / 32; ++i)
      if (lane + 32 * i < d) out[(static_cast<int64_t>(blk.row0 + row) * a.hq + h) * d + lane + 32 * i] = from_f32<T>(o[r][i] * inv);
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

// ---------------------------------------------------------------------------
// tensor-core kernel (head dimensions 64 and 128)
//
// A tile is 128 rows of queries: P = 128 / group positions with the query heads that read one key head, row = position *
// group + head.  A CTA takes two neighbouring tiles A and B of a key head (or, of few rows, one) and walks their
// sequence's keys, 128 at a time:
//   S [128 x 128 keys] = Q [128 x D] (shared memory) . K^T (shared memory)        fp32, in TMEM
//   O [128 x D]       += P [128 x 128 keys] (TMEM) . V (shared memory)            fp32, in TMEM
// At D = 128 the accumulators leave no room for P but over S, so a tile's next scores wait for its weights' product; at
// D = 64 P lies beside them, and the next scores come as soon as the softmax has these in registers.
// Each K and V tile in shared memory serves both query tiles, and while one tile's softmax runs, the other's products do.
//
// What bounds it (one B200, bf16, D = 128): the products.  16383 tokens, 16 / 8 heads: 0.84 ms, 1310 TFLOP/s; 0.72 with
// the softmax left out, 0.68 with the scores issued without waiting for the product before them.  A K . Q product of
// 128 x 128 x 16 reads 8 KB of shared memory in its 64 cycles, all that there is, next to V's 4 KB and the copies; two SMs
// that share a tile's other operand would halve that.  D = 64: the softmax warps, 1.5 us for two tiles, of which the
// special-function unit works 1.05; 16384 tokens, 32 / 8 heads: 1.34 ms, 820 TFLOP/s (1.40 with the weights over the
// scores, as at D = 128; 1.02 without the softmax).  Short prompts: a block's start and end, of which its neighbours hide a part.
// Measured and not kept, of 16383 tokens: two warps that issue the products, by kind or by query tile (0.91 and 1.03 ms:
// the tiles' softmax phases drift onto each other, where the one warp's order keeps them apart); two threads a row (1.4);
// a quarter of the exponentials as polynomials (0.88); weights checked by their sum in place of the maximum (0.86); one
// hand-over of the weights in place of two (0.87); the next block's first scores issued before the last of B (0.85).
//
// Softmax: thread = row, so nothing is exchanged.  The reference m moves only when a score exceeds it by more than 8 (in
// powers of two); only then are the sum and the accumulator rescaled (a published way of rescaling less often).  Weights
// 2^(s - m + shift) go to the tensor core in the inputs' type: rounded by half an ulp like the inputs themselves.  fp16: a
// shift of 7, so at most 2^15, and the type's subnormal steps are at most 2^-31 of a row's largest weight.  bf16, whose
// values reach fp32's range: -16, so that the sum over 2^16 keys of values near the largest stays finite (2^8 where scores
// have gone 8 above the reference).  Their sum and the accumulator are fp32 and have the same factor.
//
// Keys that a row does not see have weight 0, but 0 times a value that is not finite is not 0.  So a warp looks through
// every V tile that some row of the block does not see all of: rows behind the block's last position become zeros,
// values that are not finite become 0 and are added at the end to the rows that do see them.  The tiles before, which all
// rows see, go into the product as they are.  Where that leaves something that is not finite, the block's end sums those
// tiles' values that are not finite from memory and puts the sum in place of what the weights have made of them: which
// tiles are looked through goes by the block, so by the other sequences, and the results must not.
//
// Blocks are handed out by the hardware: a CTA that nears its end takes the next one that has not started
// (clusterlaunchcontrol), so the schedule is dynamic without a counter in memory.
//
// Twelve warps: 0-3 and 4-7 the softmax of A and B (their TMEM lanes are the rows), 8 finds the blocks, loads and watches
// the time, 9 issues the products, 10 and 11 look through V.
// ---------------------------------------------------------------------------
constexpr int kPromptThreads = 384;
constexpr int kPromptKeys = 128;
// Registers of a thread of the three warpgroups after setmaxnreg: three times the 168 that a thread of 384 has.
constexpr int kPromptRegsSoft = 208, kPromptRegsRest = 88;
static_assert(2 * kPromptRegsSoft + kPromptRegsRest == 3 * 168, "register split");
// A CTA takes its next block when it loads the last but third key tile of the one it has: a block taken earlier is out of
// other CTAs' reach for longer, one taken later is not there in time.
constexpr int kPromptAhead = 4;
constexpr float kPromptSlack = 8.f;
template <typename T>
constexpr float kPromptShift = std::is_same<T, __half>::value ? 7.f : -16.f;
constexpr float kPromptLowest = -3.0e38f;  // a row's reference without any score: finite, so differences are
enum PromptSite : int {
  kSitePrBlock = 501, kSitePrQ = 502, kSitePrK = 503, kSitePrV = 504, kSitePrDrain = 505, kSitePrDone = 506,
  kSitePrFinal = 507, kSitePrNext = 508
};

template <int D>
struct PCfg {
  static constexpr int KEYS_COLS = kPromptKeys;
  static constexpr int TB = D / 64 * kPromptKeys * 128;  // bytes of a tile of Q, K or V: panels of 64 elements
  static constexpr int KST = D == 128 ? 2 : 4, VST = D == 128 ? 2 : 4;
  static constexpr int OB = 32 * 128;  // bytes of a softmax warp's part of the output on its way out
  static constexpr int OFF_K = 2 * TB;
  static constexpr int OFF_V = OFF_K + KST * TB;
  static constexpr int OFF_O = OFF_V + VST * TB;
  static constexpr int OFF_CTRL = OFF_O + 8 * OB;
  static constexpr int CTRL = 1024;
  static constexpr int SMEM = OFF_CTRL + CTRL + 1024;
  static constexpr int S_COL = 0, O_COL = 256, COLS = 512;
  // D = 64: accumulators of half the size leave room for the weights beside the scores.
  static constexpr bool APART = D == 64;
  static constexpr int P_COL = APART ? 384 : S_COL, P_STEP = APART ? 64 : KEYS_COLS;  // of A; from A to B
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct PromptTiles {
  PromptArgs a;
  int grp, pos;     // query heads of a key head, positions of a tile
  int block;        // positions of a block: of one tile or of two
  int* status;
  const long long* limit;
};

// A block as the roles read it; positions relative to the sequence's first row.
struct PromptInfo {
  int first, row0, row1, head, n[2], valid;
};

__device__ __forceinline__ void clc_try_cancel(void* response, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(response)),
               "r"(smem_u32(bar))
               : "memory");
}
// The block taken, or -1: none was left.
__device__ __forceinline__ int clc_block(const void* response) {
  int x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 r, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, r;\n\t}\n"
      : "=r"(x)
      : "r"(smem_u32(response))
      : "memory");
  return x;
}

// Bits of a packed pair of 16-bit values that are set where one of them is not finite.
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
  else return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float2 v) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __float22half2_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// A packed pair with infinities of the type's largest value in their place (a NaN stays one).
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 top = __half2half2(__ushort_as_half(0x7BFF));
    const __half2 h = __hmax2_nan(__hmin2_nan(*reinterpret_cast<const __half2*>(&w), top), __hneg2(top));
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 top = __bfloat162bfloat162(__ushort_as_bfloat16(0x7F7F));
    const __nv_bfloat162 h = __hmax2_nan(__hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), top), __hneg2(top));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
constexpr float kPromptTop = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;  // the type's largest value

template <int D, typename T>
__global__ void __launch_bounds__(kPromptThreads, 1)
    prompt_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PromptTiles ta) {
  using C = PCfg<D>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int KEYS = kPromptKeys;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::OFF_K;
  uint8_t* sV = smem + C::OFF_V;
  uint8_t* sO = smem + C::OFF_O;
  uint64_t* tfull = reinterpret_cast<uint64_t*>(smem + C::OFF_CTRL);  // 2: a block's numbers are there
  uint64_t* tempty = tfull + 2;        //    all roles are done with them
  uint64_t* qfull = tempty + 2;        // [A, B]
  uint64_t* qempty = qfull + 2;
  uint64_t* kfull = qempty + 2;
  uint64_t* kempty = kfull + C::KST;
  uint64_t* vfull = kempty + C::KST;
  uint64_t* vready = vfull + C::VST;   // looked through
  uint64_t* vempty = vready + C::VST;
  uint64_t* sfull = vempty + C::VST;   // [A, B] scores
  uint64_t* sread = sfull + 2;         //        in registers (APART)
  uint64_t* phalf = sread + 2;         // weights of the first 64 keys, of all
  uint64_t* pfull = phalf + 2;
  uint64_t* pvdone = pfull + 2;        //    P . V complete
  uint64_t* oempty = pvdone + 2;       // accumulator read
  uint64_t* ckfull = oempty + 2;       // 2: a block's values that are not finite are known
  uint64_t* next_bar = ckfull + 2;     // a block from the hardware
  uint64_t* done = next_bar + 1;
  uint64_t* final_bar = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(final_bar + 1);
  WaitControl* ctl = reinterpret_cast<WaitControl*>(final_bar + 2);
  PromptInfo* info = reinterpret_cast<PromptInfo*>(smem + C::OFF_CTRL + 512);  // [2]
  uint32_t* odd = reinterpret_cast<uint32_t*>(smem + C::OFF_CTRL + 640);       // [2][3 tiles][128 bits]
  void* response = smem + C::OFF_CTRL + 768;
  static_assert((27 + 2 * C::KST + 3 * C::VST) * 8 + 8 + sizeof(WaitControl) <= 512 && sizeof(PromptInfo) <= 64, "control");

  const PromptArgs& a = ta.a;
  const int warp = warp_uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int P = ta.pos;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 11);  // products, two warps that look through V, eight softmax warps
      mbar_init(&qfull[i], 1);
      mbar_init(&qempty[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&sread[i], 4);
      mbar_init(&phalf[i], 4);
      mbar_init(&pfull[i], 4);
      mbar_init(&pvdone[i], 1);
      mbar_init(&oempty[i], 4);
      mbar_init(&ckfull[i], 2);
    }
    for (int i = 0; i < C::KST; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&kempty[i], 1);
    }
    for (int i = 0; i < C::VST; ++i) {
      mbar_init(&vfull[i], 1);
      mbar_init(&vready[i], 2);
      mbar_init(&vempty[i], 1);
    }
    mbar_init(next_bar, 1);
    mbar_init(done, 8);
    mbar_init(final_bar, 1);
    ctl->abort = 0;
    ctl->status = ta.status;
    ctl->limit = ta.limit;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    setmaxnreg_dec<kPromptRegsRest>();
    if (warp == 8) {
      // ---------------- blocks and TMA ----------------
      const uint64_t pol = l2_policy_evict_normal();
      uint32_t qn[2] = {0u, 0u}, kn = 0, vn = 0;  // loads so far
      uint32_t asked = 0, got = 0;                // answers to try_cancel
      auto ask = [&]() {
        if (elect_one()) {
          mbar_arrive_expect_tx(next_bar, 16);
          clc_try_cancel(response, next_bar);
        }
        __syncwarp();
        ++asked;
      };
      auto answer = [&]() {
        mbar_wait_tries(next_bar, got & 1, ctl, kSitePrNext);
        ++got;
        const int x = clc_block(response);
        fence_proxy_async_smem();  // read before the next answer is written
        __syncwarp();
        return x;
      };
      PromptInfo t;
      // Block number `x`, or the next one that has rows of a sequence; false: none is left.
      auto find = [&](int x) {
        while (x >= 0 && !ctl->abort) {
          const int slot = x / a.hk, head = x - slot * a.hk;
          PromptBlock blk;
          if (prompt_block(a, ta.block, slot, blk)) {
            if (blk.real) {
              t.first = blk.first;
              t.row0 = blk.row0 - blk.first;
              t.row1 = blk.row1 - blk.first;
              t.head = head;
              t.n[0] = (min(t.row0 + P, t.row1) - 1) / KEYS + 1;
              t.n[1] = t.row0 + P < t.row1 ? (t.row1 - 1) / KEYS + 1 : 0;
              return true;
            }
            // rows of no sequence: zeros
            const int per = ta.grp * D / 8;  // 16-byte chunks of a row
            for (int r = blk.row0; r < blk.row1; ++r) {
              uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + (static_cast<int64_t>(r) * a.hq + head * ta.grp) * D);
              for (int e = lane; e < per; e += 32) out[e] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          ask();
          x = answer();
        }
        return false;
      };
      auto load = [&](uint8_t* dst, const CUtensorMap* tm, uint64_t* full, uint32_t bytes, int head, int row) {
        if (elect_one()) {
          mbar_arrive_expect_tx(full, bytes);
#pragma unroll
          for (int c = 0; c < D / 64; ++c) tma_load_3d(dst + c * KEYS * 128, tm, full, c * 64, head, row, pol);
        }
        __syncwarp();
      };
      const uint32_t q_bytes = static_cast<uint32_t>(P * ta.grp * D * 2);
      bool ok = true;
      int x = blockIdx.x;
      for (uint32_t n = 0;; ++n) {
        const int sl = n & 1;
        const bool have = find(x);
        ok = __all_sync(0xffffffffu, mbar_wait_at(&tempty[sl], ((n >> 1) & 1) ^ 1, ctl, kSitePrBlock));
        if (!ok) break;
        if (lane == 0) {
          t.valid = have;
          info[sl] = t;
          mbar_arrive(&tfull[sl]);
        }
        __syncwarp();
        if (!have) break;
        auto load_q = [&](int w) {
          if (t.n[w] == 0) return true;
          const bool fine = mbar_wait_at(&qempty[w], (qn[w] & 1) ^ 1, ctl, kSitePrQ);
          if (!__all_sync(0xffffffffu, fine)) return false;
          load(sQ + w * C::TB, &tm_q, &qfull[w], q_bytes, t.head * ta.grp, t.first + t.row0 + w * P);
          ++qn[w];
          return true;
        };
        const int tiles = max(t.n[0], t.n[1]);
        ok = load_q(0);
        for (int i = 0; ok && i < tiles; ++i) {
          if (i == max(tiles - kPromptAhead, 0)) ask();
          const int ks = kn % C::KST, vs = vn % C::VST;
          ok = __all_sync(0xffffffffu, mbar_wait_at(&kempty[ks], ((kn / C::KST) & 1) ^ 1, ctl, kSitePrK));
          if (!ok) break;
          load(sK + ks * C::TB, &tm_k, &kfull[ks], C::TB, t.head, t.first + i * KEYS);
          ++kn;
          if (i == 0) ok = load_q(1);
          ok = ok && __all_sync(0xffffffffu, mbar_wait_at(&vempty[vs], ((vn / C::VST) & 1) ^ 1, ctl, kSitePrV));
          if (!ok) break;
          load(sV + vs * C::TB, &tm_v, &vfull[vs], C::TB, t.head, t.first + i * KEYS);
          ++vn;
        }
        if (!ok) break;
        x = answer();
      }
      if (ok) {
        mbar_wait_at(done, 0, ctl, kSitePrDone);
      } else {  // wait (bounded) for what is still on its way into this CTA's shared memory
        if (asked > got) mbar_wait_tries(next_bar, got & 1, ctl, kSitePrNext);
        for (uint32_t i = kn > C::KST ? kn - C::KST : 0; i < kn; ++i)
          mbar_wait_at(&kfull[i % C::KST], (i / C::KST) & 1, ctl, kSitePrDrain, false);
        for (uint32_t i = vn > C::VST ? vn - C::VST : 0; i < vn; ++i)
          mbar_wait_at(&vfull[i % C::VST], (i / C::VST) & 1, ctl, kSitePrDrain, false);
        for (int w = 0; w < 2; ++w)
          if (qn[w] > 0) mbar_wait_at(&qfull[w], (qn[w] - 1) & 1, ctl, kSitePrDrain, false);
      }
    } else if (warp == 9) {
      // ---------------- products ----------------
      {
        const uint32_t tm = warp_uniform(tmem);
        constexpr uint32_t idesc_s = make_idesc_f16(128, KEYS, BF16, false);
        constexpr uint32_t idesc_o = make_idesc_f16(128, D, BF16, true);
        const uint32_t q0 = smem_u32(sQ), k0 = smem_u32(sK), v0 = smem_u32(sV);
        uint32_t ks = 0, kp = 0, vs = 0, vp = 0;  // stage and parity of the next K and V tile
        uint32_t sp = 0, bp = 0;                  // parities of the next tile (bit w) and the next block of A and B
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
          ok = ok && __all_sync(0xffffffffu, mbar_wait_or_abort(bar, parity & 1u, ctl));
          return ok;
        };
        uint32_t rp = 0;                          // parity of the next scores of A and B
        // Scores of the next K tile, once the weights over which they go have been read (products of different
        // accumulators are not ordered); APART: once the scores before them have.
        auto scores = [&](int w, bool give_k, bool give_q) {
          if (!wait(C::APART ? &sread[w] : &pvdone[w], ((C::APART ? rp : sp) >> w) ^ 1u)) return;
          rp ^= 1u << w;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t at = (kk >> 2) * KEYS * 128 + (kk & 3) * 32;
            umma_f16(tm + C::S_COL + w * KEYS, make_sdesc(q0 + w * C::TB + at, 16, 1024, kLayoutSW128),
                     make_sdesc(k0 + ks * C::TB + at, 16, 1024, kLayoutSW128), idesc_s, kk > 0);
          }
          umma_commit(&sfull[w]);
          if (give_k) umma_commit(&kempty[ks]);
          if (give_q) umma_commit(&qempty[w]);
          }
          __syncwarp();
        };
        auto weighted = [&](int w, bool first, bool give_v) {
          const uint32_t o = tm + C::O_COL + w * D, p = tm + C::P_COL + w * C::P_STEP, v = v0 + vs * C::TB;
          const uint32_t parity = sp >> w;
          if (!wait(&phalf[w], parity)) return;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < KEYS / 32; ++kk)
            umma_f16_ts(o, p + kk * 8, make_sdesc(v + kk * 2048, KEYS * 128, 1024, kLayoutSW128), idesc_o, !first || kk > 0);
          }
          __syncwarp();
          if (!wait(&pfull[w], parity)) return;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
          for (int kk = KEYS / 32; kk < KEYS / 16; ++kk)
            umma_f16_ts(o, p + kk * 8, make_sdesc(v + kk * 2048, KEYS * 128, 1024, kLayoutSW128), idesc_o, 1);
          umma_commit(&pvdone[w]);
          if (give_v) umma_commit(&vempty[vs]);
          }
          __syncwarp();
          sp ^= 1u << w;
        };
        auto next_k = [&]() {
          if (++ks == C::KST) {
            ks = 0;
            kp ^= 1;
          }
        };
        for (uint32_t n = 0; ok; ++n) {
          const int sl = n & 1;
          if (!wait(&tfull[sl], n >> 1)) break;
          const int na = warp_uniform(info[sl].n[0]), nb = warp_uniform(info[sl].n[1]), valid = warp_uniform(info[sl].valid);
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[sl]);
          if (!valid) break;
          const int tiles = max(na, nb);
          const bool both = nb > 0;  // (B then needs every K and V tile, and last)
          // (Two copies of each product's instructions, which share a cache with the other roles'; with one, whose addresses
          // are worked out on the way, long prompts take 3 % longer, with six short ones.)
          // Tile i + 1's scores: the first of A and B to come to them waits for the K tile.
          auto scores_of = [&](int w, int i, bool& have_k) {
            if (i + 1 == 0 && !wait(&qfull[w], bp >> w)) return;
            if (!have_k && !wait(&kfull[ks], kp)) return;
            have_k = true;
            scores(w, w == 1 || !both, i + 2 == (w ? nb : na));
          };
          auto weights_of = [&](int w, int i, bool& have_v) {
            if (!have_v && !wait(&vready[vs], vp)) return;
            have_v = true;
            if (i == 0 && !wait(&oempty[w], (bp >> w) ^ 1u)) return;  // the block before has been read
            weighted(w, i == 0, w == 1 || !both);
          };
          auto next_v = [&]() {
            if (++vs == C::VST) {
              vs = 0;
              vp ^= 1;
            }
          };
          if constexpr (C::APART) {
            // The scores of tile i + 1 while the softmax works on tile i, and the weights of B a tile behind those of A.
            bool have_v = false;
#pragma unroll 1
            for (int i = -1; ok && i <= tiles; ++i) {
              bool have_k = false;
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                if (i + 1 < (w ? nb : na)) scores_of(w, i, have_k);
                const int j = i - 1 + w, u = 1 - w;  // B's of tile i - 1, then A's of tile i
                if (ok && j >= 0 && j < (u ? nb : na)) weights_of(u, j, have_v);
                if (w == 0 && i >= 1) {
                  next_v();
                  have_v = false;
                }
              }
              if (i + 1 < tiles) next_k();
            }
          } else {
#pragma unroll 1
            for (int i = -1; ok && i < tiles; ++i) {
              bool have_k = false, have_v = false;
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const int mine = w ? nb : na;
                if (i >= 0 && i < mine) weights_of(w, i, have_v);
                if (ok && i + 1 < mine) scores_of(w, i, have_k);
              }
              if (i + 1 < tiles) next_k();
              if (i >= 0) next_v();
            }
          }
          bp ^= both ? 3u : 1u;
        }
        if (elect_one()) {
          umma_commit(final_bar);  // every MMA issued here has completed before TMEM is released
          mbar_wait_at(final_bar, 0, ctl, kSitePrFinal, false);
        }
      }
      __syncwarp();
    } else {
      // ---------------- V tiles that are not seen as a whole: 64 rows a warp ----------------
      const int part = warp - 10;
      uint32_t vn = 0;
      for (uint32_t n = 0;; ++n) {
        const int sl = n & 1;
        if (!__all_sync(0xffffffffu, mbar_wait_or_abort(&tfull[sl], (n >> 1) & 1, ctl))) break;
        const PromptInfo t = info[sl];
        __syncwarp();
        if (!t.valid) break;
        const int tiles = max(t.n[0], t.n[1]);
        const int from = (t.row0 + 1) / KEYS;  // the first tile with a key behind the block's first position
        bool ok = true;
        for (int i = 0; i < tiles; ++i, ++vn) {
          const uint32_t vs = vn % C::VST;
          ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&vfull[vs], (vn / C::VST) & 1, ctl));
          if (!ok) break;
          if (i >= from) {
            uint8_t* tile = sV + vs * C::TB;
            const int have = t.row1 - i * KEYS;  // keys up to the block's last position
#pragma unroll 1
            for (int q = part * 2; q < part * 2 + 2; ++q) {
              uint8_t* row = tile + (q * 32 + lane) * 128;
              uint32_t bad = 0;
              if (q * 32 + lane < have) {
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {  // (the chunks of 16 bytes in an order without bank conflicts)
                  const uint4 x = *reinterpret_cast<const uint4*>(row + (c >> 3) * KEYS * 128 + (((c ^ lane) & 7) << 4));
                  bad |= not_finite2<T>(x.x) | not_finite2<T>(x.y) | not_finite2<T>(x.z) | not_finite2<T>(x.w);
                }
              } else {
#pragma unroll
                for (int c = 0; c < D / 8; ++c)
                  *reinterpret_cast<uint4*>(row + (c >> 3) * KEYS * 128 + (((c ^ lane) & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
              }
              const uint32_t word = __ballot_sync(0xffffffffu, bad != 0);
              if (bad != 0) {
#pragma unroll 1
                for (int c = 0; c < D / 2; ++c) {
                  uint32_t* x = reinterpret_cast<uint32_t*>(row + (c >> 5) * KEYS * 128 + (c & 31) * 4);
                  const uint32_t b = not_finite2<T>(*x);
                  if (b & 0x8000u) *x &= 0xFFFF0000u;
                  if (b & 0x80000000u) *x &= 0x0000FFFFu;
                }
              }
              if (lane == 0) odd[sl * 12 + (i - from) * 4 + q] = word;
            }
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&vready[vs]);
        }
        if (!ok) break;
        if (lane == 0) {
          for (int i = max(tiles - from, 0) * 4 + part * 2; i < 12; i += 4) odd[sl * 12 + i] = odd[sl * 12 + i + 1] = 0u;
          mbar_arrive(&ckfull[sl]);
          mbar_arrive(&tempty[sl]);
        }
      }
    }
  } else {
    // ---------------- softmax: thread = row ----------------
    setmaxnreg_inc<kPromptRegsSoft>();
    const int w = warp >> 2;  // query tile
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_tm = lanes + C::S_COL + w * KEYS, o_tm = lanes + C::O_COL + w * D;
    const uint32_t p_tm = lanes + C::P_COL + w * C::P_STEP;
    const int p = row / ta.grp, g = row - p * ta.grp;
    const float sc = a.scale_log2;
    uint32_t it = 0;  // score tiles so far
    for (uint32_t n = 0;; ++n) {
      const int sl = n & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_or_abort(&tfull[sl], (n >> 1) & 1, ctl))) break;
      const PromptInfo t = info[sl];
      if (!t.valid) break;
      if (t.n[w] == 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[sl]);
        continue;
      }
      const int pos0 = t.row0 + w * P;  // the tile's first position
      const int pos = pos0 + p;
      float m = kPromptLowest;
      float2 l2[2] = {};
      bool ok = true;
#pragma unroll 1
      for (int i = 0; i < t.n[w]; ++i, ++it) {
        ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&sfull[w], it & 1, ctl));
        if (!ok) break;
        tc_fence_after();
        float x[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_tm + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&x[c * 32]));
        tmem_ld_wait();
        if constexpr (C::APART) {  // the next scores may come
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sread[w]);
        }
        if (i * KEYS + KEYS - 1 > pos0) {  // keys that some row does not see
          const int see = pos - i * KEYS + 1;
#pragma unroll
          for (int c = 0; c < 128; ++c) x[c] = c < see ? x[c] : -INFINITY;
        }
        float top[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) top[c] = fmaxf(x[c * 16], x[c * 16 + 1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2)
#pragma unroll
          for (int c = 0; c < 8; ++c) top[c] = max3(top[c], x[c * 16 + e], x[c * 16 + e + 1]);
        const float best = fmaxf(max3(max3(top[0], top[1], top[2]), top[3], top[4]), max3(top[5], top[6], top[7])) * sc;
        if constexpr (C::APART) {  // the weights before have been read
          ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&pvdone[w], (it & 1) ^ 1, ctl));
          if (!ok) break;
          tc_fence_after();
        }
        if (i == 0) {
          m = fmaxf(best, kPromptLowest);
        } else if (__any_sync(0xffffffffu, best > m + kPromptSlack)) {
          // the accumulator is still: these scores were issued behind its last product (APART: which is waited for)
          const float to = best > m + kPromptSlack ? best : m;
          const float f = exp2_approx(m - to);
          m = to;
#pragma unroll
          for (int e = 0; e < 2; ++e) l2[e] = __fmul2_rn(l2[e], make_float2(f, f));
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_tm + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(o_tm + c, o);
          }
          tmem_st_wait();
        }
        const float2 sc2 = make_float2(sc, sc), m2 = make_float2(kPromptShift<T> - m, kPromptShift<T> - m);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t packed[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int e = h * 64 + 2 * c;
            const float2 z = __ffma2_rn(make_float2(x[e], x[e + 1]), sc2, m2);
            const float2 v = make_float2(exp2_approx(z.x), exp2_approx(z.y));
            l2[c % 2] = __fadd2_rn(l2[c % 2], v);
            packed[c] = pack2<T>(v);
          }
          tmem_st32(p_tm + h * 32, packed);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(h == 0 ? &phalf[w] : &pfull[w]);
        }
      }
      if (!ok) break;
      // ---- the block's end ----
      ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&pvdone[w], (it - 1) & 1, ctl) &&
                                       mbar_wait_or_abort(&ckfull[sl], (n >> 1) & 1, ctl));
      if (!ok) break;
      tc_fence_after();
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < 12; ++k) any |= odd[sl * 12 + k];
      const float2 l4 = __fadd2_rn(l2[0], l2[1]);
      const float sum = l4.x + l4.y;
      const float inv = sum == 0.f ? 0.f : __frcp_rn(sum);
      const bool mine = p < P && pos < t.row1;
      // 64 elements of the rows at a time through shared memory, so that a store has 128 bytes of each of four rows: 16
      // bytes of 32 rows each took a quarter of the time of 24 prompts of up to 1021 tokens.
      T* out = static_cast<T*>(a.o) + ((static_cast<int64_t>(t.first) + pos0) * a.hq + t.head * ta.grp) * D;
      const int at = mine ? (p * a.hq + g) * D : -1;  // of this lane's row
      uint8_t* stage = sO + warp * C::OB;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 64) {
        float most = 0.f;  // of the row's elements; NaN if one is
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_tm + c0 + c, o);
          tmem_ld_wait();
          float y[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = __uint_as_float(o[e]) * inv;
#pragma unroll
          for (int e = 0; e < 32; e += 2) most = max3_nan(most, fabsf(y[e]), fabsf(y[e + 1]));
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((((c + e) >> 3) ^ (lane & 7)) << 4)) =
                make_uint4(pack2<T>(make_float2(y[e], y[e + 1])), pack2<T>(make_float2(y[e + 2], y[e + 3])),
                           pack2<T>(make_float2(y[e + 4], y[e + 5])), pack2<T>(make_float2(y[e + 6], y[e + 7])));
        }
        const int from = (t.row0 + 1) / KEYS * KEYS;  // keys before it are in tiles that all rows see
        const T* v = static_cast<const T*>(a.v) + static_cast<int64_t>(t.first) * a.v_st + t.head * a.v_sh + c0;
        if (__builtin_expect(__any_sync(0xffffffffu, mine && !(most <= kPromptTop<T>)), 0)) {
          // (The code here is kept small: more of it makes all blocks slower, 24 prompts of up to 1021 tokens 101.5 us for 100.9
          // with 32 keys at a time below.)
          // A mean of values near the type's largest that the weights' rounding has carried past it: their sum takes them unrounded.
#pragma unroll 1
          for (int c = 0; c < 32; ++c) {
            uint32_t* x = reinterpret_cast<uint32_t*>(stage + lane * 128 + c * 4);
            *x = finite2<T>(*x);
          }
          __syncwarp();
        }
        if (__builtin_expect(from > 0 && __any_sync(0xffffffffu, mine && sum == sum && !(most <= 3.402823466e38f)), 0)) {
          // values that are not finite, of the keys that all rows see: lane = two elements, eight keys at a time
          float2 z = make_float2(0.f, 0.f);
#pragma unroll 1
          for (int key = 0; key < from; key += 8) {
            uint32_t x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const uint32_t*>(v + (key + u) * a.v_st + 2 * lane);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const uint32_t b = not_finite2<T>(x[u]);
              const T* h = reinterpret_cast<const T*>(&x[u]);
              if (b & 0x8000u) z.x += to_f32(h[0]);
              if (b & 0x80000000u) z.y += to_f32(h[1]);
            }
          }
          const uint32_t nan_rows = __ballot_sync(0xffffffffu, sum != sum);  // (of scores, not of values)
#pragma unroll 1
          for (int r = 0; r < 32; ++r) {
            T* y = reinterpret_cast<T*>(stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            if (nan_rows >> r & 1) continue;
            if (z.x != 0.f) y[0] = from_f32<T>(z.x);
            if (z.y != 0.f) y[1] = from_f32<T>(z.y);
          }
          __syncwarp();
        }
        if (any != 0 && mine) {
          // values that are not finite, of the keys that this row sees among those that not all see
#pragma unroll 1
          for (int k = 0; k < 12; ++k) {
#pragma unroll 1
            for (uint32_t word = odd[sl * 12 + k]; word != 0; word &= word - 1) {
              const int key = from + k * 32 + __ffs(word) - 1;
              if (key > pos) continue;
#pragma unroll 1
              for (int e = 0; e < 64; ++e) {
                const float z = to_f32(v[key * a.v_st + e]);
                T* y = reinterpret_cast<T*>(stage + lane * 128 + (((e >> 3) ^ (lane & 7)) << 4)) + (e & 7);
                if (!is_finite(z)) *y = from_f32<T>(to_f32(*y) + z);
              }
            }
          }
        }
        __syncwarp();
        uint4 line[8];
        int to[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = 4 * k + (lane >> 3);
          to[k] = __shfl_sync(0xffffffffu, at, r);
          line[k] = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane ^ r) & 7) << 4));
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (to[k] >= 0) *reinterpret_cast<uint4*>(out + to[k] + c0 + (lane & 7) * 8) = line[k];
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&oempty[w]);
        mbar_arrive(&tempty[sl]);
      }
    }
    if (lane == 0) mbar_arrive(done);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, C::COLS);
}

static bool tma_rows(const void* p, int64_t st, int64_t sh) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st % 8 == 0 && sh % 8 == 0 && st > 0 && sh > 0 &&
         st < (int64_t{1} << 38) && sh < (int64_t{1} << 38);
}

template <int D, typename T>
static int launch_tiles(const PromptArgs& a, cudaStream_t st) {
  using C = PCfg<D>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return check_cuda(e, "cudaGetDevice");
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(prompt_tile_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (int s = check_cuda(attr_err[dev], "cudaFuncSetAttribute(prompt_tile_kernel)")) return s;
  PromptTiles ta = {};
  ta.a = a;
  ta.grp = a.hq / a.hk;
  ta.pos = 128 / ta.grp;
  // Few rows: blocks of one tile, so that twice as many SMs share them and each walks its keys faster (1.4 us for 128 keys,
  // 1.75 with two tiles); once two-tile blocks fill the SMs, those.  16 / 8 heads of 128, one prompt, us with one tile and
  // with two: 1024 tokens 18.3 and 20.5, 2048 (128 two-tile blocks) 30.9 and 34.2, 3000 (188) 60.7 and 46.1.
  const bool few = (a.n / (2 * ta.pos) + a.b) * a.hk <= num_sms();
  ta.block = few ? ta.pos : 2 * ta.pos;
  if (int s = device_wait_ptrs(&ta.status, &ta.limit)) return s;
  const CUtensorMapDataType dt =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tq, tk, tv;
  auto map = [&](CUtensorMap* m, const void* p, int64_t s_tok, int64_t s_head, int heads, uint32_t box_h, uint32_t box_n) {
    const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(heads), static_cast<uint64_t>(a.n)};
    const uint64_t strides[2] = {static_cast<uint64_t>(s_head) * 2, static_cast<uint64_t>(s_tok) * 2};
    const uint32_t box[3] = {64, box_h, box_n};
    return make_tmap_3d(m, p, dt, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (int s = map(&tq, a.q, a.q_st, a.q_sh, a.hq, ta.grp, ta.pos)) return s;
  if (int s = map(&tk, a.k, a.k_st, a.k_sh, a.hk, 1, kPromptKeys)) return s;
  if (int s = map(&tv, a.v, a.v_st, a.v_sh, a.hk, 1, kPromptKeys)) return s;
  const int64_t slots = a.n / ta.block + a.b + 2;
  prompt_tile_kernel<D, T><<<static_cast<unsigned>(slots * a.hk), kPromptThreads, C::SMEM, st>>>(tq, tk, tv, ta);
  return check_launch("prompt_tile_kernel");
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
  a.n = static_cast<int>(n);
  a.b = static_cast<int>(b);
  a.hq = static_cast<int>(hq);
  a.hk = static_cast<int>(hk);
  a.d = static_cast<int>(d);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The tensor-core kernel: rows that TMA can copy, a positive scale (it takes maxima before it scales), and blocks that
  // a grid can number.  (A dimension of one has any stride.)
  if (hq == 1) a.q_sh = d;
  if (hk == 1) a.k_sh = a.v_sh = d;
  if (n == 1) {
    a.q_st = a.q_sh * hq;
    a.k_st = a.k_sh * hk;
    a.v_st = a.v_sh * hk;
  }
  if ((d == 64 || d == 128) && hq / hk <= 128 && softmax_scale > 0.f && softmax_scale <= 3.402823466e38f &&
      tma_rows(q, a.q_st, a.q_sh) && tma_rows(k, a.k_st, a.k_sh) && tma_rows(v, a.v_st, a.v_sh) &&
      reinterpret_cast<uintptr_t>(out) % 16 == 0 && (n / (128 / (hq / hk)) + b + 2) * hk <= INT32_MAX) {
    if (dtype == BW_DTYPE_BF16) return d == 128 ? launch_tiles<128, __nv_bfloat16>(a, st) : launch_tiles<64, __nv_bfloat16>(a, st);
    return d == 128 ? launch_tiles<128, __half>(a, st) : launch_tiles<64, __half>(a, st);
  }
  return dtype == BW_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(a, st) : launch_rows<__half>(a, st);
}
