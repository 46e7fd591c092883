// Rotary positions and the paged int8 KV cache: rotate, quantise as written, read back, move.
//
// Rotation.  Pair i of a head's first `rot` elements turns by the angle theta = pos * f_i:
//   (a, b) -> m (a cos theta - b sin theta, a sin theta + b cos theta)
// with pairs (i, i + rot/2) (half) or (2i, 2i + 1) (interleaved).  f_i comes as a 64-bit fixed-point
// number of turns per position, round(f_i / 2 pi * 2^64), so pos * step modulo 2^64 is the angle's
// fraction of a turn with no range reduction and no rounding: at position 131071 a fp32 product
// pos * f_i is off by up to 4e-3 radians, this by 2e-7 (the fraction's own rounding to fp32).
// No sine table is read; the sines cost one sincospi per pair and token.
//
// Quantisation.  One fp32 scale per token and head, s = max|x| / 127 (NaN ignored, 0 for a row of
// zeros), code = clamp(rne(x / s), +-127) with the IEEE quotient (NaN -> 0).  Rotated keys are
// quantised from their 32-bit values: rounding them to 16 bits first would add an error of the
// order of a bf16 ulp to codes of 1/127 of the row's maximum.
#include <stdio.h>

#include <type_traits>

#include "kv_cache.cuh"
#include "quant_math.cuh"

namespace bw {

int check_kv_cache(const KvCache& c, int64_t b, const char* op) {
  if (c.pages < 0 || c.heads < 1 || c.page < 1 || c.d < 1 || c.d > kKvMaxDim)
    return fail(BW_ERR_INVALID_ARGUMENT, "%s: need pages >= 0, heads >= 1, page >= 1 and 1 <= d <= %d", op, kKvMaxDim);
  if (c.table_cols < 0 || c.table_ld < c.table_cols)
    return fail(BW_ERR_INVALID_ARGUMENT, "%s: table row stride too small", op);
  if (c.pages > 0 && (!c.k || !c.v || !c.ks || !c.vs)) return fail(BW_ERR_INVALID_ARGUMENT, "%s: null cache pointer", op);
  if (b > 0 && c.table_cols > 0 && !c.table) return fail(BW_ERR_INVALID_ARGUMENT, "%s: null table", op);
  return BW_OK;
}

// ---------------------------------------------------------------------------
// rotation and quantised write
// ---------------------------------------------------------------------------
struct RowSet {  // [b, t, heads, d] with unit stride in d
  const void* p;
  int64_t sb, st, sh;
  int heads;
};

struct RotArgs {
  RowSet q, k, v;      // v only where a cache is written
  void* q_out;         // contiguous [b, t, heads, d]
  void* k_out;         // the same, where no cache is written
  int64_t b, t;
  int d, rot, interleaved;
  float mag;
  const void* pos;     // [b, t], 32 or 64 bits
  int pos64;
  const unsigned long long* step;  // [rot / 2] turns per position, 2^-64 each
  KvCache cache;
  const int* start;    // [b] first slot
  const int* counts;   // [b] tokens of a sequence, or null: all t
};

__device__ __forceinline__ void turn(int64_t pos, unsigned long long step, float mag, float& co, float& si) {
  const unsigned long long ph = static_cast<unsigned long long>(pos) * step;
  // the top 32 bits as a signed fraction of half a turn in [-1, 1)
  const float t = static_cast<float>(static_cast<int>(ph >> 32)) * 0x1p-31f;
  sincospif(t, &si, &co);
  co *= mag;
  si *= mag;
}

__device__ __forceinline__ int64_t position_of(const RotArgs& a, int64_t tok) {
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[tok] : static_cast<int64_t>(static_cast<const int*>(a.pos)[tok]);
}

// Element e of a row, rotated if the row turns.
template <typename T>
__device__ __forceinline__ float row_value(const RotArgs& a, const T* x, int e, bool turns, int64_t pos) {
  if (!turns || e >= a.rot) return to_f32(x[e]);
  const int half = a.rot / 2;
  const int i = a.interleaved ? e >> 1 : (e < half ? e : e - half);
  const bool second = a.interleaved ? (e & 1) : (e >= half);
  const int other = a.interleaved ? (e ^ 1) : (second ? e - half : e + half);
  float co, si;
  turn(pos, a.step[i], a.mag, co, si);
  const float x0 = to_f32(x[e]), x1 = to_f32(x[other]);
  return second ? x1 * si + x0 * co : x0 * co - x1 * si;
}

// Any layout: one warp per (token, head) row.
template <typename T, bool WRITE>
__global__ void __launch_bounds__(256) rotary_rows_kernel(const __grid_constant__ RotArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t per_tok = a.q.heads + a.k.heads + a.v.heads;
  const int64_t rows = a.b * a.t * per_tok;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int64_t tok = r / per_tok;
    int h = static_cast<int>(r - tok * per_tok);
    const int64_t b = tok / a.t, t = tok - b * a.t;
    const int which = h < a.q.heads ? 0 : (h < a.q.heads + a.k.heads ? 1 : 2);
    h -= which == 0 ? 0 : (which == 1 ? a.q.heads : a.q.heads + a.k.heads);
    const RowSet& s = which == 0 ? a.q : (which == 1 ? a.k : a.v);
    const T* x = static_cast<const T*>(s.p) + b * s.sb + t * s.st + h * s.sh;
    const bool turns = which < 2 && a.rot > 0;
    const int64_t pos = turns ? position_of(a, tok) : 0;
    if (!WRITE || which == 0) {
      T* y = static_cast<T*>(which == 0 ? a.q_out : a.k_out) + (tok * s.heads + h) * a.d;
      for (int e = lane; e < a.d; e += 32) y[e] = from_f32<T>(row_value<T>(a, x, e, turns, pos));
      continue;
    }
    if (a.counts != nullptr && t >= a.counts[b]) continue;
    const int64_t row0 = kv_row(a.cache, b, static_cast<int64_t>(a.start[b]) + t);
    if (row0 < 0) continue;
    const int64_t row = row0 + static_cast<int64_t>(h) * a.cache.page;
    float v[kKvMaxDim / 32];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kKvMaxDim / 32; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < a.d ? row_value<T>(a, x, e, turns, pos) : 0.f;
      m = fmaxf(m, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float sc = __fdiv_rn(m, 127.0f);
    const float rcp = __frcp_rn(sc);
    int8_t* q = (which == 1 ? a.cache.k : a.cache.v) + row * a.d;
#pragma unroll
    for (int i = 0; i < kKvMaxDim / 32; ++i) {
      const int e = lane + 32 * i;
      if (e < a.d) q[e] = quant_fast<BW_DTYPE_F32>(v[i], sc, rcp);
    }
    if (lane == 0) (which == 1 ? a.cache.ks : a.cache.vs)[row] = sc;
  }
}

// Eight 16-bit values of a 16-byte chunk <-> fp32.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
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
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Codes of 16 values of a row with scale sc, rcp = RN(1 / sc): clamp(rne(RN(x / sc)), +-127), NaN -> 0.
// The IEEE quotient without a division (Markstein 1990): q = RN(x rcp), and twice q = RN(q + (x - q sc) rcp)
// with the remainder exact in an FMA; the first step leaves q within an ulp of x / sc, the second rounds it
// correctly.  Adding 1.5 * 2^23 rounds to the nearest even integer and leaves the code in the low byte;
// |x| <= 127 sc keeps it in range.  Rows whose remainders could be subnormal, or with a NaN or an infinity,
// take the divisions.  (Multiplying once and dividing only near a half, as the weight quantisers do, does not
// pay here: bf16 values over a bf16 maximum meet exact halves in almost every warp.)
__device__ __forceinline__ void codes16(const float* x, float sc, float rcp, uint2& lo, uint2& hi) {
  constexpr float kMagic = 12582912.0f;
  float y[16];
  const float2 s2 = make_float2(-sc, -sc), r2 = make_float2(rcp, rcp);
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 v = make_float2(x[i], x[i + 1]);
    sum = __fadd2_rn(sum, make_float2(fabsf(v.x), fabsf(v.y)));
    float2 q = __fmul2_rn(v, r2);
    q = __ffma2_rn(__ffma2_rn(q, s2, v), r2, q);
    q = __ffma2_rn(__ffma2_rn(q, s2, v), r2, q);
    const float2 z = __fadd2_rn(q, make_float2(kMagic, kMagic));
    y[i] = z.x;
    y[i + 1] = z.y;
  }
  if (!(sum.x + sum.y <= 3.402823466e38f) || !(sc > 0x1p-100f && sc <= 3.402823466e38f)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = kMagic + static_cast<float>(quant_one<BW_DTYPE_F32>(x[i], sc));
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __byte_perm(__float_as_uint(y[4 * i]), __float_as_uint(y[4 * i + 1]), 0x0040);
    const uint32_t b = __byte_perm(__float_as_uint(y[4 * i + 2]), __float_as_uint(y[4 * i + 3]), 0x0040);
    w[i] = __byte_perm(a, b, 0x5410);
  }
  lo = make_uint2(w[0], w[1]);
  hi = make_uint2(w[2], w[3]);
}

// Aligned rows of D = 16 L elements, rot a multiple of 16.  L lanes hold a row, 16 elements each in two
// 16-byte chunks: of the part that turns, lane j elements 8 j .. and rot/2 + 8 j .., so every pair of either
// layout lies in one lane; the rest, and rows that do not turn, in the same way.  A CTA's 256 threads hold
// the row groups of one to sixteen tokens and compute each of their sines once, one a thread, into shared
// memory; a group takes every `gpt`-th row of its token.  Bound by the bytes where tokens are many (which
// wants many warps: with each lane's sines in its registers four warps a scheduler did not cover the
// latency), by latency where they are few, for which the host spreads a token over more groups.
template <typename T, int L, bool WRITE, bool INTER>
__global__ void __launch_bounds__(256, WRITE ? 3 : 4) rotary_vec_kernel(const __grid_constant__ RotArgs a, int gpt) {
  constexpr int D = 16 * L;
  // (cos, sin) of the CTA's tokens' pairs: 256 / (gpt L) tokens of rot / 2 <= 8 L pairs, so gpt is 8 at least
  __shared__ __align__(16) float2 turns_of[256];
  const int j = threadIdx.x % L;
  const int64_t group = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int64_t tok = group / gpt;
  const int g = static_cast<int>(group - tok * gpt);
  const int half = a.rot / 2;
  // gpt * L is a power of two: whole tokens in a CTA, or a part of one
  const int in_cta = max(1, 256 / (gpt * L));
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * 256 / (gpt * L);
  const int64_t b = tok / a.t, t = tok - b * a.t;
  const bool turns = j < a.rot / 16;
  const int e0 = turns ? 8 * j : a.rot / 2 + 8 * j;  // (the rest starts at rot, at lane rot / 16)
  const int e1 = turns ? a.rot / 2 + 8 * j : D / 2 + 8 * j;
  const int hq = a.q.heads, hqk = hq + a.k.heads;
  const int rows = tok < a.b * a.t ? hqk + a.v.heads : 0;  // (the same for a whole group: the shuffles stay inside one)
  int64_t krow = -1;
  if (WRITE && rows > 0 && (a.counts == nullptr || t < a.counts[b]))
    krow = kv_row(a.cache, b, static_cast<int64_t>(a.start[b]) + t);
  const unsigned lanes = L == 32 ? 0xffffffffu : ((1u << L) - 1u) << ((threadIdx.x & 31) / L * L);
  // The next row is on its way while one is turned, the first while the sines are computed.  8191 tokens of 72
  // rows: 56 us, 5.4 TB/s; two rows ahead 60, three 68 (their registers spill).  The write of 4096 tokens' 32
  // query rows with 16 rows into the cache: 27 us, 3.4 TB/s (24 without any quotient: three CTAs an SM and two
  // and a third waves more than the instructions).
  auto fetch = [&](int h, uint4 (&raw)[2]) {
    if (h >= rows) return;
    const int which = h < hq ? 0 : (h < hqk ? 1 : 2);
    const int hh = which == 0 ? h : (which == 1 ? h - hq : h - hqk);
    const RowSet& s = which == 0 ? a.q : (which == 1 ? a.k : a.v);
    const T* x = static_cast<const T*>(s.p) + b * s.sb + t * s.st + hh * s.sh;
    raw[0] = *reinterpret_cast<const uint4*>(x + (which == 2 ? 8 * j : e0));
    raw[1] = *reinterpret_cast<const uint4*>(x + (which == 2 ? D / 2 + 8 * j : e1));
  };
  uint4 next[2];
  fetch(g, next);
  for (int e = threadIdx.x; e < in_cta * half; e += 256) {
    const int k = e / half;
    if (tok0 + k < a.b * a.t) {
      float co, si;
      turn(position_of(a, tok0 + k), a.step[e - k * half], a.mag, co, si);
      turns_of[e] = make_float2(co, si);
    }
  }
  __syncthreads();
  // pairs of the lane: eight of the half layout, four of each chunk of the interleaved one
  const float4* cs0 = reinterpret_cast<const float4*>(turns_of + static_cast<int>(tok - tok0) * half) +
                      (INTER ? e0 / 4 : 4 * j);
  const float4* cs1 = INTER ? cs0 - e0 / 4 + e1 / 4 : cs0 + 2;
#pragma unroll 1
  for (int h = g; h < rows; h += gpt) {
    const uint4 raw[2] = {next[0], next[1]};
    fetch(h + gpt, next);
    const int which = h < hq ? 0 : (h < hqk ? 1 : 2);
    const int hh = which == 0 ? h : (which == 1 ? h - hq : h - hqk);
    const bool plain = which == 2;  // values do not turn
    const int f0 = plain ? 8 * j : e0, f1 = plain ? D / 2 + 8 * j : e1;
    float v[16];
    unpack8<T>(raw[0], v);
    unpack8<T>(raw[1], v + 8);
    if (turns && !plain) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {  // two pairs
        const float4 cs = p < 2 ? cs0[p] : cs1[p - 2];
        // half layout: elements 2 p, 2 p + 1 with their partners 8 on; interleaved: four neighbours
        float& x0 = v[INTER ? 4 * p : 2 * p];
        float& x1 = v[INTER ? 4 * p + 1 : 2 * p + 8];
        float& y0 = v[INTER ? 4 * p + 2 : 2 * p + 1];
        float& y1 = v[INTER ? 4 * p + 3 : 2 * p + 9];
        const float u0 = x0, u1 = x1, w0 = y0, w1 = y1;
        x0 = u0 * cs.x - u1 * cs.y;
        x1 = u0 * cs.y + u1 * cs.x;
        y0 = w0 * cs.z - w1 * cs.w;
        y1 = w0 * cs.w + w1 * cs.z;
      }
    }
    if (!WRITE || which == 0) {
      T* y = static_cast<T*>(which == 0 ? a.q_out : a.k_out) + (tok * (which == 0 ? hq : a.k.heads) + hh) * D;
      *reinterpret_cast<uint4*>(y + f0) = pack8<T>(v);
      *reinterpret_cast<uint4*>(y + f1) = pack8<T>(v + 8);
      continue;
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(lanes, m, o));
    if (krow < 0) continue;
    const int64_t row = krow + static_cast<int64_t>(hh) * a.cache.page;
    const float sc = __fdiv_rn(m, 127.0f);
    const float rcp = __frcp_rn(sc);
    int8_t* q = (which == 1 ? a.cache.k : a.cache.v) + row * D;
    uint2 lo, hi;
    codes16(v, sc, rcp, lo, hi);
    *reinterpret_cast<uint2*>(q + f0) = lo;
    *reinterpret_cast<uint2*>(q + f1) = hi;
    if (j == 0) (which == 1 ? a.cache.ks : a.cache.vs)[row] = sc;
  }
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
static bool rows_aligned(const RowSet& s) {
  return s.heads == 0 || (aligned16(s.p) && s.sb % 8 == 0 && s.st % 8 == 0 && s.sh % 8 == 0);
}

template <typename T, int L>
static int launch_rotary_vec(const RotArgs& a, bool write, cudaStream_t st) {
  // Row groups of a token: eight (a lane's sines then serve many rows), more where the tokens alone do not
  // fill the SMs, up to one for each row.
  const int rows = a.q.heads + a.k.heads + a.v.heads;
  const int64_t tokens = a.b * a.t;
  int gpt = 8;
  while (gpt < rows && tokens * gpt * L < 1024L * num_sms()) gpt *= 2;
  const int64_t blocks = (tokens * gpt * L + 255) / 256;
  if (blocks > INT32_MAX) return fail(BW_ERR_INVALID_ARGUMENT, "rotary: too many tokens");
  const unsigned grid = static_cast<unsigned>(blocks);
  if (write) {
    if (a.interleaved) rotary_vec_kernel<T, L, true, true><<<grid, 256, 0, st>>>(a, gpt);
    else rotary_vec_kernel<T, L, true, false><<<grid, 256, 0, st>>>(a, gpt);
  } else {
    if (a.interleaved) rotary_vec_kernel<T, L, false, true><<<grid, 256, 0, st>>>(a, gpt);
    else rotary_vec_kernel<T, L, false, false><<<grid, 256, 0, st>>>(a, gpt);
  }
  return check_launch("rotary_vec_kernel");
}

template <typename T>
static int launch_rotary(const RotArgs& a, bool write, cudaStream_t st) {
  const int64_t rows = a.b * a.t * (a.q.heads + a.k.heads + a.v.heads);
  if (rows == 0) return BW_OK;
  if (a.rot % 16 == 0 && rows_aligned(a.q) && rows_aligned(a.k) && rows_aligned(a.v) && aligned16(a.q_out) &&
      aligned16(a.k_out) && aligned16(a.cache.k) && aligned16(a.cache.v)) {
    switch (a.d) {
      case 32: return launch_rotary_vec<T, 2>(a, write, st);
      case 64: return launch_rotary_vec<T, 4>(a, write, st);
      case 128: return launch_rotary_vec<T, 8>(a, write, st);
      case 256: return launch_rotary_vec<T, 16>(a, write, st);
      default: break;
    }
  }
  const int64_t blocks = (rows + 7) / 8;
  const int grid = static_cast<int>(blocks < 16L * num_sms() ? blocks : 16L * num_sms());
  if (write) rotary_rows_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else rotary_rows_kernel<T, false><<<grid, 256, 0, st>>>(a);
  return check_launch("rotary_rows_kernel");
}

static int check_rows(const RowSet& s, int64_t b, int64_t t, int d, const char* name, const char* op) {
  if (s.heads < 0) return fail(BW_ERR_INVALID_ARGUMENT, "%s: need %s heads >= 0", op, name);
  if (s.heads > 0 && b > 0 && t > 0 && !s.p) return fail(BW_ERR_INVALID_ARGUMENT, "%s: null pointer (%s)", op, name);
  if (s.sb < 0 || s.st < 0 || s.sh < 0) return fail(BW_ERR_INVALID_ARGUMENT, "%s: negative stride (%s)", op, name);
  return BW_OK;
}

static int check_rot(const RotArgs& a, int dtype, const char* op) {
  if (dtype != BW_DTYPE_F16 && dtype != BW_DTYPE_BF16)
    return fail(BW_ERR_INVALID_ARGUMENT, "%s: inputs must be fp16 or bf16 (dtype %d)", op, dtype);
  if (a.b < 0 || a.t < 0 || a.d < 1 || a.d > kKvMaxDim)
    return fail(BW_ERR_INVALID_ARGUMENT, "%s: need b, t >= 0 and 1 <= d <= %d", op, kKvMaxDim);
  if (a.b > INT32_MAX || a.t > INT32_MAX) return fail(BW_ERR_INVALID_ARGUMENT, "%s: dimension too large", op);
  if (a.rot < 0 || a.rot > a.d || a.rot % 2) return fail(BW_ERR_INVALID_ARGUMENT, "%s: need an even rot <= d", op);
  if (int s = check_rows(a.q, a.b, a.t, a.d, "q", op)) return s;
  if (int s = check_rows(a.k, a.b, a.t, a.d, "k", op)) return s;
  if (int s = check_rows(a.v, a.b, a.t, a.d, "v", op)) return s;
  if (a.rot > 0 && a.b > 0 && a.t > 0 && (!a.pos || !a.step))
    return fail(BW_ERR_INVALID_ARGUMENT, "%s: null pointer (positions or steps)", op);
  return BW_OK;
}

// ---------------------------------------------------------------------------
// read back
// ---------------------------------------------------------------------------
struct ReadArgs {
  KvCache c;
  int64_t layers, layer_rows;  // rows of one layer in codes and scales
  int64_t b, n;
  const int* start;  // [b] or null: 0
  const int* lens;   // [b] or null: n
  void* k_out;       // [layers, b, n, heads, d]
  void* v_out;
};

// Any layout: one warp per (layer, sequence, slot, head) row of k and of v.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_rows_kernel(const __grid_constant__ ReadArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.layers * a.b * a.n * a.c.heads;
  for (int64_t r = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; r < rows;
       r += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int64_t tok = r / a.c.heads, h = r - tok * a.c.heads;
    const int64_t lb = tok / a.n, i = tok - lb * a.n;
    const int64_t layer = lb / a.b, b = lb - layer * a.b;
    int64_t row = -1;
    if (a.lens == nullptr || i < a.lens[b]) row = kv_row(a.c, b, (a.start != nullptr ? a.start[b] : 0) + i);
    if (row >= 0) row += layer * a.layer_rows + h * a.c.page;
    const float ks = row >= 0 ? a.c.ks[row] : 0.f, vs = row >= 0 ? a.c.vs[row] : 0.f;
    T* ko = static_cast<T*>(a.k_out) + r * a.c.d;
    T* vo = static_cast<T*>(a.v_out) + r * a.c.d;
    for (int e = lane; e < a.c.d; e += 32) {
      ko[e] = from_f32<T>(row >= 0 ? static_cast<float>(a.c.k[row * a.c.d + e]) * ks : 0.f);
      vo[e] = from_f32<T>(row >= 0 ? static_cast<float>(a.c.v[row * a.c.d + e]) * vs : 0.f);
    }
  }
}

// 8 codes -> 8 values, 16 bytes.
template <typename T>
__device__ __forceinline__ uint4 values8(const uint2& c, float s) {
  // code + 128 in the low byte of 2^23, less 2^23 + 128: an addition where an int-to-float conversion runs at
  // a quarter of the rate (and bound the whole read)
  const uint32_t w[2] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u};
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    f[i] = (__uint_as_float(__byte_perm(w[i >> 2], 0x4B000000u, 0x7440 | (i & 3))) - 8388736.0f) * s;
  return pack8<T>(f);
}

// 32 bytes in one store (a whole sector), first to leave L2.
__device__ __forceinline__ void st_global_32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// Aligned rows of D = 16 C elements, C a power of two: 16 codes of k and of v -> one 32-byte store each.  A
// warp has one head and reads consecutive slots, which lie side by side in a page; the CTA's eight warps have
// eight heads, which lie side by side in the output.  UNROLL slots a lane are on their way at once.
// blockIdx.x: slots; y: layer and sequence.
template <typename T, int C>
__global__ void __launch_bounds__(256) kv_read_vec_kernel(const __grid_constant__ ReadArgs a) {
  constexpr int UNROLL = 2, ACROSS = 32 / C, SLOTS = ACROSS * UNROLL;
  const int lane = threadIdx.x & 31;
  const int ch = lane % C;
  const unsigned layer = blockIdx.y / static_cast<unsigned>(a.b);
  const int64_t b = blockIdx.y - layer * static_cast<unsigned>(a.b);
  const int64_t start = a.start != nullptr ? a.start[b] : 0;
  const int64_t len = min(a.lens != nullptr ? static_cast<int64_t>(a.lens[b]) : a.n, a.n);
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * SLOTS + lane / C;
  int64_t row[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    row[u] = i0 + u * ACROSS < len ? kv_row(a.c, b, start + i0 + u * ACROSS) : -1;
    if (row[u] >= 0) row[u] += layer * a.layer_rows;
  }
  const int8_t* codes = blockIdx.z ? a.c.v : a.c.k;
  const float* scales = blockIdx.z ? a.c.vs : a.c.ks;
  uint4* out = static_cast<uint4*>(blockIdx.z ? a.v_out : a.k_out);
  for (int h = threadIdx.x >> 5; h < a.c.heads; h += 8) {
    uint4 x[UNROLL];
    float sc[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      sc[u] = 0.f;
      if (row[u] < 0) continue;
      const int64_t r = row[u] + static_cast<int64_t>(h) * a.c.page;
      x[u] = __ldg(reinterpret_cast<const uint4*>(codes + r * (16 * C)) + ch);
      sc[u] = __ldg(scales + r);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t i = i0 + u * ACROSS;
      if (i >= a.n) continue;
      st_global_32(out + (((blockIdx.y * a.n + i) * a.c.heads + h) * C + ch) * 2,
                   values8<T>(make_uint2(x[u].x, x[u].y), sc[u]), values8<T>(make_uint2(x[u].z, x[u].w), sc[u]));
    }
  }
}

template <typename T, int C>
static int launch_read_vec(const ReadArgs& a, cudaStream_t st) {
  constexpr int SLOTS = 32 / C * 2;
  const dim3 grid(static_cast<unsigned>((a.n + SLOTS - 1) / SLOTS), static_cast<unsigned>(a.layers * a.b), 2);
  kv_read_vec_kernel<T, C><<<grid, 256, 0, st>>>(a);
  return check_launch("kv_read_vec_kernel");
}

template <typename T>
static int launch_read(const ReadArgs& a, cudaStream_t st) {
  if (a.layers * a.b <= 65535 && aligned16(a.c.k) && aligned16(a.c.v) &&
      (reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)) % 32 == 0) {
    switch (a.c.d) {
      case 32: return launch_read_vec<T, 2>(a, st);
      case 64: return launch_read_vec<T, 4>(a, st);
      case 128: return launch_read_vec<T, 8>(a, st);
      case 256: return launch_read_vec<T, 16>(a, st);
      default: break;
    }
  }
  const int64_t blocks = (a.layers * a.b * a.n * a.c.heads + 7) / 8;
  const int grid = static_cast<int>(blocks < 16L * num_sms() ? blocks : 16L * num_sms());
  kv_read_rows_kernel<T><<<grid, 256, 0, st>>>(a);
  return check_launch("kv_read_rows_kernel");
}

// ---------------------------------------------------------------------------
// move accepted nodes
// ---------------------------------------------------------------------------
// One CTA per (sequence, head, layer): the accepted rows are all read before the first is written
// (a node's slot may be another one's target), so the order of `path` does not matter.
__global__ void __launch_bounds__(256) kv_move_kernel(const __grid_constant__ KvCache c, int64_t layer_rows, int t,
                                                      const int* __restrict__ start, const int* __restrict__ path,
                                                      int64_t path_ld, const int* __restrict__ taken) {
  __shared__ int8_t buf[2][kTreeMaxNodes * kKvMaxDim];
  __shared__ float sc[2][kTreeMaxNodes];
  __shared__ int64_t src[kTreeMaxNodes], dst[kTreeMaxNodes];
  const int64_t b = blockIdx.x, h = blockIdx.y, layer = blockIdx.z;
  int n = taken[b];
  n = n < t - 1 ? n : t - 1;
  if (n <= 0) return;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int node = path[b * path_ld + i];
    int64_t s = -1, d = -1;
    if (node >= 0 && node < t) {
      s = kv_row(c, b, static_cast<int64_t>(start[b]) + node);
      d = kv_row(c, b, static_cast<int64_t>(start[b]) + 1 + i);
    }
    const bool ok = s >= 0 && d >= 0 && s != d;
    src[i] = ok ? layer * layer_rows + h * c.page + s : -1;
    dst[i] = ok ? layer * layer_rows + h * c.page + d : -1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * c.d; e += blockDim.x) {
    const int i = e / c.d, j = e - i * c.d;
    if (src[i] < 0) continue;
    buf[0][e] = c.k[src[i] * c.d + j];
    buf[1][e] = c.v[src[i] * c.d + j];
    if (j == 0) {
      sc[0][i] = c.ks[src[i]];
      sc[1][i] = c.vs[src[i]];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * c.d; e += blockDim.x) {
    const int i = e / c.d, j = e - i * c.d;
    if (src[i] < 0) continue;
    c.k[dst[i] * c.d + j] = buf[0][e];
    c.v[dst[i] * c.d + j] = buf[1][e];
    if (j == 0) {
      c.ks[dst[i]] = sc[0][i];
      c.vs[dst[i]] = sc[1][i];
    }
  }
}

// Aligned rows of a multiple of 16 bytes: one CTA per (sequence, layer), so the slots are looked up once for
// all heads; four heads' rows at a time are read into registers (16-byte chunks), then written.
template <int PER>  // chunks of a head's k and v rows a thread holds
__global__ void __launch_bounds__(128) kv_move_vec_kernel(const __grid_constant__ KvCache c, int64_t layer_rows, int t,
                                                          const int* __restrict__ start, const int* __restrict__ path,
                                                          int64_t path_ld, const int* __restrict__ taken) {
  constexpr int HEADS = 4;
  __shared__ int64_t src[kTreeMaxNodes], dst[kTreeMaxNodes];
  const int64_t b = blockIdx.x, layer = blockIdx.y;
  int n = taken[b];
  n = n < t - 1 ? n : t - 1;
  if (n <= 0) return;
  if (threadIdx.x < n) {
    const int node = path[b * path_ld + threadIdx.x];
    int64_t s = -1, d = -1;
    if (node >= 0 && node < t) {
      s = kv_row(c, b, static_cast<int64_t>(start[b]) + node);
      d = kv_row(c, b, static_cast<int64_t>(start[b]) + 1 + threadIdx.x);
    }
    const bool ok = s >= 0 && d >= 0 && s != d;
    src[threadIdx.x] = ok ? layer * layer_rows + s : -1;
    dst[threadIdx.x] = ok ? layer * layer_rows + d : -1;
  }
  __syncthreads();
  const int chunks = c.d / 16;           // of a row
  const int per_head = n * chunks;       // of k, and as many of v
  for (int h0 = 0; h0 < c.heads; h0 += HEADS) {
    uint4 buf[HEADS][PER];
    float sc[HEADS];
#pragma unroll
    for (int hh = 0; hh < HEADS; ++hh) {
      const int64_t hrow = static_cast<int64_t>(h0 + hh) * c.page;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int e = threadIdx.x + 128 * k;
        if (h0 + hh >= c.heads || e >= 2 * per_head) continue;
        const int r = (e < per_head ? e : e - per_head) / chunks, ch = (e < per_head ? e : e - per_head) - r * chunks;
        if (src[r] >= 0)
          buf[hh][k] = *(reinterpret_cast<const uint4*>((e < per_head ? c.k : c.v) + (src[r] + hrow) * c.d) + ch);
      }
      if (h0 + hh < c.heads && threadIdx.x < 2 * n) {
        const int r = threadIdx.x < n ? threadIdx.x : threadIdx.x - n;
        if (src[r] >= 0) sc[hh] = (threadIdx.x < n ? c.ks : c.vs)[src[r] + hrow];
      }
    }
    __syncthreads();  // these heads' rows are all read
#pragma unroll
    for (int hh = 0; hh < HEADS; ++hh) {
      const int64_t hrow = static_cast<int64_t>(h0 + hh) * c.page;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int e = threadIdx.x + 128 * k;
        if (h0 + hh >= c.heads || e >= 2 * per_head) continue;
        const int r = (e < per_head ? e : e - per_head) / chunks, ch = (e < per_head ? e : e - per_head) - r * chunks;
        if (src[r] >= 0)
          *(reinterpret_cast<uint4*>((e < per_head ? c.k : c.v) + (dst[r] + hrow) * c.d) + ch) = buf[hh][k];
      }
      if (h0 + hh < c.heads && threadIdx.x < 2 * n) {
        const int r = threadIdx.x < n ? threadIdx.x : threadIdx.x - n;
        if (src[r] >= 0) (threadIdx.x < n ? c.ks : c.vs)[dst[r] + hrow] = sc[hh];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// a draft tree's masks and positions
// ---------------------------------------------------------------------------
// parent[i] < i for a node of the tree; node 0 is the root.  Any other parent takes a node out of
// the tree: it sees nothing and stands at its sequence's own position.
__global__ void __launch_bounds__(kTreeMaxNodes) tree_positions_kernel(const int* __restrict__ parents, int64_t ld,
                                                                       const int* __restrict__ ctx, int t,
                                                                       unsigned long long* __restrict__ mask,
                                                                       int* __restrict__ pos) {
  __shared__ int up[kTreeMaxNodes];
  const int64_t b = blockIdx.x;
  const int i = threadIdx.x;
  if (i < t) up[i] = parents[b * ld + i];
  __syncthreads();
  if (i >= t) return;
  unsigned long long bits = 0;
  int at = i;
  while (at > 0 && up[at] >= 0 && up[at] < at) {  // strictly descending: ends
    bits |= 1ull << at;
    at = up[at];
  }
  bits = at == 0 ? bits | 1ull : 0ull;
  mask[b * t + i] = bits;
  pos[b * t + i] = (ctx != nullptr ? ctx[b] : 0) + (bits ? __popcll(bits) - 1 : 0);
}

static KvCache make_cache(void* k, void* v, float* ks, float* vs, int64_t pages, int64_t heads, int64_t page, int64_t d,
                          const int* table, int64_t table_ld, int64_t table_cols) {
  KvCache c;
  c.k = static_cast<int8_t*>(k);
  c.v = static_cast<int8_t*>(v);
  c.ks = ks;
  c.vs = vs;
  c.pages = pages;
  // out of int range: 0, which check_kv_cache refuses
  c.heads = heads > 0 && heads <= 65535 ? static_cast<int>(heads) : 0;
  c.page = page > 0 && page <= (1 << 24) ? static_cast<int>(page) : 0;
  c.shift = page_shift(c.page);
  c.d = d > 0 && d <= kKvMaxDim ? static_cast<int>(d) : 0;
  c.table = table;
  c.table_ld = table_ld;
  c.table_cols = table_cols >= 0 && table_cols <= INT32_MAX ? static_cast<int>(table_cols) : -1;
  return c;
}

}  // namespace bw

extern "C" int bw_rotary(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int hq, const void* k, int64_t k_sb,
                         int64_t k_st, int64_t k_sh, int hk, void* q_out, void* k_out, int dtype, int64_t b, int64_t t,
                         int64_t d, const void* positions, int positions64, const uint64_t* steps, float magnitude,
                         int64_t rot, int interleaved, void* stream) {
  using namespace bw;
  RotArgs a = {};
  a.q = {q, q_sb, q_st, q_sh, hq};
  a.k = {k, k_sb, k_st, k_sh, hk};
  a.q_out = q_out;
  a.k_out = k_out;
  a.b = b;
  a.t = t;
  a.d = d > 0 && d <= kKvMaxDim ? static_cast<int>(d) : 0;
  a.rot = rot >= 0 && rot <= kKvMaxDim ? static_cast<int>(rot) : -1;
  a.interleaved = interleaved;
  a.mag = magnitude;
  a.pos = positions;
  a.pos64 = positions64;
  a.step = reinterpret_cast<const unsigned long long*>(steps);
  if (int s = check_rot(a, dtype, "rotary")) return s;
  if (b == 0 || t == 0) return BW_OK;
  if ((hq > 0 && !q_out) || (hk > 0 && !k_out)) return fail(BW_ERR_INVALID_ARGUMENT, "rotary: null output pointer");
  if (int s = require_sm100()) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == BW_DTYPE_BF16 ? launch_rotary<__nv_bfloat16>(a, false, st) : launch_rotary<__half>(a, false, st);
}

extern "C" int bw_rotary_kv_write_int8(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int hq, const void* k,
                                       int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb,
                                       int64_t v_st, int64_t v_sh, void* q_out, int dtype, int64_t b, int64_t t,
                                       const void* positions, int positions64, const uint64_t* steps, float magnitude,
                                       int64_t rot, int interleaved, int8_t* cache_k, int8_t* cache_v, float* k_scale,
                                       float* v_scale, int64_t pages, int64_t heads, int64_t page, int64_t d,
                                       const int32_t* table, int64_t table_ld, int64_t table_cols,
                                       const int32_t* start, const int32_t* counts, void* stream) {
  using namespace bw;
  RotArgs a = {};
  a.cache = make_cache(cache_k, cache_v, k_scale, v_scale, pages, heads, page, d, table, table_ld, table_cols);
  if (int s = check_kv_cache(a.cache, b, "kv_write_int8")) return s;
  a.q = {q, q_sb, q_st, q_sh, hq};
  a.k = {k, k_sb, k_st, k_sh, a.cache.heads};
  a.v = {v, v_sb, v_st, v_sh, a.cache.heads};
  a.q_out = q_out;
  a.b = b;
  a.t = t;
  a.d = a.cache.d;
  a.rot = rot >= 0 && rot <= kKvMaxDim ? static_cast<int>(rot) : -1;
  a.interleaved = interleaved;
  a.mag = magnitude;
  a.pos = positions;
  a.pos64 = positions64;
  a.step = reinterpret_cast<const unsigned long long*>(steps);
  a.start = start;
  a.counts = counts;
  if (int s = check_rot(a, dtype, "kv_write_int8")) return s;
  if (b == 0 || t == 0) return BW_OK;
  if (!start || (hq > 0 && !q_out)) return fail(BW_ERR_INVALID_ARGUMENT, "kv_write_int8: null pointer");
  if (int s = require_sm100()) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == BW_DTYPE_BF16 ? launch_rotary<__nv_bfloat16>(a, true, st) : launch_rotary<__half>(a, true, st);
}

extern "C" int bw_kv_read_int8(const int8_t* cache_k, const int8_t* cache_v, const float* k_scale,
                               const float* v_scale, int64_t layers, int64_t pages, int64_t heads, int64_t page,
                               int64_t d, const int32_t* table, int64_t table_ld, int64_t table_cols,
                               const int32_t* start, const int32_t* lens, int64_t b, int64_t n, void* k_out,
                               void* v_out, int dtype, void* stream) {
  using namespace bw;
  ReadArgs a = {};
  a.c = make_cache(const_cast<int8_t*>(cache_k), const_cast<int8_t*>(cache_v), const_cast<float*>(k_scale),
                   const_cast<float*>(v_scale), pages, heads, page, d, table, table_ld, table_cols);
  if (int s = check_kv_cache(a.c, b, "kv_read_int8")) return s;
  if (layers < 0 || b < 0 || n < 0 || layers > INT32_MAX || b > INT32_MAX || n > INT32_MAX)
    return fail(BW_ERR_INVALID_ARGUMENT, "kv_read_int8: need 0 <= layers, b, n < 2^31");
  if (dtype != BW_DTYPE_F16 && dtype != BW_DTYPE_BF16)
    return fail(BW_ERR_INVALID_ARGUMENT, "kv_read_int8: outputs must be fp16 or bf16 (dtype %d)", dtype);
  if (layers == 0 || b == 0 || n == 0) return BW_OK;
  if (!k_out || !v_out) return fail(BW_ERR_INVALID_ARGUMENT, "kv_read_int8: null pointer");
  a.layers = layers;
  a.layer_rows = pages * heads * page;
  a.b = b;
  a.n = n;
  a.start = start;
  a.lens = lens;
  a.k_out = k_out;
  a.v_out = v_out;
  if (int s = require_sm100()) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == BW_DTYPE_BF16 ? launch_read<__nv_bfloat16>(a, st) : launch_read<__half>(a, st);
}

extern "C" int bw_kv_move_int8(int8_t* cache_k, int8_t* cache_v, float* k_scale, float* v_scale, int64_t layers,
                               int64_t pages, int64_t heads, int64_t page, int64_t d, const int32_t* table,
                               int64_t table_ld, int64_t table_cols, const int32_t* start, const int32_t* path,
                               int64_t path_ld, const int32_t* taken, int64_t b, int64_t t, void* stream) {
  using namespace bw;
  const KvCache c = make_cache(cache_k, cache_v, k_scale, v_scale, pages, heads, page, d, table, table_ld, table_cols);
  if (int s = check_kv_cache(c, b, "kv_move_int8")) return s;
  if (layers < 0 || layers > 65535 || b < 0 || b > INT32_MAX)
    return fail(BW_ERR_INVALID_ARGUMENT, "kv_move_int8: need 0 <= layers < 65536 and 0 <= b < 2^31");
  if (t < 0 || t > kTreeMaxNodes || path_ld < t)
    return fail(BW_ERR_INVALID_ARGUMENT, "kv_move_int8: need 0 <= t <= %d and a path row stride >= t", kTreeMaxNodes);
  if (layers == 0 || b == 0 || t <= 1) return BW_OK;
  if (!start || !path || !taken) return fail(BW_ERR_INVALID_ARGUMENT, "kv_move_int8: null pointer");
  if (int s = require_sm100()) return s;
  // chunks of 16 bytes that a thread of 128 holds for a head: at most (t - 1) rows of k and v; beyond four
  // (trees of 33 nodes and more at d = 128) the registers run out, and the rows go through shared memory
  const int64_t held = (2 * (t - 1) * (d / 16) + 127) / 128;
  if (d % 16 == 0 && held <= 4 && aligned16(cache_k) && aligned16(cache_v)) {
    const dim3 vgrid(static_cast<unsigned>(b), static_cast<unsigned>(layers));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (held <= 2)
      kv_move_vec_kernel<2><<<vgrid, 128, 0, st>>>(c, pages * heads * page, static_cast<int>(t), start, path, path_ld, taken);
    else
      kv_move_vec_kernel<4><<<vgrid, 128, 0, st>>>(c, pages * heads * page, static_cast<int>(t), start, path, path_ld, taken);
    return check_launch("kv_move_vec_kernel");
  }
  const dim3 grid(static_cast<unsigned>(b), static_cast<unsigned>(heads), static_cast<unsigned>(layers));
  kv_move_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(c, pages * heads * page, static_cast<int>(t),
                                                                      start, path, path_ld, taken);
  return check_launch("kv_move_kernel");
}

extern "C" int bw_tree_positions(const int32_t* parents, int64_t parents_ld, const int32_t* ctx_lens, int64_t b,
                                 int64_t t, uint64_t* mask, int32_t* positions, void* stream) {
  using namespace bw;
  if (b < 0 || b > INT32_MAX || t < 0 || t > kTreeMaxNodes || parents_ld < t)
    return fail(BW_ERR_INVALID_ARGUMENT, "tree_positions: need 0 <= t <= %d and a row stride >= t", kTreeMaxNodes);
  if (b == 0 || t == 0) return BW_OK;
  if (!parents || !mask || !positions) return fail(BW_ERR_INVALID_ARGUMENT, "tree_positions: null pointer");
  if (int s = require_sm100()) return s;
  tree_positions_kernel<<<static_cast<unsigned>(b), kTreeMaxNodes, 0, static_cast<cudaStream_t>(stream)>>>(
      parents, parents_ld, ctx_lens, static_cast<int>(t), reinterpret_cast<unsigned long long*>(mask), positions);
  return check_launch("tree_positions_kernel");
}
