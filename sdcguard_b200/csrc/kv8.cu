// Paged KV cache held in 8 bits (sm_100a): appending rotated keys and values, and attention over the cache.
//
// Cache of one layer: codes [num_blocks][2 (K, V)][kv_heads][16 tokens][128] E4M3, scales [num_blocks][kv_heads][2]
// float32. A value is code * scale; one scale serves the 16 tokens of a page for one kv head and K or V.
//
// append (`kv8_append_kernel`). k' = R(pos) n(k), v' = v in fp32 (n: optional RMSNorm with a weight, R: the rotation of
// the first `rotary` dims), one rounding to E4M3. The tokens of a call that follow one another in a page are its run;
// the page's tokens before the run are kept, those behind it are dead. The page's scale becomes
//     s' = max(s of the kept tokens, the least power of two with amax(run) <= 448 s', 2^-60)
// and kept codes move to it: code' = rne(code * s / s'). s / s' is a power of two, so a kept value changes only where
// it falls below E4M3's normal range. Powers of two make code * scale exact in bf16 and in fp32.
// A value that is not finite is stored as NaN and does not raise the scale.
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "tma_host.h"

namespace sdc {
namespace kv8 {

constexpr int D = 128;
constexpr int PAGE = 16;
// Biases of the decode kernel's weights and row sums (powers of two), see there.
constexpr float SUM_BIAS = 30.f;
constexpr float W_SCALE = 1.f / 65536.f;    // 2^(14 - SUM_BIAS)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
  return v;
}
// E4M3 pair (low 8 bits = lo) of two floats, round to nearest even; |x| <= 448 or NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two E4M3 codes (low 16 bits) -> two halves, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_h2_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ float2 h2_to_f2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// The least power of two s >= 2^-60 with amax <= 448 s: 448 = 1.75 * 2^8, so from amax's exponent and fraction.
__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -60 ? -60 : e;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
constexpr float FLOAT_MAX = 3.402823466e38f;
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= FLOAT_MAX; }

struct AppendParams {
  const __nv_bfloat16* qkv;   // [T] rows of (nq + 2 nkv) x 128, `ld` apart
  long long ld;
  int T, nq, nkv;
  const int* pos;             // [T]
  const long long* slots;     // [T] block * 16 + place; negative: not stored
  const __nv_bfloat16* qw;
  const __nv_bfloat16* kw;
  double eps;                 // keys decided in double
  float epsf;
  const float2* cs;           // [table_rows][rotary / 2] (cos, sin)
  int table_rows, rotary;
  __nv_bfloat16* q_out;       // [T][nq][128]
  uint8_t* codes;
  float* scales;
  long long capacity;         // num_blocks * 16
  const int* rows;            // check mode: the sampled tokens
  unsigned long long* check;
};

__device__ __forceinline__ const float2* angles_of(const AppendParams& p, int pos) {
  return p.cs + static_cast<long long>(pos) * (p.rotary / 2);
}
// The slot token t is stored at; -1: skipped; -2: its slot or position lies outside the cache or the table.
__device__ __forceinline__ long long slot_of(const AppendParams& p, int t) {
  const long long s = p.slots[t];
  if (s >= p.capacity) return -2;
  if (p.rotary > 0) {
    const int ps = p.pos[t];
    if (ps < 0 || ps >= p.table_rows) return -2;
  }
  return s < 0 ? -1 : s;
}

// How the 16 lanes of a half warp share a row: a lane holds two quads of dims, v[0..3] and v[4..7], such that v[i] and
// v[4 + i] are a rotation's pair, so no value crosses lanes. Halves: quads 4l and rotary / 2 + 4l, and behind the
// rotated part two neighbouring quads. Interleaved (INTER): dims 8l .. 8l + 7, the even ones in v[0..3].
template <bool INTER>
struct RowLane {
  int d0, d1, ci;      // dims of the two quads in memory, first (cos, sin) of the lane
  bool rot;
  __device__ __forceinline__ RowLane(int l, int rotary) {
    const int half = rotary / 2;
    ci = 4 * l;
    if (INTER) {
      d0 = 8 * l;
      d1 = d0 + 4;
      rot = d0 < rotary;
    } else {
      rot = 4 * l < half;
      d0 = rot ? 4 * l : rotary + 8 * (l - half / 4);
      d1 = rot ? half + 4 * l : d0 + 4;
    }
  }
  __device__ __forceinline__ uint4 load(const __nv_bfloat16* row) const {
    const uint2 a = *reinterpret_cast<const uint2*>(row + d0), b = *reinterpret_cast<const uint2*>(row + d1);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) const {
    uint4 w = u;
    if (INTER)
      w = make_uint4(__byte_perm(u.x, u.y, 0x5410), __byte_perm(u.z, u.w, 0x5410), __byte_perm(u.x, u.y, 0x7632),
                     __byte_perm(u.z, u.w, 0x7632));
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(x[i] << 16);
      v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ uint4 pack(const float (&v)[8]) const {
    if (INTER)
      return make_uint4(pack_bf16x2(v[0], v[4]), pack_bf16x2(v[1], v[5]), pack_bf16x2(v[2], v[6]), pack_bf16x2(v[3], v[7]));
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
  // The lane's cosines and sines from its position's row of the table.
  __device__ __forceinline__ void angles(const float2* cs, float (&c)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = i < 4 ? 1.f : 0.f;
    if (!rot) return;
    const float4* a = reinterpret_cast<const float4*>(cs + ci);
    const float4 x = __ldg(a), y = __ldg(a + 1);
    c[0] = x.x;
    c[1] = x.z;
    c[2] = y.x;
    c[3] = y.z;
    c[4] = x.y;
    c[5] = x.w;
    c[6] = y.y;
    c[7] = y.w;
  }
  // The codes of u[8] (scaled values) as the two words at d0 and d1.
  __device__ __forceinline__ uint2 codes(const float (&u)[8]) const {
    if (INTER)
      return make_uint2(e4m3x2(u[0], u[4]) | (e4m3x2(u[1], u[5]) << 16), e4m3x2(u[2], u[6]) | (e4m3x2(u[3], u[7]) << 16));
    return make_uint2(e4m3x2(u[0], u[1]) | (e4m3x2(u[2], u[3]) << 16), e4m3x2(u[4], u[5]) | (e4m3x2(u[6], u[7]) << 16));
  }
};

template <typename T>
__device__ __forceinline__ T half_warp_sum(T v) {
#pragma unroll
  for (int m = 8; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// 1 / sqrt(mean of squares + eps) of the row a half warp holds.
template <typename T>
__device__ __forceinline__ T norm_of(const T (&v)[8], T eps) {
  T ss = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
  return rsqrt(half_warp_sum(ss) * static_cast<T>(1.0 / D) + eps);
}
// Rotates the pairs (v[i], v[4 + i]) by c: four cosines, four sines (1 and 0 where nothing is rotated).
template <typename T>
__device__ __forceinline__ void rotate(T (&v)[8], const float (&c)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T a = v[i], b = v[4 + i], co = c[i], si = c[4 + i];
    v[i] = a * co - b * si;
    v[4 + i] = b * co + a * si;
  }
}

// d * inv as the float that rounds to the same E4M3 code: cut, with the last bit set where bits were lost, so that the
// second rounding sees on which side of a tie the value lies. Not finite (in fp32): NaN.
__device__ __forceinline__ float to_odd(double d, double inv) {
  if (!(fabs(d) <= FLOAT_MAX)) return __int_as_float(0x7fffffff);
  const double u = d * inv;
  const float f = __double2float_rz(u);
  return static_cast<double>(f) == u ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ float amax_of(const float (&v)[8], float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));      // passes over NaN
  return m;
}
__device__ __forceinline__ float finite_amax(const float (&v)[8], float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (finite(v[i])) m = fmaxf(m, fabsf(v[i]));
  return m;
}

// A key's row in double, weights `kw` (or null), angles at `cs` (of its position). Every lane of the warp takes part.
template <bool INTER>
__device__ __forceinline__ void exact_key(const __nv_bfloat16* row, const __nv_bfloat16* kw, const float2* cs, int rotary,
                                          double eps, int l, double (&d)[8]) {
  const RowLane<INTER> L(l, rotary);
  float v[8], c[8];
  L.unpack(L.load(row), v);
  L.angles(cs, c);
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = v[i];
  if (kw != nullptr) {
    const double inv = norm_of(d, eps);
    L.unpack(L.load(kw), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = d[i] * inv * v[i];
  }
  rotate(d, c);
}
// Its codes at scale 1 / up.
template <bool INTER>
__device__ __forceinline__ uint2 exact_codes(const __nv_bfloat16* row, const __nv_bfloat16* kw, const float2* cs, int rotary,
                                          double eps, int l, float up) {
  double d[8];
  exact_key<INTER>(row, kw, cs, rotary, eps, l, d);
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = to_odd(d[i], up);
  return RowLane<INTER>(l, rotary).codes(u);
}
// The largest finite magnitude among the lane's values, rounded up to a float.
template <bool INTER>
__device__ __forceinline__ float exact_amax(const __nv_bfloat16* row, const __nv_bfloat16* kw, const float2* cs, int rotary,
                                         double eps, int l) {
  double d[8];
  exact_key<INTER>(row, kw, cs, rotary, eps, l, d);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (fabs(d[i]) <= FLOAT_MAX) m = fmaxf(m, __double2float_ru(fabs(d[i])));
  return m;
}

// A CTA has one of two roles, by its index. Queries: a warp takes two tokens (a row per half warp) and eight heads, so
// the tokens' (cos, sin) are read once for eight rows, which are all in flight together. Keys and values: a warp takes
// one head and the runs that begin among TG consecutive tokens (up to 16 rows of one page), so one warp alone writes a
// page's scale and codes of a head; keys wait for the scale in shared memory, values as they were read in registers.
// TG = 1 gives each token of a decode step its own warps (latency); TG = 16 gives a page one warp and leaves none
// without work; TG = 4 lies between.
//
// Scales and codes are the correctly rounded ones of the formulas, so they do not depend on the order of operations
// here (a replay, another kernel or a CPU can compare bits). Values are exact products. Keys are computed in fp32; with
// u = 2^-24, the norm's factor errs by 10.5 u of itself (rsqrt 4, the sum of squares and its root 6.5), the products
// with it and the rotation by 4 u of the pair's length, at most sqrt(2) of the run's largest magnitude. Where a code
// differs within 11 u of the key plus 6 u of that magnitude, or the scale within 2^-19, the row is computed again in
// double: one pair of rows in thirty. (The sum of squares is fp32: keys stay below 2^60.)
//
// Measured (32 query, 8 kv heads, device time): 8 x 2048 tokens 60.5 us, 3.9 TB/s, bound by instructions and the latency
// of the keys' chain (rows, norm, scale, codes), 20 warps an SM; 256 x 1 token 6.3 us, 1 x 1 3.5 us, latency. At 8 x 2048
// one row a warp took 303 us, a row to a half warp 118, queries in warps of their own 91, keys waiting in shared memory
// instead of registers 63.
constexpr float KEY_RELATIVE = 11.f / 16777216.f, KEY_ABSOLUTE = 6.f / 16777216.f, SCALE_MARGIN = 32.f / 16777216.f;
constexpr int AW = 4;             // warps of a CTA
constexpr int QH = 8;             // heads of a query warp
constexpr int HALF = PAGE / 2;    // rows of a run that each half warp holds

template <bool INTER>
__device__ __forceinline__ void append_queries(const AppendParams& p, int group, int h0) {
  const int lane = threadIdx.x & 31, hw = lane >> 4;
  const int t = 2 * (group * AW + (threadIdx.x >> 5)) + hw;
  const RowLane<INTER> L(lane & 15, p.rotary);
  const bool in = t < p.T;
  const __nv_bfloat16* row = p.qkv + (in ? t : 0) * p.ld + static_cast<long long>(h0) * D;
  uint4 raw[QH];
#pragma unroll
  for (int j = 0; j < QH; ++j) raw[j] = in && h0 + j < p.nq ? L.load(row + j * D) : make_uint4(0, 0, 0, 0);
  const bool out = in && slot_of(p, t) == -2;
  float c[8] = {1.f, 1.f, 1.f, 1.f, 0.f, 0.f, 0.f, 0.f};
  if (in && !out) L.angles(angles_of(p, p.rotary > 0 ? p.pos[t] : 0), c);
  if (out) {                                              // a slot or position outside must not pass unseen
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __int_as_float(0x7fffffff);
  }
  float w[8];
  if (p.qw != nullptr) L.unpack(L.load(p.qw), w);
  __nv_bfloat16* dst = p.q_out + (static_cast<long long>(in ? t : 0) * p.nq + h0) * D;
#pragma unroll
  for (int j = 0; j < QH; ++j) {
    if (h0 + j >= p.nq) break;
    float v[8];
    L.unpack(raw[j], v);
    if (p.qw != nullptr) {
      const float inv = norm_of(v, p.epsf);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
    }
    rotate(v, c);
    const uint4 o = L.pack(v);
    if (in) {
      *reinterpret_cast<uint2*>(dst + j * D + L.d0) = make_uint2(o.x, o.y);
      *reinterpret_cast<uint2*>(dst + j * D + L.d1) = make_uint2(o.z, o.w);
    }
  }
}

template <int TG, bool INTER>
__device__ __forceinline__ void append_keys_values(const AppendParams& p, int t0, int u, float4 (*keep)[2][32]) {
  const int lane = threadIdx.x & 31, hw = lane >> 4, l = lane & 15;
  const bool is_k = u < p.nkv;
  const int kvh = is_k ? u : u - p.nkv;
  const __nv_bfloat16* col = p.qkv + static_cast<long long>(p.nq + u) * D;
  const RowLane<INTER> L(l, p.rotary);
  const RowLane<false> V(l, 0);                            // dims 8l .. 8l + 7 in order
  // the group's rows are on their way to L2 before its slots say which of them this warp stores
  if (t0 + (lane >> 1) < p.T && lane < 2 * TG)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(col + (t0 + (lane >> 1)) * p.ld + (lane & 1) * 64));
  // lane j looks at token t0 - 1 + j: the token before the group, the group, and the tokens a run may reach behind it
  const int tl = t0 - 1 + lane;
  const bool look = lane < TG + PAGE && tl >= 0 && tl < p.T;
  const int ps = look && is_k && p.rotary > 0 ? p.pos[tl] : 0;
  const long long sl = look ? slot_of(p, tl) : -1;
  const bool norm = is_k && p.kw != nullptr;
  float w[8];
  if (norm) L.unpack(L.load(p.kw), w);
  const long long before = __shfl_up_sync(0xffffffffu, sl, 1);
  const bool follows = lane > 0 && sl >= 0 && before >= 0 && sl == before + 1 && sl % PAGE != 0;
  const uint32_t chain = __ballot_sync(0xffffffffu, follows);
  uint32_t starts = __ballot_sync(0xffffffffu, sl >= 0 && !follows && lane >= 1 && lane <= TG);
  while (starts != 0) {
    const int first = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t rest = ~(chain >> 1 >> first);          // bit i: token first + 1 + i does not continue the run
    const int len = 1 + (rest == 0 ? 31 : __ffs(rest) - 1);   // <= 16: a run stays in its page
    const long long slot = __shfl_sync(0xffffffffu, sl, first);
    const long long blk = slot / PAGE;
    const int at = static_cast<int>(slot % PAGE);
    const __nv_bfloat16* rows = col + (t0 - 1 + first) * p.ld;
    float* sp = p.scales + (blk * p.nkv + kvh) * 2 + (is_k ? 0 : 1);
    const float old = at > 0 ? *sp : 0.f;
    uint8_t* page = p.codes + ((blk * 2 + (is_k ? 0 : 1)) * p.nkv + kvh) * (PAGE * D);
    float m = 0.f, s;
    if (is_k) {
      const auto place = [&](int j) { return min(2 * j + hw, len - 1); };   // a row of zeros pairs up with the last one
#pragma unroll 1
      for (int j0 = 0; 2 * j0 < len; j0 += 4) {
        uint4 raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          raw[j] = 2 * (j0 + j) + hw < len ? L.load(rows + (2 * (j0 + j) + hw) * p.ld) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (2 * (j0 + j) >= len) break;                  // (uniform)
          const int pos = __shfl_sync(0xffffffffu, ps, first + place(j0 + j));
          float v[8], c[8];
          L.unpack(raw[j], v);
          L.angles(angles_of(p, pos), c);
          if (norm) {
            const float inv = norm_of(v, p.epsf);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
          }
          rotate(v, c);
          m = amax_of(v, m);
          keep[j0 + j][0][lane] = make_float4(v[0], v[1], v[2], v[3]);
          keep[j0 + j][1][lane] = make_float4(v[4], v[5], v[6], v[7]);
        }
      }
      m = warp_max(m);
      const bool inf = m > FLOAT_MAX;                      // then the largest finite one
      if (inf) {
        m = 0.f;
        for (int j = 0; 2 * j < len; ++j) {
          const float4 a = keep[j][0][lane], b = keep[j][1][lane];
          const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          m = finite_amax(v, m);
        }
        m = warp_max(m);
      }
      s = scale_of(m);
      const bool exact = !norm && p.rotary == 0;
      if (!exact && scale_of(m * (1.f - SCALE_MARGIN)) != scale_of(m * (1.f + SCALE_MARGIN))) {
        float top = 0.f;
        for (int j = 0; 2 * j < len; ++j) {
          const int pos = __shfl_sync(0xffffffffu, ps, first + place(j));
          top = fmaxf(top, exact_amax<INTER>(rows + place(j) * p.ld, p.kw, angles_of(p, pos), p.rotary, p.eps, l));
        }
        s = scale_of(warp_max(top));
      }
      s = fmaxf(s, old);
      const float up = 1.f / s;
      const float far = exact ? 0.f : KEY_ABSOLUTE * m * up;
      const float up1 = exact ? up : up * (1.f + KEY_RELATIVE), up0 = exact ? up : up * (1.f - KEY_RELATIVE);
#pragma unroll 2
      for (int j = 0; 2 * j < len; ++j) {
        const float4 a = keep[j][0][lane], b = keep[j][1][lane];
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        float x[8], y[8];                                // the ends of the interval around the scaled key
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = copysignf(far, v[i]);
          x[i] = fmaf(v[i], up1, f);
          y[i] = fmaf(v[i], up0, -f);
        }
        uint2 code = L.codes(x);
        const uint2 other = L.codes(y);
        if (__any_sync(0xffffffffu, code.x != other.x || code.y != other.y || inf)) {
          const int pos = __shfl_sync(0xffffffffu, ps, first + place(j));
          code = exact_codes<INTER>(rows + place(j) * p.ld, p.kw, angles_of(p, pos), p.rotary, p.eps, l, up);
        }
        if (2 * j + hw < len) {
          uint8_t* dst = page + (at + 2 * j + hw) * D;
          *reinterpret_cast<uint32_t*>(dst + L.d0) = code.x;
          *reinterpret_cast<uint32_t*>(dst + L.d1) = code.y;
        }
      }
      __syncwarp();
    } else {
      __nv_bfloat162 top = __float2bfloat162_rn(0.f);        // (the maximum passes over NaN)
#pragma unroll 1
      for (int j0 = 0; 2 * j0 < len; j0 += 4) {
        uint4 raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          raw[j] = 2 * (j0 + j) + hw < len ? V.load(rows + (2 * (j0 + j) + hw) * p.ld) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          *reinterpret_cast<uint4*>(&keep[j0 + j][0][lane]) = raw[j];
          const uint32_t x[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[i])));
        }
      }
      m = fmaxf(__low2float(top), __high2float(top));
      m = warp_max(m);
      const bool inf = m > FLOAT_MAX;                      // then the largest finite one
      if (inf) {
        m = 0.f;
        for (int j = 0; 2 * j < len; ++j) {
          float v[8];
          V.unpack(*reinterpret_cast<const uint4*>(&keep[j][0][lane]), v);
          m = finite_amax(v, m);
        }
        m = warp_max(m);
      }
      s = fmaxf(scale_of(m), old);
      const float up = 1.f / s;
#pragma unroll 2
      for (int j = 0; 2 * j < len; ++j) {
        float v[8];
        V.unpack(*reinterpret_cast<const uint4*>(&keep[j][0][lane]), v);
        if (inf) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = finite(v[i]) ? v[i] : __int_as_float(0x7fffffff);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= up;
        if (2 * j + hw < len) *reinterpret_cast<uint2*>(page + (at + 2 * j + hw) * D + 8 * l) = V.codes(v);
      }
      __syncwarp();
    }
    if (old < s && at > 0) {
      const float r = old / s;
      for (int j = 0; j < at; ++j) {
        uint32_t* c = reinterpret_cast<uint32_t*>(page + j * D + 4 * lane);
        const float2 a = h2_to_f2(e4m3x2_to_h2(*c)), b = h2_to_f2(e4m3x2_to_h2_hi(*c));
        *c = e4m3x2(a.x * r, a.y * r) | (e4m3x2(b.x * r, b.y * r) << 16);
      }
    }
    __syncwarp();
    if (lane == 0) *sp = s;
  }
}

template <int TG, bool INTER>
__global__ void __launch_bounds__(AW * 32, 5) kv8_append_kernel(const AppendParams p) {
  __shared__ float4 keep[AW][HALF][2][32];
  const int per = (2 * p.nkv + AW - 1) / AW;               // key / value CTAs of a token group
  const int kv_ctas = (p.T + TG - 1) / TG * per;
  const int i = blockIdx.x;
  if (i < kv_ctas) {
    const int u = i % per * AW + (threadIdx.x >> 5);
    if (u < 2 * p.nkv) append_keys_values<TG, INTER>(p, i / per * TG, u, keep[threadIdx.x >> 5]);
  } else {
    const int q = (p.nq + QH - 1) / QH;
    append_queries<INTER>(p, (i - kv_ctas) / q, (i - kv_ctas) % q * QH);
  }
}

// Check mode: one warp per (sampled token, head) recomputes the row (keys in double: the same bits) and compares it
// with what the append stored: the query's bits, or the codes at the page's scale, which must cover the row. Valid
// until a later append moves the page.
template <bool INTER>
__global__ void __launch_bounds__(256) kv8_append_check_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 31, l = lane & 15, h = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int heads = p.nq + 2 * p.nkv;
  if (h >= heads) return;
  const int t = p.rows[blockIdx.x];
  if (blockIdx.x == 0 && h == 0 && lane == 0) atomicAdd(p.check + 2, 1ull);
  if (t < 0 || t >= p.T) return;
  const long long slot = slot_of(p, t);
  const bool is_q = h < p.nq, is_k = !is_q && h < p.nq + p.nkv;
  if (!is_q && slot < 0) return;
  const RowLane<INTER> L(l, p.rotary);
  const __nv_bfloat16* row = p.qkv + t * p.ld + static_cast<long long>(h) * D;
  const __nv_bfloat16* nw = is_q ? p.qw : is_k ? p.kw : nullptr;
  float w[8];
  if (nw != nullptr) L.unpack(L.load(nw), w);
  const int pos = p.rotary > 0 && slot != -2 ? p.pos[t] : 0;
  int bad = D;                                             // the lane's first differing dim (both halves hold the row)
  if (is_q) {
    float v[8];
    L.unpack(L.load(row), v);
    float c[8];
    L.angles(angles_of(p, pos), c);
    if (nw != nullptr) {
      const float inv = norm_of(v, p.epsf);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
    }
    rotate(v, c);
    uint4 o = L.pack(v);
    if (slot == -2) o.x = o.y = o.z = o.w = 0x7fff7fffu;
    const uint4 have = L.load(p.q_out + (static_cast<long long>(t) * p.nq + h) * D);
    const int e3 = bf16x2_diff(o.w, have.w), e2 = bf16x2_diff(o.z, have.z), e1 = bf16x2_diff(o.y, have.y),
              e0 = bf16x2_diff(o.x, have.x);
    bad = e0 >= 0 ? L.d0 + e0 : e1 >= 0 ? L.d0 + 2 + e1 : e2 >= 0 ? L.d1 + e2 : e3 >= 0 ? L.d1 + 2 + e3 : D;
  } else {
    const int kvh = is_k ? h - p.nq : h - p.nq - p.nkv;
    const long long blk = slot / PAGE;
    const float s = p.scales[(blk * p.nkv + kvh) * 2 + (is_k ? 0 : 1)];
    float m;
    uint2 want;
    if (is_k) {
      m = exact_amax<INTER>(row, nw, angles_of(p, pos), p.rotary, p.eps, l);
      want = exact_codes<INTER>(row, nw, angles_of(p, pos), p.rotary, p.eps, l, 1.f / s);
    } else {
      float v[8];
      L.unpack(L.load(row), v);
      m = finite_amax(v, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = finite(v[i]) ? v[i] * (1.f / s) : __int_as_float(0x7fffffff);
      want = L.codes(v);
    }
    const bool covers = s >= scale_of(warp_max(m));
    const uint8_t* have = p.codes + ((blk * 2 + (is_k ? 0 : 1)) * p.nkv + kvh) * (PAGE * D) + (slot % PAGE) * D;
    const uint32_t ws[2] = {want.x, want.y};
    const uint32_t hs[2] = {*reinterpret_cast<const uint32_t*>(have + L.d0), *reinterpret_cast<const uint32_t*>(have + L.d1)};
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const uint32_t a = (ws[i >> 2] >> (8 * (i & 3))) & 0xffu, b = (hs[i >> 2] >> (8 * (i & 3))) & 0xffu;
      const bool same = a == b || ((a | b) & 0x7fu) == 0 || ((a & 0x7fu) == 0x7fu && (b & 0x7fu) == 0x7fu);
      if (!same || !covers) bad = (i < 4 ? L.d0 : L.d1) + (i & 3);
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) bad = min(bad, __shfl_xor_sync(0xffffffffu, bad, k));
  if (bad < D && lane == 0)
    report_replay_mismatch(p.check, (static_cast<unsigned long long>(t) * heads + h) * D + bad);
}

// ------------------------------------------------------------------------------------------------ pages to bf16
// Pages of the list in bf16 (exact while scales are powers of two), for the tensor-core prefill: a prefill reads each
// page once for every 256 / group of its query rows, so expanding it once costs less than expanding it in every CTA.
// One warp per (page, K / V, kv head): 2 KB in, 4 KB out; 1024 pages of 8 heads 15 us, 6.7 TB/s. A page id outside the
// cache gives NaN. With `check`: every `step`-th page of the list from `from` on is compared instead of written.
struct ExpandParams {
  const uint8_t* codes;
  const float* scales;
  const int* pages;
  int npages, nkv;
  long long num_blocks;
  __nv_bfloat16* out;
  int from, step;
  unsigned long long* check;
};

__global__ void __launch_bounds__(256) kv8_expand_kernel(const ExpandParams p) {
  const long long gt = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  pdl_trigger();                           // the prefill may start, and waits before it reads a page
  const long long gw = gt >> 5;
  const int lane = threadIdx.x & 31, per = 2 * p.nkv;
  const long long i = p.check == nullptr ? gw / per : p.from + gw / per * static_cast<long long>(p.step);
  if (i >= p.npages) return;
  const int unit = static_cast<int>(gw % per), kv = unit / p.nkv, h = unit % p.nkv;
  const int blk = p.pages[i];
  const bool in = blk >= 0 && blk < p.num_blocks;
  const float s = in ? p.scales[(static_cast<long long>(blk) * p.nkv + h) * 2 + kv] : __int_as_float(0x7fffffff);
  const uint2* src = reinterpret_cast<const uint2*>(
      p.codes + ((static_cast<long long>(in ? blk : 0) * 2 + kv) * p.nkv + h) * (PAGE * D));
  uint4* dst = reinterpret_cast<uint4*>(p.out + ((i * 2 + kv) * p.nkv + h) * (PAGE * D));
  // eight codes to a lane and 16 bytes out, so that a store writes whole lines
  uint2 c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = src[j * 32 + lane];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 f0 = h2_to_f2(e4m3x2_to_h2(c[j].x)), f1 = h2_to_f2(e4m3x2_to_h2_hi(c[j].x));
    const float2 f2 = h2_to_f2(e4m3x2_to_h2(c[j].y)), f3 = h2_to_f2(e4m3x2_to_h2_hi(c[j].y));
    const uint4 o = make_uint4(pack_bf16x2(f0.x * s, f0.y * s), pack_bf16x2(f1.x * s, f1.y * s),
                               pack_bf16x2(f2.x * s, f2.y * s), pack_bf16x2(f3.x * s, f3.y * s));
    if (p.check == nullptr) {
      dst[j * 32 + lane] = o;
    } else {
      const uint4 d = dst[j * 32 + lane];
      bad |= bf16x2_diff(o.x, d.x) >= 0 || bf16x2_diff(o.y, d.y) >= 0 || bf16x2_diff(o.z, d.z) >= 0 ||
             bf16x2_diff(o.w, d.w) >= 0;
    }
  }
  if (p.check != nullptr) {
    const unsigned who = __ballot_sync(0xffffffffu, bad);
    if (who && lane == 0) report_replay_mismatch(p.check, static_cast<unsigned long long>(i) * per + unit);
  }
}

// ------------------------------------------------------------------------------------------------ decode
// One new token per sequence, o = sum_j w_j v_j / sum_j w_j with w_j = exp(scale q . k_j). Bound by the cache bytes
// (256 a key and kv head); the queries of a kv head (<= 16) share every key that is read.
//
// Tensor cores on converted codes (mma.m16n8k16, f16 inputs, fp32 sums): E4M3 is exact in f16, so scales stay outside
// the products. Both products have the cache as their A operand, whose fragments a lane fills from 16-byte reads of the
// page in shared memory: S^T (16 keys x heads) = K Q^T, with the order of the dims permuted alike in K and Q so that a
// lane's four codes of a k step are neighbours; O^T (dims x heads) += V^T P^T, with the pairs of keys put together by
// byte permutes. Pages come by TMA into a ring of each warp (three pages deep), which no other warp waits for.
//   q: bf16 values times a power of two per head (largest in [2^14, 2^15)), exact in f16 down to 2^-38 of the largest.
//   x = log2(e) scale s_K q . k, and with V's page scale in the exponent y = x + log2 s_V. The running maximum M is of
//   y, so the weights w = 2^(x - M + 14) s_V <= 2^15 are the largest f16 can hold whatever the pages' scales; the row
//   sum takes 2^(x - M + 30) in fp32: x - M reaches from 60 (a page of the least scale) to -128 and below, so the bias
//   keeps both ends inside fp32. Rounding w to f16 costs 2^-11 of it, less than the output's rounding to bf16 (2^-8).
//   Masked keys: x = -inf and V's codes cleared (0 * NaN); rows without keys give 0, rows with scores of NaN, or of -inf
//   alone, NaN.
//
// A CTA (4 warps) takes one segment of seg_pages pages of one (sequence, kv head), warp w its pages w, w + 4, ...; a
// sequence of one segment is written at once, else a partial record per segment and head goes to `part` and
// kv8_combine_kernel merges them in order. Segments start at absolute multiples, so a row's arithmetic does not depend
// on the batch around it: running a subset of rows again with the same plan gives the same bits (check mode).
// A sequence whose length or table row does not fit gives NaN, as does a page id outside the cache.
//
// Measured (16 query, 8 kv heads, device time): 256 x 1600 keys 135 us, 6.2 TB/s, 0.95 of a copy's rate: DRAM bounds it.
// 1 x 131072 keys 53 us, 5.1 TB/s, with the merge of its segments and the start of the CTAs in it; 61 ragged ones up to
// 4100 keys 59 us, 4.5 TB/s, the longest rows' tail. 1 x 37 keys 3.8 us, latency. More than 8 query heads a kv head pay a
// second set of products for the same bytes, at 3 CTAs an SM: 64 x 2048 keys, 2 kv heads, of 8, 9 and 16 queries each: 29.6,
// 34.1 and 42.1 us (bytes: 10.4); 256 x 1600, 4 kv heads, of 8 and 16: 74 and 94 us (65). Loads into registers instead of the
// ring: 162 us for the first; a ring filled by cp.async: 159; two warps a CTA: 131, but 67 and 76 us for the next two.
constexpr int WARPS = 4;
constexpr int REC = D + 4;               // floats a record: o[D], M, l, pad

struct DecodeParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  const uint8_t* codes;
  const float2* scales;      // [num_blocks][nkv] (K, V)
  long long num_blocks;
  const int* table;          // [table_rows][max_pages], rows `table_ld` apart
  int table_rows, max_pages;
  long long table_ld;
  const int* seq_req;
  const int* ctx;
  const int* seq_idx;
  int nseqs;                 // sequences of q (bound of seq_idx)
  int nq, nkv, G;
  int seg_pages, max_segs;
  float scale_log2;
  float* part;               // [nseqs][nkv][max_segs][G][REC]
  float* row_sq;
  unsigned long long* check;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's pages wait in shared memory, K then V of one head, 16 rows of 128 bytes each as TMA lays them out: 16-byte
// piece j of row r at piece j ^ (r & 7). Matrix row i stands for key key_of(i) (and 8 + i for 8 + key_of(i)); this order
// makes both reads below free of bank conflicts: eight lanes meet eight different pieces.
constexpr int STAGES = 3;                // pages of a warp in shared memory: one in use, the others on their way
constexpr int PAGE_BYTES = PAGE * D;
__device__ __forceinline__ int key_of(int i) { return i ^ ((i & 1) << 2); }
__device__ __forceinline__ uint4 piece(const uint8_t* rows, int key, int j) {
  return *reinterpret_cast<const uint4*>(rows + key * D + ((j ^ (key & 7)) << 4));
}
__device__ __forceinline__ uint32_t word(const uint4& u, int j) { return j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w; }

// The value at output element i of row (sequence b), or its comparison with what is there.
__device__ __forceinline__ float put(const DecodeParams& p, int b, int head, int d, float v) {
  const long long at = (static_cast<long long>(b) * p.nq + head) * D + d;
  const __nv_bfloat16 r = __float2bfloat16(v);
  const float x = __bfloat162float(r);
  if (p.check == nullptr) {
    p.o[at] = r;
  } else {
    const float y = __bfloat162float(p.o[at]);
    if (!(x == y) && !(x != x && y != y)) report_replay_mismatch(p.check, static_cast<unsigned long long>(at));
  }
  return x * x;
}

__device__ __forceinline__ int pages_of(int n) { return n / PAGE + (n % PAGE > 0 ? 1 : 0); }
__device__ __forceinline__ bool row_fits(const DecodeParams& p, int n, int req) {
  return n >= 0 && pages_of(n) <= p.max_pages && pages_of(n) <= p.max_segs * p.seg_pages && req >= 0 &&
         req < p.table_rows;
}

// The dim of float i of a row of sums: dim 16g + 2i + e lies at 2 (8i + g) + e, so that the lanes of a store meet
// different banks.
__device__ __forceinline__ int dim_of(int i) { return 16 * ((i >> 1) & 7) + 2 * (i >> 4) + (i & 1); }

template <int NT>
struct DecodeSmem {
  union {
    uint8_t ring[WARPS][STAGES][2 * PAGE_BYTES];
    float o[WARPS][NT * 8][D + 4];       // the warps' sums (see dim_of), once the pages are done with
  };
  float m[WARPS][NT * 8], l[WARPS][NT * 8];
  uint64_t full[WARPS][STAGES];
};

// NT: groups of eight heads (1: up to 8 queries a kv head, 2: up to 16).
template <int NT>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 4 : 3) kv8_decode_kernel(const __grid_constant__ CUtensorMap tm,
                                                                     const DecodeParams p) {
  pdl_trigger();
  extern __shared__ unsigned char decode_smem[];
  // the pages' swizzle counts from 1 KB boundaries
  DecodeSmem<NT>& sm = *reinterpret_cast<DecodeSmem<NT>*>(decode_smem + ((1024 - (smem_u32(decode_smem) & 1023)) & 1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int b = p.seq_idx ? p.seq_idx[blockIdx.x] : blockIdx.x;
  const int kvh = blockIdx.y;
  if (p.check != nullptr && blockIdx.x == 0 && kvh == 0 && blockIdx.z == 0 && tid == 0) atomicAdd(p.check + 2, 1ull);
  if (b < 0 || b >= p.nseqs) return;
  const int n = p.ctx[b], req = p.seq_req[b];
  const int pages = pages_of(n);
  const bool fits = row_fits(p, n, req);
  if (!fits || n == 0) {
    if (blockIdx.z != 0) return;
    const float v = fits ? 0.f : __int_as_float(0x7fffffff);
    for (int h = 0; h < p.G; ++h)
      for (int i = tid; i < D; i += WARPS * 32) put(p, b, kvh * p.G + h, i, v);
    if (!fits && p.check == nullptr && p.row_sq != nullptr && tid == 0) atomicAdd(p.row_sq + b, v);
    return;
  }
  const int nseg = (pages + p.seg_pages - 1) / p.seg_pages;
  if (static_cast<int>(blockIdx.z) >= nseg) return;
  if (lane == 0) {
    tma_prefetch_desc(&tm);
#pragma unroll
    for (int i = 0; i < STAGES; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  int fetched = 0, used = 0;             // this warp's pages so far: page i waits in stage i % STAGES
  bool ok = true;
  // A segment's pages of this warp. Lane i holds the place (in units of a head's page) and the scales of page 32 c + i:
  // of the 32 pages around page k, and of the next 32.
  const int* row = p.table + req * p.table_ld;
  int first = 0, count = 0, unit0, unit1;
  float2 sc0, sc1;
  const auto look_up = [&](int k, int& unit, float2& sc) {
    const int id = k < count ? row[first + WARPS * k] : 0;
    const bool in = id >= 0 && id < p.num_blocks;
    unit = (in ? id : 0) * 2 * p.nkv + kvh;
    sc = k < count ? p.scales[static_cast<long long>(in ? id : 0) * p.nkv + kvh] : make_float2(0.f, 0.f);
    if (!in) sc.x = sc.y = __int_as_float(0x7fffffff);
  };
  const auto fetch = [&](int k, int base) {                // page k, base <= k < base + 64
    const int u0 = __shfl_sync(0xffffffffu, unit0, k & 31), u1 = __shfl_sync(0xffffffffu, unit1, k & 31);
    if (k >= count) return;
    if (lane == 0) {
      const int stage = fetched % STAGES, unit = k - base < 32 ? u0 : u1;
      uint64_t* bar = &sm.full[warp][stage];
      mbar_arrive_expect_tx(bar, 2 * PAGE_BYTES);
      tma_load_2d(sm.ring[warp][stage], &tm, bar, 0, unit * PAGE);
      tma_load_2d(sm.ring[warp][stage] + PAGE_BYTES, &tm, bar, 0, (unit + p.nkv) * PAGE);
    }
    ++fetched;
  };
  const auto begin = [&](int seg) {
    first = seg * p.seg_pages + warp;
    const int end = min(pages, (seg + 1) * p.seg_pages);
    count = first < end ? (end - first + WARPS - 1) / WARPS : 0;
    look_up(lane, unit0, sc0);
    look_up(32 + lane, unit1, sc1);
#pragma unroll 1
    for (int k = 0; k < STAGES - 1; ++k) fetch(k, 0);
  };
  begin(blockIdx.z);                     // the first pages are on their way before the queries are read
  // Q^T fragments: b0 = dims 64c + 16t + 4j + {0, 1}, b1 = + {2, 3} of head g, k step 4c + j
  uint32_t qb[NT][8][2];
  float f[NT][2];                    // heads 2t, 2t + 1: scale log2(e) / (the head's power of two)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + g;
    uint32_t w[16];
    float m = 0.f;
    const __nv_bfloat16* row = p.q + (static_cast<long long>(b) * p.nq + kvh * p.G + (h < p.G ? h : 0)) * D;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 u = h < p.G ? *reinterpret_cast<const uint4*>(row + 64 * c + 16 * t + 8 * e) : make_uint4(0, 0, 0, 0);
        w[c * 8 + e * 4] = u.x;
        w[c * 8 + e * 4 + 1] = u.y;
        w[c * 8 + e * 4 + 2] = u.z;
        w[c * 8 + e * 4 + 3] = u.w;
      }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      m = fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y)));
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
    e = e < -100 ? -100 : e > 127 ? 14 : e;            // not finite: as it is
    const float up = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
    const float down = __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      qb[nt][i >> 1][i & 1] = pack_h2(x.x * up, x.y * up);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) f[nt][c] = p.scale_log2 * __shfl_sync(0xffffffffu, down, (2 * t + c) * 4);
  }
  for (int seg = blockIdx.z; seg < nseg; seg += gridDim.z) {
    if (seg != static_cast<int>(blockIdx.z)) begin(seg);
    float M[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      M[nt][0] = M[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
    }
    for (int k = 0; k < count; ++k) {
      if (k > 0 && (k & 31) == 0) {
        unit0 = unit1;
        sc0 = sc1;
        look_up(k + 32 + lane, unit1, sc1);
      }
      __syncwarp();                      // the stage of page k + STAGES - 1 was read in the turn before
      fetch(k + STAGES - 1, k & ~31);
      ok = mbar_wait(&sm.full[warp][used % STAGES], (used / STAGES) & 1, nullptr);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const uint8_t* kpage = sm.ring[warp][used % STAGES];
      const uint8_t* vpage = kpage + PAGE_BYTES;
      ++used;
      const float ks = __shfl_sync(0xffffffffu, sc0.x, k & 31), vs = __shfl_sync(0xffffffffu, sc0.y, k & 31);
      const int key0 = (first + WARPS * k) * PAGE;
      {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint4 k0 = piece(kpage, key_of(g), 4 * c + t), k8 = piece(kpage, 8 + key_of(g), 4 * c + t);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w0 = word(k0, j), w1 = word(k8, j);
            const uint32_t a0 = e4m3x2_to_h2(w0), a2 = e4m3x2_to_h2_hi(w0);
            const uint32_t a1 = e4m3x2_to_h2(w1), a3 = e4m3x2_to_h2_hi(w1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a0, a1, a2, a3, qb[nt][4 * c + j][0], qb[nt][4 * c + j][1]);
          }
        }
        const float ev = static_cast<float>(max(static_cast<int>((__float_as_uint(vs) >> 23) & 255u) - 127, -60));
        const float vw = vs * W_SCALE;       // s_V 2^(14 - SUM_BIAS)
        const bool in0 = key0 + key_of(g) < n, in1 = key0 + key_of(g) + 8 < n;
        uint32_t pb[NT][2];
        bool moved = false;
        float a[NT][2], Mn[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float fk = f[nt][c] * ks;
            s[nt][c] = in0 ? s[nt][c] * fk : -INFINITY;
            s[nt][2 + c] = in1 ? s[nt][2 + c] * fk : -INFINITY;
            float mx = fmaxf(s[nt][c], s[nt][2 + c]) + ev;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            Mn[nt][c] = fmaxf(M[nt][c], mx);
            moved |= Mn[nt][c] != M[nt][c];
          }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              a[nt][c] = Mn[nt][c] == M[nt][c] ? 1.f : ex2(M[nt][c] - Mn[nt][c]);
              M[nt][c] = Mn[nt][c];
              l[nt][c] *= a[nt][c];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[nt][i][0] *= a[nt][0];
              o[nt][i][1] *= a[nt][1];
              o[nt][i][2] *= a[nt][0];
              o[nt][i][3] *= a[nt][1];
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float ref = M[nt][c] == -INFINITY ? 0.f : M[nt][c] - SUM_BIAS;
            const float p0 = ex2(s[nt][c] - ref), p1 = ex2(s[nt][2 + c] - ref);
            l[nt][c] += p0 + p1;
            w[c] = p0 * vw;
            w[2 + c] = p1 * vw;
          }
          pb[nt][0] = transpose8(pack_h2(w[0], w[1]));
          pb[nt][1] = transpose8(pack_h2(w[2], w[3]));
        }
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = piece(vpage, key_of(2 * t + (i & 1)) + (i >> 1) * 8, g);
        if (key0 + PAGE > n) {         // the sequence's last page: nothing behind its end may reach a product
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + key_of(2 * t + (i & 1)) + (i >> 1) * 8 >= n) v[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w0 = word(v[0], j), w1 = word(v[1], j), w2 = word(v[2], j), w3 = word(v[3], j);
          const uint32_t x01 = __byte_perm(w0, w1, 0x5140), y01 = __byte_perm(w0, w1, 0x7362);
          const uint32_t x23 = __byte_perm(w2, w3, 0x5140), y23 = __byte_perm(w2, w3, 0x7362);
          const uint32_t a0 = e4m3x2_to_h2(x01), a1 = e4m3x2_to_h2_hi(x01);
          const uint32_t a2 = e4m3x2_to_h2(x23), a3 = e4m3x2_to_h2_hi(x23);
          const uint32_t c0 = e4m3x2_to_h2(y01), c1 = e4m3x2_to_h2_hi(y01);
          const uint32_t c2 = e4m3x2_to_h2(y23), c3 = e4m3x2_to_h2_hi(y23);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(o[nt][2 * j], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            mma_f16(o[nt][2 * j + 1], c0, c1, c2, c3, pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    if (!ok) {                           // a wait ran out: the row becomes NaN, and what is on its way must land
      for (; used < fetched; ++used) mbar_wait(&sm.full[warp][used % STAGES], (used / STAGES) & 1, nullptr);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __int_as_float(0x7fffffff);
    }
    __syncthreads();                     // every warp is done with its pages
    // merge of the warps: o[nt][i] holds dims 16g + 2i + {0, 1} of heads 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = nt * 8 + 2 * t + c;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float2*>(&sm.o[warp][h][2 * (8 * i + g)]) = make_float2(o[nt][i][c], o[nt][i][2 + c]);
        float s = l[nt][c];
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        s += __shfl_xor_sync(0xffffffffu, s, 8);
        s += __shfl_xor_sync(0xffffffffu, s, 16);
        if (g == 0) {
          sm.m[warp][h] = M[nt][c];
          sm.l[warp][h] = s;
        }
      }
    }
    __syncthreads();
    float sq = 0.f;
    for (int h = 0; h < p.G; ++h) {
      float m = sm.m[0][h];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) m = fmaxf(m, sm.m[w][h]);
      const float ref = m == -INFINITY ? 0.f : m;
      float acc[D / (WARPS * 32)] = {}, ls = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float e = ex2(sm.m[w][h] - ref);
#pragma unroll
        for (int i = 0; i < D / (WARPS * 32); ++i) acc[i] = fmaf(sm.o[w][h][tid + i * WARPS * 32], e, acc[i]);
        ls = fmaf(sm.l[w][h], e, ls);
      }
      if (nseg == 1) {
        const float inv = 1.f / W_SCALE / ls;          // no weight (scores of -inf alone): 0 / 0
#pragma unroll
        for (int i = 0; i < D / (WARPS * 32); ++i)
          sq += put(p, b, kvh * p.G + h, dim_of(tid + i * WARPS * 32), acc[i] * inv);
      } else {
        float* rec = p.part + (((static_cast<long long>(b) * p.nkv + kvh) * p.max_segs + seg) * p.G + h) * REC;
#pragma unroll
        for (int i = 0; i < D / (WARPS * 32); ++i) rec[tid + i * WARPS * 32] = acc[i];
        if (tid == 0) {
          rec[D] = m;
          rec[D + 1] = ls;
        }
      }
    }
    if (nseg == 1 && p.check == nullptr && p.row_sq != nullptr) {
      sq = warp_sum(sq);
      if (lane == 0) atomicAdd(p.row_sq + b, sq);
    }
    fence_proxy_async_smem();            // the sums lay where the next segment's pages go
    __syncthreads();
  }
}

// Merges the segments of each (sequence, head), in segment order within four interleaved parts: thread (part, dim).
constexpr int PARTS = 4;
constexpr int MAX_SEGS = 256;
__global__ void __launch_bounds__(PARTS * D) kv8_combine_kernel(const DecodeParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float wsm[MAX_SEGS], red[PARTS * D / 32], osm[PARTS][D], lsum;
  const int tid = threadIdx.x, part = tid / D, d = tid % D;
  const int b = p.seq_idx ? p.seq_idx[blockIdx.x] : blockIdx.x;
  if (b < 0 || b >= p.nseqs) return;
  const int head = blockIdx.y, kvh = head / p.G, h = head % p.G;
  const int n = p.ctx[b];
  const int nseg = (pages_of(n) + p.seg_pages - 1) / p.seg_pages;
  if (!row_fits(p, n, p.seq_req[b]) || nseg <= 1) return;
  const long long step = static_cast<long long>(p.G) * REC;
  const float* base = p.part + (((static_cast<long long>(b) * p.nkv + kvh) * p.max_segs) * p.G + h) * REC;
  const float m = tid < nseg ? base[tid * step + D] : -INFINITY;
  const float wm = warp_max(m);
  if ((tid & 31) == 0) red[tid >> 5] = wm;
  __syncthreads();
  float M = red[0];
#pragma unroll
  for (int i = 1; i < PARTS * D / 32; ++i) M = fmaxf(M, red[i]);
  const float ref = M == -INFINITY ? 0.f : M;
  float lp = 0.f;
  if (tid < nseg) {
    const float e = ex2(m - ref);
    wsm[tid] = e;
    lp = base[tid * step + D + 1] * e;
  }
  __syncthreads();
  lp = warp_sum(lp);
  if ((tid & 31) == 0) red[tid >> 5] = lp;
  float acc = 0.f;
#pragma unroll 8
  for (int s = part; s < nseg; s += PARTS) acc = fmaf(base[s * step + d], wsm[s], acc);
  osm[part][d] = acc;
  __syncthreads();
  if (tid == 0) {
    float s = 0.f;
    for (int i = 0; i < PARTS * D / 32; ++i) s += red[i];
    lsum = s;
  }
  __syncthreads();
  if (part != 0) return;
  const float o = (osm[0][d] + osm[1][d]) + (osm[2][d] + osm[3][d]);
  float sq = put(p, b, head, dim_of(d), o / lsum * (1.f / W_SCALE));
  if (p.check == nullptr && p.row_sq != nullptr) {
    sq = warp_sum(sq);
    if ((tid & 31) == 0) atomicAdd(p.row_sq + b, sq);
  }
}

// The tokens of prefill tiles (request, first token or place in row_idx, tokens, -1 or that place) as sequences of the
// decode kernel: request and keys (position + 1) of token t, and the list of the tokens to run: a prefill's token t at
// place t, a replay's behind them as row_idx lists it; -1 elsewhere. A position outside the table has no keys. One CTA: a
// few hundred tokens, 2 us.
struct TokensParams {
  const int4* tiles;
  int ntiles, tile_tokens;
  const int* row_idx;
  int nrows;
  const int* pos;
  int limit;                 // keys that a row of the table has room for
  int T;
  int* req;                  // [T]
  int* ctx;                  // [T]
  int* idx;                  // [T + nrows]
};
__global__ void __launch_bounds__(1024) kv8_tokens_kernel(const TokensParams p) {
  for (int i = threadIdx.x; i < p.T + p.nrows; i += 1024) p.idx[i] = -1;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < p.ntiles; i += 32) {
    const int4 tl = p.tiles[i];
    for (int j = lane; j < min(tl.z, p.tile_tokens); j += 32) {
      if (tl.w >= 0 && tl.w + j >= p.nrows) break;
      const int t = tl.w >= 0 ? p.row_idx[tl.w + j] : tl.y + j;
      if (t < 0 || t >= p.T) continue;
      const int ps = p.pos[t];
      p.req[t] = tl.x;
      p.ctx[t] = ps >= 0 && ps < p.limit ? ps + 1 : 0;
      p.idx[tl.w >= 0 ? p.T + tl.w + j : t] = t;
    }
  }
}

template <int NT>
static int launch_decode(const CUtensorMap& tm, const DecodeParams& p, int nrun, int z, cudaStream_t st) {
  // the attribute belongs to a device; one bit for each that has it (setting it twice does no harm)
  static std::atomic<unsigned long long> ready{0};
  constexpr int smem = static_cast<int>(sizeof(DecodeSmem<NT>)) + 1024;   // + room to align the pages
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(kv8_decode_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev <= 63) ready.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return static_cast<int>(e);
  kv8_decode_kernel<NT><<<dim3(nrun, p.nkv, z), WARPS * 32, smem, st>>>(tm, p);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.max_segs == 1) return static_cast<int>(e);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(nrun, p.nq);
  cfg.blockDim = dim3(PARTS * D);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kv8_combine_kernel, p));
}

}  // namespace kv8
}  // namespace sdc

using namespace sdc::kv8;

// Each entry takes its arguments in one struct, natural alignment: through ctypes a call costs microseconds less than
// with twenty arguments, which is what the smallest calls are made of.
extern "C" {

struct Kv8AppendArgs {
  const void* qkv;
  long long ld;
  int T;
  int nq;
  int nkv;
  const int* pos;
  const long long* slots;
  const void* qw;
  const void* kw;
  double eps;
  const void* cos_sin;
  int table_rows;
  int rotary;
  int interleaved;
  void* q_out;
  void* codes;
  void* scales;
  long long num_blocks;
  const int* rows;
  int nrows;
  void* check;
  void* stream;
};
int sdc_kv8_append(const Kv8AppendArgs* args) {
  const auto& [qkv, ld, T, nq, nkv, pos, slots, qw, kw, eps, cos_sin, table_rows, rotary, interleaved, q_out,
               codes, scales, num_blocks, rows, nrows, check, stream] = *args;
  if (T <= 0 || (check != nullptr && nrows <= 0)) return 0;
  if (ld % 4 || rotary < 0 || rotary > D || rotary % 8 || nq < 0 || nkv < 1 || (check != nullptr) != (rows != nullptr))
    return -1;
  AppendParams p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.ld = ld;
  p.T = T;
  p.nq = nq;
  p.nkv = nkv;
  p.pos = pos;
  p.slots = slots;
  p.qw = static_cast<const __nv_bfloat16*>(qw);
  p.kw = static_cast<const __nv_bfloat16*>(kw);
  p.eps = eps;
  p.epsf = static_cast<float>(eps);
  p.cs = static_cast<const float2*>(cos_sin);
  p.table_rows = table_rows;
  p.rotary = rotary;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<float*>(scales);
  p.capacity = num_blocks * PAGE;
  p.rows = rows;
  p.check = static_cast<unsigned long long*>(check);
  const int gy = (nq + 2 * nkv + 7) / 8;
  auto st = static_cast<cudaStream_t>(stream);
  // one token, four or a page to a warp of keys or values: a decode step's tokens lie in as many pages, a prompt's share
  // them, and only their number is known here. Of 1, 4, 16: 256 x 1 token 6.9, 10.4, 32.9 us; 512 x 1 10.7, 12.2, 33.3;
  // 1 x 512 10.1, 8.7, 8.6; 1024 x 1 18.5, 17.5, 37.2; 5 x 300 16.7, 12.2, 14.2; 1 x 2048 21.8, 13.9, 11.9 us
  const int tg = T < 512 ? 1 : T < 2048 ? 4 : PAGE;
  const long long ctas = static_cast<long long>((T + tg - 1) / tg) * ((2 * nkv + AW - 1) / AW) +
                         static_cast<long long>((T + 2 * AW - 1) / (2 * AW)) * ((nq + QH - 1) / QH);
  const unsigned grid = static_cast<unsigned>(ctas);
  const dim3 sample(nrows, gy);
  if (p.check != nullptr) {
    if (interleaved) kv8_append_check_kernel<true><<<sample, 256, 0, st>>>(p);
    else kv8_append_check_kernel<false><<<sample, 256, 0, st>>>(p);
  } else if (tg == 1) {
    if (interleaved) kv8_append_kernel<1, true><<<grid, AW * 32, 0, st>>>(p);
    else kv8_append_kernel<1, false><<<grid, AW * 32, 0, st>>>(p);
  } else if (tg == 4) {
    if (interleaved) kv8_append_kernel<4, true><<<grid, AW * 32, 0, st>>>(p);
    else kv8_append_kernel<4, false><<<grid, AW * 32, 0, st>>>(p);
  } else {
    if (interleaved) kv8_append_kernel<PAGE, true><<<grid, AW * 32, 0, st>>>(p);
    else kv8_append_kernel<PAGE, false><<<grid, AW * 32, 0, st>>>(p);
  }
  return static_cast<int>(cudaGetLastError());
}

struct Kv8ExpandArgs {
  const void* codes;
  const void* scales;
  long long num_blocks;
  const int* pages;
  int npages;
  int nkv;
  void* out;
  int from;
  int step;
  void* check;
  void* stream;
};
int sdc_kv8_expand(const Kv8ExpandArgs* args) {
  const auto& [codes, scales, num_blocks, pages, npages, nkv, out, from, step, check, stream] = *args;
  if (npages <= 0) return 0;
  if (nkv < 1 || num_blocks < 1 || (check != nullptr && (from < 0 || step < 1))) return -1;
  ExpandParams p;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = static_cast<const float*>(scales);
  p.pages = pages;
  p.npages = npages;
  p.nkv = nkv;
  p.num_blocks = num_blocks;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.from = from;
  p.step = step;
  p.check = static_cast<unsigned long long*>(check);
  const long long n = check == nullptr ? npages : (npages - static_cast<long long>(from) + step - 1) / step;
  if (n <= 0) return 0;
  const long long blocks = (n * 2 * nkv * 32 + 255) / 256;
  kv8_expand_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return static_cast<int>(cudaGetLastError());
}

struct Kv8TokensArgs {
  const void* tiles;
  int ntiles;
  int tile_tokens;
  const int* row_idx;
  int nrows;
  const int* pos;
  int limit;
  int T;
  void* req;
  void* ctx;
  void* idx;
  void* stream;
};
static int list_tokens(const Kv8TokensArgs& args) {
  const auto& [tiles, ntiles, tile_tokens, row_idx, nrows, pos, limit, T, req, ctx, idx, stream] = args;
  if (T <= 0) return 0;
  if (ntiles < 0 || nrows < 0 || (nrows > 0 && row_idx == nullptr)) return -1;
  const TokensParams p{static_cast<const int4*>(tiles), ntiles, tile_tokens, row_idx, nrows, pos, limit, T,
                       static_cast<int*>(req), static_cast<int*>(ctx), static_cast<int*>(idx)};
  kv8_tokens_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return static_cast<int>(cudaGetLastError());
}

// part: nseqs * nkv * max_segs * (nq / nkv) * 132 floats (not read where max_segs is 1); rows of `nrun` sequences are
// computed: seq_idx's, or the first nrun.
struct Kv8DecodeArgs {
  const void* q;
  void* o;
  const void* codes;
  const void* scales;
  long long num_blocks;
  const int* table;
  int table_rows;
  int max_pages;
  long long table_ld;
  const int* seq_req;
  const int* ctx;
  const int* seq_idx;
  int nrun;
  int nseqs;
  int nq;
  int nkv;
  int seg_pages;
  int max_segs;
  float scale;
  void* part;
  void* row_sq;
  void* check;
  void* stream;
};
int sdc_kv8_decode(const Kv8DecodeArgs* args) {
  const auto& [q, o, codes, scales, num_blocks, table, table_rows, max_pages, table_ld, seq_req, ctx, seq_idx,
               nrun, nseqs, nq, nkv, seg_pages, max_segs, scale, part, row_sq, check, stream] = *args;
  if (nrun <= 0) return 0;
  if (nkv < 1 || nq % nkv || nq / nkv < 1 || nq / nkv > 16 || seg_pages < 1 || max_segs < 1 || max_segs > MAX_SEGS ||
      (max_segs > 1 && part == nullptr) || (check != nullptr && seq_idx == nullptr) ||
      (seq_idx == nullptr && nrun > nseqs) || num_blocks * 2 * nkv * PAGE > 0x7fffffffll)
    return -1;
  // the layer's codes as [num_blocks * 2 * nkv * 16][128] bytes; one box is one page of K or V of a head
  CUtensorMap tm;
  if (!make_map_u8_sw128(&tm, codes, num_blocks * 2 * nkv * PAGE, D, D, D, PAGE)) return -2;
  DecodeParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.o = static_cast<__nv_bfloat16*>(o);
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = static_cast<const float2*>(scales);
  p.num_blocks = num_blocks;
  p.table = table;
  p.table_rows = table_rows;
  p.max_pages = max_pages;
  p.table_ld = table_ld;
  p.seq_req = seq_req;
  p.ctx = ctx;
  p.seq_idx = seq_idx;
  p.nseqs = nseqs;
  p.nq = nq;
  p.nkv = nkv;
  p.G = nq / nkv;
  p.seg_pages = seg_pages;
  p.max_segs = max_segs;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(part);
  p.row_sq = static_cast<float*>(row_sq);
  p.check = static_cast<unsigned long long*>(check);
  // every segment its own CTA while that is at most 32768 CTAs (an empty one costs nanoseconds); else CTAs take several
  const long long rows = static_cast<long long>(nrun) * nkv;
  long long z = 32768 / rows;
  z = z < 1 ? 1 : z > max_segs ? max_segs : z;
  auto st = static_cast<cudaStream_t>(stream);
  return p.G <= 8 ? launch_decode<1>(tm, p, nrun, static_cast<int>(z), st)
                  : launch_decode<2>(tm, p, nrun, static_cast<int>(z), st);
}

// A prefill of few tokens: its tiles' tokens as sequences (lists that `decode` reads), then those.
struct Kv8FewArgs {
  Kv8TokensArgs tokens;
  Kv8DecodeArgs decode;
};
int sdc_kv8_prefill_few(const Kv8FewArgs* args) {
  const int rc = list_tokens(args->tokens);
  return rc != 0 ? rc : sdc_kv8_decode(&args->decode);
}

}  // extern "C"

// run-time wait limit of this unit (see common.cuh)
SDC_WAIT_LIMIT_SETTER(kv8)
