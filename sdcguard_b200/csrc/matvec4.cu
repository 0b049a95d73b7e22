// Products of a few rows with 4-bit weights and group scales (sm_100a): y = x W^T, x [M][K] bf16, M <= 32, with W read
// as its codes (a quarter of the bytes of the bf16 matrix).
//
//   W = rnd((q - z) s)            "subtract": z per group and output, or 8
//   W = rnd(q s + zs), zs = -rnd(s z)   "fma";     W = rnd(rnd(q s) + zs)   "two roundings"
// rnd rounds to bf16: the effective weights of csrc/quant.cu bit for bit, so the products are those of the layer's
// arithmetic whichever kernel serves it. Sums in fp32, one rounding of y to bf16.
//
// Bound by the codes' bytes (N K / 2), so the work per code is what is counted. A code becomes bf16 by its bits:
// 0x4300 | q is 128 + q exactly, less (128 + z) is q - z exactly, times s is W with its one rounding: 7.5 instructions
// for 4 pairs of weights, then one mma.m16n8k16 (A = W: 16 outputs, B = x^T: 8 rows of x) takes 8 weights of each
// lane. The order of k within a product is free, so a lane takes 16 bytes (32 weights) of a row as they lie in memory,
// pairs (i, i + 4) of each word as they come out of the nibbles, and reads x in the same order.
//
// A CTA of 8 warps computes 16 MT outputs; its warps take every 8th block of 128 k and merge in warp order. Each
// output's arithmetic depends on its codes and x's row alone (not on M, MT or the CTA), so running some blocks of 16
// outputs again gives the same bits: check mode compares them with y.
#include "common.cuh"

namespace sdc {
namespace matvec4 {

constexpr int WARPS = 8;
constexpr int KB = 128;       // k per warp step: 4 lanes x 32

enum { ZERO_SUBTRACT = 0, ZERO_FMA = 1, ZERO_TWO = 2 };

struct Params {
  const uint8_t* codes;            // [N][K / 2]
  const __nv_bfloat16* scales;     // [N][K / group]
  const uint8_t* zeros;            // [N][K / group] or null (8)
  const __nv_bfloat16* x;          // M rows, `ldx` apart
  long long ldx;
  const float* bias;               // [N] or null, added before y is rounded
  __nv_bfloat16* y;                // M rows, `ldy` apart
  long long ldy;
  int M, N, K, group, ng;
  const int* blocks;               // check mode: blocks of 16 outputs
  unsigned long long* check;
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t word(const uint4& u, int j) { return j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w; }

// Weights (i, i + 4) of a word of eight codes.
template <int MODE>
__device__ __forceinline__ uint32_t pair(uint32_t w, int i, __nv_bfloat162 zero, __nv_bfloat162 scale, __nv_bfloat162 zs) {
  const uint32_t q = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;        // 128 + q
  const __nv_bfloat162 v = __hsub2_rn(as_bf2(q), zero);                   // q - z, or q: exact
  if (MODE == ZERO_SUBTRACT) return as_u32(__hmul2_rn(v, scale));
  if (MODE == ZERO_FMA) return as_u32(__hfma2(v, scale, zs));
  return as_u32(__hadd2_rn(__hmul2_rn(v, scale), zs));
}

// NT: groups of eight rows of x; MT: groups of 16 outputs a warp holds.
template <int NT, int MT, int MODE>
__global__ void __launch_bounds__(WARPS * 32) matvec4_kernel(const Params p) {
  pdl_trigger();
  __shared__ float red[WARPS][NT * 8][MT * 16 + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = (p.blocks ? p.blocks[blockIdx.x] : static_cast<int>(blockIdx.x) * MT) * 16;
  if (p.check != nullptr && blockIdx.x == 0 && tid == 0) atomicAdd(p.check + 2, 1ull);
  if (n0 < 0 || n0 >= p.N) return;
  float acc[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  const __nv_bfloat162 magic = as_bf2(0x43004300u);
  const int nkb = (p.K + KB - 1) / KB;
#pragma unroll 2
  for (int kb = warp; kb < nkb; kb += WARPS) {
    const int k = kb * KB + 32 * t;
    const bool in = k < p.K;             // K is a multiple of 32
    uint4 w[MT][2];
    __nv_bfloat162 sc[MT][2], ze[MT][2], zs[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int n = n0 + i * 16 + r * 8 + g;
        const bool ok = in && n < p.N;
        w[i][r] = ok ? ld_stream(p.codes + static_cast<long long>(n) * (p.K / 2) + k / 2) : make_uint4(0, 0, 0, 0);
        const long long gi = static_cast<long long>(n) * p.ng + k / p.group;
        const __nv_bfloat16 s = ok ? p.scales[gi] : __float2bfloat16(0.f);
        const int z = p.zeros == nullptr ? 8 : ok ? p.zeros[gi] : 0;
        sc[i][r] = __bfloat162bfloat162(s);
        if (MODE == ZERO_SUBTRACT) {
          ze[i][r] = __bfloat162bfloat162(__int2bfloat16_rn(128 + z));
        } else {
          ze[i][r] = magic;
          zs[i][r] = __bfloat162bfloat162(__float2bfloat16_rn(-__bfloat162float(s) * static_cast<float>(z)));
        }
      }
    uint4 xr[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int m = j * 8 + g;
      const uint4* src = reinterpret_cast<const uint4*>(p.x + m * p.ldx + k);
#pragma unroll
      for (int c = 0; c < 4; ++c) xr[j][c] = in && m < p.M ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {          // word c: k + 8c .. k + 8c + 7
      uint32_t b[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        b[j][0] = __byte_perm(xr[j][c].x, xr[j][c].z, 0x5410);    // x0, x4
        b[j][1] = __byte_perm(xr[j][c].x, xr[j][c].z, 0x7632);    // x1, x5
        b[j][2] = __byte_perm(xr[j][c].y, xr[j][c].w, 0x5410);    // x2, x6
        b[j][3] = __byte_perm(xr[j][c].y, xr[j][c].w, 0x7632);    // x3, x7
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint32_t w0 = word(w[i][0], c), w1 = word(w[i][1], c);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a[4] = {pair<MODE>(w0, 2 * h, ze[i][0], sc[i][0], zs[i][0]),
                                 pair<MODE>(w1, 2 * h, ze[i][1], sc[i][1], zs[i][1]),
                                 pair<MODE>(w0, 2 * h + 1, ze[i][0], sc[i][0], zs[i][0]),
                                 pair<MODE>(w1, 2 * h + 1, ze[i][1], sc[i][1], zs[i][1])};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma(acc[i][j], a, b[j][2 * h], b[j][2 * h + 1]);
        }
      }
    }
  }
  // acc[i][j]: outputs 16 i + g (+ 8), rows 8 j + 2t (+ 1)
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][j * 8 + 2 * t + (e & 1)][i * 16 + g + (e >> 1) * 8] = acc[i][j][e];
  __syncthreads();
  for (int i = tid; i < p.M * MT * 16; i += WARPS * 32) {
    const int m = i / (MT * 16), c = i % (MT * 16), n = n0 + c;
    if (n >= p.N) continue;
    float s = red[0][m][c];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) s += red[w][m][c];
    if (p.bias != nullptr) s += p.bias[n];
    __nv_bfloat16* dst = p.y + m * p.ldy + n;
    const __nv_bfloat16 r = __float2bfloat16(s);
    if (p.check == nullptr) {
      *dst = r;
    } else {
      const float a = __bfloat162float(r), b = __bfloat162float(*dst);
      if (!(a == b) && !(a != a && b != b))
        report_replay_mismatch(p.check, static_cast<unsigned long long>(m) * p.N + n);
    }
  }
}

template <int NT, int MT>
static int launch(const Params& p, int mode, int grid, cudaStream_t st) {
  switch (mode) {
    case ZERO_SUBTRACT: matvec4_kernel<NT, MT, ZERO_SUBTRACT><<<grid, WARPS * 32, 0, st>>>(p); break;
    case ZERO_FMA: matvec4_kernel<NT, MT, ZERO_FMA><<<grid, WARPS * 32, 0, st>>>(p); break;
    default: matvec4_kernel<NT, MT, ZERO_TWO><<<grid, WARPS * 32, 0, st>>>(p); break;
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace matvec4
}  // namespace sdc

using namespace sdc::matvec4;

extern "C" int sdc_matvec4(const void* x, long long ldx, int M, int N, int K, int group, const void* codes,
                           const void* scales, const void* zeros, int mode, const void* bias, void* y,
                           long long ldy, const int* blocks, int nblocks, void* check, void* stream) {
  if (M <= 0 || N <= 0) return 0;
  if (M > 32 || K <= 0 || K % 32 || group <= 0 || group % 32 || K % group || ldx % 8 || mode < 0 || mode > 2 ||
      (mode != ZERO_SUBTRACT && zeros == nullptr) || (check != nullptr) != (blocks != nullptr))
    return -1;
  Params p;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = static_cast<const __nv_bfloat16*>(scales);
  p.zeros = static_cast<const uint8_t*>(zeros);
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.ldx = ldx;
  p.bias = static_cast<const float*>(bias);
  p.y = static_cast<__nv_bfloat16*>(y);
  p.ldy = ldy;
  p.M = M;
  p.N = N;
  p.K = K;
  p.group = group;
  p.ng = K / group;
  p.blocks = blocks;
  p.check = static_cast<unsigned long long*>(check);
  auto st = static_cast<cudaStream_t>(stream);
  if (blocks != nullptr) {
    if (nblocks <= 0) return 0;
    return M <= 8 ? launch<1, 1>(p, mode, nblocks, st)
                  : M <= 16 ? launch<2, 1>(p, mode, nblocks, st) : launch<4, 1>(p, mode, nblocks, st);
  }
  if (M <= 8) return launch<1, 1>(p, mode, (N + 15) / 16, st);
  if (M <= 16) return launch<2, 2>(p, mode, (N + 31) / 32, st);
  return launch<4, 2>(p, mode, (N + 31) / 32, st);
}
