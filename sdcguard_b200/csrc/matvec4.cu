// Products of a few rows with 4-bit weights and group scales (sm_100a): y = x W^T, x [M][K] bf16, M <= 32, with W read
// as its codes (a quarter of the bytes of the bf16 matrix).
//
//   W = rnd((q - z) s)            "subtract": z per group and output, or 8
//   W = rnd(q s + zs), zs = -rnd(s z)   "fma";     W = rnd(rnd(q s) + zs)   "two roundings"
// rnd rounds to bf16: the effective weights of csrc/quant.cu bit for bit, so the products are those of the layer's
// arithmetic whichever kernel serves it. Sums in fp32, one rounding of y to bf16.
//
// Codes become bf16 weights in pairs without a conversion (see `weights`), then one mma.m16n8k16 (A = W: 16 outputs, B =
// x^T: 8 rows of x) takes 8 weights of each lane. The order of k within a product is free, so a lane takes 16 bytes (32
// weights) of a row as they lie in memory, pairs (i, i + 4) of each word as masks give them, and reads x in the same
// order.
//
// The bytes that must move are the codes' (N K / 2). Device times: 1 x 4096 x 4096 4.6 us (its bytes alone 1.3), launch and
// one wave of CTAs; 1 x 28672 x 4096 19.2 us, 13 x 28672 x 4096 with zero points 28 us, against 10 of a bare read of the
// matrix and 13 of this kernel without forming the weights and without reading x and scales. The last runs at 1.75
// instructions a cycle and waits for loads longest (3.2 warps of 15 at each issue): x comes to each CTA from L2 and the scales
// two bytes at a time, beside three instructions a pair of weights. Codes through shared memory (TMA or cp.async rings),
// scales staged there behind a barrier and CTAs that walk over tiles gave the same times.
//
// A CTA computes 16 MT outputs. The k blocks (128 each) of an output go to its WARPS warps in turn, whose sums merge in
// order at the end; WARPS follows from the matrix's shape. Each output's arithmetic depends on its codes and x's row alone
// (not on M, MT or the CTA), so a row of x gives the same bits in any batch, and running some blocks of 16 outputs again
// gives them too: check mode compares them with y.
#include "common.cuh"

namespace sdc {
namespace matvec4 {

constexpr int KB = 128;       // k per block: 4 lanes x 32

enum { ZERO_SUBTRACT = 0, ZERO_FMA = 1, ZERO_TWO = 2, ZERO_EIGHT = 3 };   // EIGHT: subtract without zero points

struct Params {
  const uint8_t* codes;            // [N][K / 2]
  const __nv_bfloat16* scales;     // [N][K / group]
  const uint8_t* zeros;            // [N][K / group] or null (8)
  const __nv_bfloat16* x;          // M rows, `ldx` apart
  long long ldx;
  const float* bias;               // [N] or null, added before y is rounded
  __nv_bfloat16* y;                // M rows, `ldy` apart
  long long ldy;
  int M, N, K, ng;
  float per_group;                 // 32 / group
  uint4* packed;                   // x in the order the products take it (pack_x), or null: read from x
  const int* blocks;               // check mode: blocks of 16 outputs
  unsigned long long* check;
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 r;
  asm("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t word(const uint4& u, int j) { return j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w; }

__device__ const uint4 no_x[4] = {};     // what lanes behind K read for x

// bf16 bits below 256 are the numbers 0 .. 255 times 2^-133: the subnormals and the first binade have one spacing. So a
// masked word is a pair of codes as it stands (in bits 0-3 of each half q, in bits 4-7 16 q), one shift serves four
// codes, and a scale times 2^100 (2^96) takes the exponent back, to W 2^-33. With z = 8 the product and 8 s, a power of
// two times s, meet in one fma and its one rounding: 9 instructions for 8 weights. Scales below 2^27 fit the factor
// (larger ones give NaN), and W is exact from 2^-93 up.
constexpr float BACK = 8589934592.f;     // 2^33
struct Factor {
  __nv_bfloat162 s, z, add;              // scale 2^100, zero point (a code's form), what is added behind the product
};
template <int MODE>
__device__ __forceinline__ Factor factor_of(uint32_t scale, uint32_t z) {
  Factor f;
  const __nv_bfloat162 s = as_bf2(scale * 0x10001u);
  f.s = __hmul2_rn(s, as_bf2(0x71807180u));                                          // 2^100
  f.z = as_bf2(z * 0x10001u);
  if (MODE == ZERO_EIGHT) f.add = __hmul2_rn(s, as_bf2(0xb080b080u));                // -8 2^-33
  if (MODE == ZERO_FMA || MODE == ZERO_TWO)
    f.add = __hmul2_rn(__hmul2_rn(s, __float2bfloat162_rn(-static_cast<float>(z))), as_bf2(0x2f002f00u));   // rnd, 2^-33
  return f;
}
// The same for codes in bits 4-7: 16 times larger.
template <int MODE>
__device__ __forceinline__ Factor high_factor(const Factor& f) {
  Factor h = f;
  h.s = __hmul2_rn(f.s, as_bf2(0x3d803d80u));                                        // 1 / 16
  if (MODE == ZERO_SUBTRACT) h.z = __hmul2_rn(f.z, as_bf2(0x41804180u));             // 16
  return h;
}
template <int MODE>
__device__ __forceinline__ uint32_t weights(uint32_t q, const Factor& f) {
  const __nv_bfloat162 v = as_bf2(q);
  if (MODE == ZERO_SUBTRACT) return as_u32(__hmul2_rn(__hsub2_rn(v, f.z), f.s));
  if (MODE == ZERO_TWO) return as_u32(__hadd2_rn(__hmul2_rn(v, f.s), f.add));
  return as_u32(__hfma2(v, f.s, f.add));
}
// x for `PACKED` products: for each block of 128 k, word c of the codes and group j of eight rows, the four pairs of every
// lane side by side. With more than eight rows each CTA reads more bytes of x than of codes, 16 at a time from 32 places;
// packed once, they come in whole lines and without permutes.
__device__ __forceinline__ uint4 pairs_of(const uint4& x) {
  return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632),     // (x0, x4), (x1, x5)
                    __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));    // (x2, x6), (x3, x7)
}
template <int NT>
__global__ void __launch_bounds__(256) pack_x_kernel(const Params p) {
  pdl_trigger();
  const int i = blockIdx.x * 256 + threadIdx.x, lane = i & 31, j = (i >> 5) % NT, kc = (i >> 5) / NT;
  const int k = (kc >> 2) * KB + 32 * (lane & 3) + 8 * (kc & 3), m = j * 8 + (lane >> 2);
  if ((kc >> 2) * KB >= p.K) return;
  p.packed[i] = k < p.K && m < p.M ? pairs_of(*reinterpret_cast<const uint4*>(p.x + m * p.ldx + k)) : make_uint4(0, 0, 0, 0);
}

// NT: groups of eight rows of x; MT: groups of 16 outputs; PF: k blocks in flight per warp. Outputs behind N and rows of
// x behind M are computed from the last ones there are and not written, which costs no predicates in the loop.
template <int NT, int MT, int WARPS, int PF, int CTAS, int MODE, bool PACKED>
__global__ void __launch_bounds__(WARPS * 32, CTAS) matvec4_kernel(const Params p) {
  pdl_trigger();
  __shared__ float red[WARPS][NT * 8][MT * 16 + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = (p.blocks ? p.blocks[blockIdx.x] : static_cast<int>(blockIdx.x) * MT) * 16;
  if (p.check != nullptr && blockIdx.x == 0 && tid == 0) atomicAdd(p.check + 2, 1ull);
  if (n0 < 0 || n0 >= p.N) return;
  const int nkb = (p.K + KB - 1) / KB;
  const uint8_t* code[MT][2];
  int meta[MT][2];                       // of the outputs' scales and zero points
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int n = min(n0 + i * 16 + r * 8 + g, p.N - 1);
      code[i][r] = p.codes + static_cast<long long>(n) * (p.K / 2);
      meta[i][r] = n * p.ng;
    }
  const __nv_bfloat16* xrow[NT];
  if (!PACKED)
#pragma unroll
  for (int j = 0; j < NT; ++j) xrow[j] = p.x + min(j * 8 + g, p.M - 1) * p.ldx;
  uint4 w[PF][MT][2];                    // a lane's 32 codes, scale and zero point of 2 MT outputs
  uint32_t ws[PF][MT][2], wz[PF][MT][2];
  int lk = warp;                         // the next block to load: every WARPS-th is this warp's
  const auto load_next = [&](int f) {
    if (lk < nkb) {
      const int k = lk * KB + 32 * t;
      const int kc = k < p.K ? k : 0;    // the last block may end early (K is a multiple of 32): x is 0 there
      const int gi = static_cast<int>((static_cast<float>(kc >> 5) + 0.5f) * p.per_group);     // kc / group
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          w[f][i][r] = ld_stream(code[i][r] + (kc >> 1));
          ws[f][i][r] = __ldg(reinterpret_cast<const unsigned short*>(p.scales) + meta[i][r] + gi);
          if (MODE != ZERO_EIGHT) wz[f][i][r] = __ldg(p.zeros + meta[i][r] + gi);
        }
    }
    lk += WARPS;
  };
#pragma unroll
  for (int f = 0; f < PF; ++f) load_next(f);
  if (PACKED) pdl_wait();                // the codes are on their way meanwhile
  float acc[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  for (int kb = warp; kb < nkb; kb += WARPS * PF) {
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      const int kc = kb + f * WARPS;
      if (kc < nkb) {                  // (uniform)
        const int k = kc * KB + 32 * t;
        const uint4* xp[NT];
        if (!PACKED)
#pragma unroll
        for (int j = 0; j < NT; ++j) xp[j] = k < p.K ? reinterpret_cast<const uint4*>(xrow[j] + k) : no_x;
        Factor lo[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) lo[i][r] = factor_of<MODE>(ws[f][i][r], MODE == ZERO_EIGHT ? 8u : wz[f][i][r]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {        // word c: k + 8c .. k + 8c + 7
          uint32_t b[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 x = PACKED ? p.packed[((kc * 4 + c) * NT + j) * 32 + lane] : pairs_of(__ldg(xp[j] + c));
            b[j][0] = x.x;
            b[j][1] = x.y;
            b[j][2] = x.z;
            b[j][3] = x.w;
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const uint32_t w0 = word(w[f][i][0], c), w1 = word(w[f][i][1], c);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t u0 = h ? w0 >> 8 : w0, u1 = h ? w1 >> 8 : w1;
              const uint32_t a[4] = {weights<MODE>(u0 & 0x000f000fu, lo[i][0]), weights<MODE>(u1 & 0x000f000fu, lo[i][1]),
                               weights<MODE>(u0 & 0x00f000f0u, high_factor<MODE>(lo[i][0])),
                               weights<MODE>(u1 & 0x00f000f0u, high_factor<MODE>(lo[i][1]))};
#pragma unroll
              for (int j = 0; j < NT; ++j) mma(acc[i][j], a, b[j][2 * h], b[j][2 * h + 1]);
            }
          }
        }
      }
      load_next(f);
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
    s *= BACK;
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

template <int NT, int MT, int WARPS, int PF, int CTAS, int MODE, bool PACKED>
static int launch_mode(const Params& p, int grid, cudaStream_t st) {
  if constexpr (!PACKED) {
    matvec4_kernel<NT, MT, WARPS, PF, CTAS, MODE, false><<<grid, WARPS * 32, 0, st>>>(p);
    return static_cast<int>(cudaGetLastError());
  } else {
    const int nkb = (p.K + KB - 1) / KB;
    pack_x_kernel<NT><<<(nkb * 4 * NT * 32 + 255) / 256, 256, 0, st>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, matvec4_kernel<NT, MT, WARPS, PF, CTAS, MODE, true>, p));
  }
}
template <int NT, int MT, int WARPS, int PF, int CTAS, bool PACKED = false>
static int launch(const Params& p, int mode, int grid, cudaStream_t st) {
  if (mode == ZERO_FMA) return launch_mode<NT, MT, WARPS, PF, CTAS, ZERO_FMA, PACKED>(p, grid, st);
  if (mode == ZERO_TWO) return launch_mode<NT, MT, WARPS, PF, CTAS, ZERO_TWO, PACKED>(p, grid, st);
  if (p.zeros != nullptr) return launch_mode<NT, MT, WARPS, PF, CTAS, ZERO_SUBTRACT, PACKED>(p, grid, st);
  return launch_mode<NT, MT, WARPS, PF, CTAS, ZERO_EIGHT, PACKED>(p, grid, st);
}

}  // namespace matvec4
}  // namespace sdc

using namespace sdc::matvec4;

// The arguments in one struct (see kv8.cu).
struct Matvec4Args {
  const void* x;
  long long ldx;
  int M;
  int N;
  int K;
  int group;
  const void* codes;
  const void* scales;
  const void* zeros;
  int mode;
  const void* bias;
  void* y;
  long long ldy;
  void* packed;
  const int* blocks;
  int nblocks;
  void* check;
  void* stream;
};
extern "C" int sdc_matvec4(const Matvec4Args* args) {
  const auto& [x, ldx, M, N, K, group, codes, scales, zeros, mode, bias, y, ldy, packed, blocks, nblocks,
               check, stream] = *args;
  if (M <= 0 || N <= 0) return 0;
  // scale indices fit 32 bits, and (k / 32 + 1/2) * (32 / group) in fp32 finds a k's group up to K = 2^25
  if (static_cast<long long>(N) * (K / 32) > 0x7fffffffll || K > (1 << 25)) return -1;
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
  p.ng = K / group;
  p.per_group = 32.f / static_cast<float>(group);
  p.packed = static_cast<uint4*>(packed);
  p.blocks = blocks;
  p.check = static_cast<unsigned long long*>(check);
  auto st = static_cast<cudaStream_t>(stream);
  // 8 warps a CTA; few outputs and a long k leave each warp much to do and the SMs with few warps, so that 16 take it
  // (8 x 4096 x 14336: 12.4 us, with 8 17.0; 1 x 4096 x 8192: 8.4 and 9.8; 1 x 9216 x 4096 the other way: 8.8 and 7.6)
  const bool deep = N <= 148 * 32 && K >= 8192;
  if (blocks != nullptr) {
    if (nblocks <= 0) return 0;
    if (deep)
      return M <= 8 ? launch<1, 1, 16, 2, 2>(p, mode, nblocks, st)
                    : M <= 16 ? launch<2, 1, 16, 2, 1>(p, mode, nblocks, st) : launch<4, 1, 16, 2, 1>(p, mode, nblocks, st);
    return M <= 8 ? launch<1, 1, 8, 2, 4>(p, mode, nblocks, st)
                  : M <= 16 ? launch<2, 1, 8, 2, 3>(p, mode, nblocks, st) : launch<4, 1, 8, 2, 2>(p, mode, nblocks, st);
  }
  // two groups of 16 outputs a warp share the reads of x, where nearly two CTAs per SM remain (16 x 9216 x 4096: 10.2 us
  // against 13.0 with one group, 1 x 28672 x 4096 19.2 and 20.6; the other way 1 x 9216 x 4096: 8.0 and 7.6, 16 x 6144 x
  // 4096: 9.6 and 8.5), of 16 warps one (8 x 4096 x 14336: 12.3 us against 13.9; 8 x 1024 x 4096: 4.6 and 3.7)
  const bool wide = N >= 8192;
  const int g1 = (N + 15) / 16, g2 = (N + 31) / 32;
  if (deep) {
    if (M <= 8) return N > 148 * 16 ? launch<1, 2, 16, 1, 1>(p, mode, g2, st) : launch<1, 1, 16, 2, 2>(p, mode, g1, st);
    if (M <= 16) return packed ? launch<2, 1, 16, 1, 2, true>(p, mode, g1, st) : launch<2, 1, 16, 2, 1>(p, mode, g1, st);
    return packed ? launch<4, 1, 16, 1, 2, true>(p, mode, g1, st) : launch<4, 1, 16, 2, 1>(p, mode, g1, st);
  }
  if (M <= 8) return wide ? launch<1, 2, 8, 1, 3>(p, mode, g2, st) : launch<1, 1, 8, 2, 4>(p, mode, g1, st);
  if (M <= 16) {
    if (packed) return wide ? launch<2, 2, 8, 1, 2, true>(p, mode, g2, st) : launch<2, 1, 8, 2, 3, true>(p, mode, g1, st);
    return launch<2, 2, 8, 1, 2>(p, mode, g2, st);
  }
  if (packed) return wide ? launch<4, 2, 8, 1, 2, true>(p, mode, g2, st) : launch<4, 1, 8, 2, 2, true>(p, mode, g1, st);
  return launch<4, 2, 8, 2, 1>(p, mode, g2, st);
}
