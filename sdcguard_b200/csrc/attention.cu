// Paged-KV attention for serving (sm_100a): causal prefill (tcgen05 MMAs with S and O in TMEM, online softmax
// with a conditional rescale) and single-token decode (split-KV, TMA-staged chunks, mma.m16n8k16), for
// grouped-query attention with head_dim 128 and 16-token KV pages.
//
// KV cache layout for one layer: [num_blocks][2 (K, V)][kv_heads][16][128] bf16; a request's pages are listed
// in its row of the block table.
//
// Row determinism. The arithmetic that produces one output row depends only on that row's query, its
// position and the keys: key tiles start at absolute multiples of the tile size, tiles that are fully masked for a row
// leave its running max, sum and accumulator bit-identical (scale exp2(0) = 1, p = 0), and reductions run in
// a fixed order. So running the same kernel again on any subset of rows (the `row_idx` list) reproduces their
// outputs exactly. The serving check uses this: a rotating 1/64 sample of rows is recomputed on different
// CTAs/SMs at a different time and compared bit for bit (sdcguard_b200/ops/attention.py). The reference checks
// attention by a sampled fp32 recompute against an error bound (src/sdcguard/serve_attn.py:5-48, kernels
// `_attn_part` :335 and `_attn_judge` :414); an exact replay needs no bound and sees every flipped bit.
#include <atomic>
#include <cstdlib>

#include "common.cuh"
#include "tma_host.h"

namespace sdc {
namespace attn {

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr int ROWS = 128;  // (token, head) rows per prefill CTA

struct PrefillParams {
  const __nv_bfloat16* q;     // [T, nq, D]
  __nv_bfloat16* o;           // [T, nq, D]
  const __nv_bfloat16* cache; // layer cache
  const int* block_table;     // [R, max_pages]
  int max_pages;
  const int* pos;             // [T] absolute position of each token; from `limit` on: a row without keys
  int limit;
  const int4* tiles;          // (request, first token, tokens, offset into row_idx or -1)
  const int* row_idx;
  int nq, nkv;
  float scale_log2;           // softmax scale * log2(e)
  float* row_sq;              // [T] += ||o_token||^2 over heads (zeroed by the caller), or null
  unsigned long long* check;  // check mode: compare with o instead of writing (state row), or null
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------------------------------- prefill, tcgen05
// The same tiles and row determinism as `prefill_kernel`, on the 5th-generation tensor cores:
//   warp 0   TMA: the request's K and V pages of a 128-key tile (one 16-row x 128-byte box per page, half the head
//            dim, K or V, 128-byte swizzle) into one of two stages; V rows behind the last key that a row of the tile
//            sees are cleared (see v_rows);
//   warp 1   MMA: S = Q K^T into one of two TMEM accumulators (M = 128 rows, N = 128 keys, K = 128), and
//            O += P V into a third (V as an MN-major operand, dims contiguous); S of tile j+1 is computed while
//            the softmax works on tile j;
//   warps 4-7 one thread per row: read S from TMEM, causal mask, running max with a conditional rescale (the
//            reference maximum only moves when a row's maximum grows by more than 2^8, so O in TMEM is rescaled
//            rarely), P = exp2(S - max) as bf16 into shared memory (the A operand of PV), the row sum of the bf16
//            weights, and at the end O / l to the output (or compared with it in check mode).
// Every decision is per row, key tiles start at absolute multiples of 128, and fully masked tiles change nothing,
// so a replay of any subset of rows reproduces their outputs bit for bit.
namespace pf {
constexpr int KT = 128;                   // keys per tile
constexpr int HALF_B = 128 * 128;         // one dims-half (64 bf16 = 128 B) of a 128-row tile
constexpr int TILE_B = 2 * HALF_B;        // 32 KB: 128 rows x 128 dims bf16
constexpr int OFF_Q = 0, OFF_K = TILE_B, OFF_V = 3 * TILE_B, OFF_P = 5 * TILE_B, OFF_CTL = 6 * TILE_B;
constexpr float RESCALE_LOG2 = 8.f;
constexpr int PG_BYTES = PAGE * D * 2;    // one page of K (or V) of one kv head
struct Ctl {
  uint64_t k_full[2], v_full[2], kv_empty[2], s_full[2], s_empty[2];
  uint64_t p_full, pv_done, q_ready, drain;
  uint32_t tmem_base;
  int abort_flag;
  int maxpos;
  int tok[ROWS];
  int pos[ROWS];
  float xm[2][2][ROWS];                   // [tile parity][warpgroup][row] partial maxima of a tile
  float xl[2][ROWS];                      // [warpgroup][row] partial row sums at the end
};
constexpr int SMEM = OFF_CTL + static_cast<int>(sizeof(Ctl)) + 1024;
constexpr int SOFT = 2 * ROWS;            // softmax threads: warpgroup g takes keys / dims [64 g, 64 g + 64)
}  // namespace pf

// The reference maximum of a row without a score above -inf so far. Maxima pass over NaN: with -inf in its place scores of
// NaN would look like masked ones; against this one their weights are NaN, and those of -inf 0.
constexpr float NO_SCORE = -3.402823466e38f;

// V of a key tile, of which rows [0, n) are keys that some row of the query tiles sees. The weights of the others are zero,
// but the MMA multiplies V by them, and 0 * NaN is NaN: what a page holds behind its sequence's end is whatever was stored
// there last, as is shared memory that nothing was loaded to. So only keys are loaded (the last page's one by one, through
// `tr`, whose box is one row) and the rest is cleared. (Keys that one row sees and another does not stay: a V of NaN reaches
// its dim in rows of the same query tile up to 254 places before it.) One warp; returns behind the clearing, which the loads'
// barrier publishes.
constexpr int V_HALF = 128 * 128;         // bytes of 64 dims of a tile
__device__ __forceinline__ void clear_v(uint8_t* buf, int n, int lane) {
  for (int i = lane; i < (128 - n) * 16; i += 32) {
    const int r = n + (i >> 4), c = i & 15;
    *reinterpret_cast<uint4*>(buf + (c >> 3) * V_HALF + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}
// The keys of the last, partial page: `row` is its first row in the map, n the tile's keys.
__device__ __forceinline__ void load_v_rest(uint8_t* buf, const CUtensorMap* tr, uint64_t* bar, int row, int n, int lane) {
  const int r = lane >> 1, half = lane & 1;
  if (r < n % PAGE) tma_load_2d(buf + half * V_HALF + (n / PAGE * PAGE + r) * 128, tr, bar, half * 64, row + r);
}

__global__ void __launch_bounds__(128 + 2 * ROWS, 1) prefill_tc_kernel(const __grid_constant__ CUtensorMap tm,
                                                            const __grid_constant__ CUtensorMap tr,
                                                            const PrefillParams p) {
  pdl_trigger();   // a dependent GEMM may start its prologue and weight loads now
  using namespace pf;
  extern __shared__ uint8_t pf_raw[];
  uint8_t* sm = pf_raw + ((1024 - (smem_u32(pf_raw) & 1023)) & 1023);
  Ctl* ctl = reinterpret_cast<Ctl*>(sm + OFF_CTL);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.nq / p.nkv;
  const int tpc = ROWS / G;
  const int4 tile = p.tiles[blockIdx.x];
  const int req = tile.x, kvh = blockIdx.y;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->k_full[i], 1);
      mbar_init(&ctl->v_full[i], 1);
      mbar_init(&ctl->kv_empty[i], 1);
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->s_empty[i], SOFT);
    }
    mbar_init(&ctl->p_full, SOFT);
    mbar_init(&ctl->pv_done, 1);
    mbar_init(&ctl->q_ready, SOFT);
    mbar_init(&ctl->drain, 1);
    ctl->abort_flag = 0;
    ctl->maxpos = -1;
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tm);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid >= 128 && tid < 128 + ROWS) {
    const int r = tid - 128;
    const int ti = r / G;
    int tok = -1;
    if (ti < tile.z && ti < tpc) tok = tile.w >= 0 ? p.row_idx[tile.w + ti] : tile.y + ti;
    ctl->tok[r] = tok;
    int ps = tok >= 0 ? p.pos[tok] : -1;
    if (ps >= p.limit) ps = -1;
    ctl->pos[r] = ps;
    if (ps >= 0) atomicMax(&ctl->maxpos, ps);
  }
  __syncthreads();
  const int maxpos = ctl->maxpos;
  const int ntiles = maxpos >= 0 ? maxpos / KT + 1 : 0;
  const uint32_t tmem = ctl->tmem_base;
  volatile int* abort_flag = &ctl->abort_flag;
  const int* bt = p.block_table + static_cast<long long>(req) * p.max_pages;

  if (warp == 0 && ntiles > 0) {
    // ------------------------------------------------------------ TMA producer (all 32 lanes issue)
    pdl_wait();                           // the pages may come from the kernel before (launched with overlap)
    bool ok = true;
    int last = -1;                        // last tile whose loads were issued
    for (int j = 0; j < ntiles && ok; ++j) {
      const int st = j & 1;
      bool got = true;
      if (lane == 0) got = mbar_wait(&ctl->kv_empty[st], ((j >> 1) & 1u) ^ 1u, abort_flag);
      if (!__shfl_sync(0xffffffffu, got ? 1 : 0, 0)) {
        ok = false;
        break;
      }
      const int nkeys = min(KT, maxpos + 1 - j * KT), npg = (nkeys + PAGE - 1) / PAGE;
      uint8_t* kbuf = sm + OFF_K + st * TILE_B;
      uint8_t* vbuf = sm + OFF_V + st * TILE_B;
      if (nkeys < KT) clear_v(vbuf, nkeys, lane);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_expect_tx(&ctl->k_full[st], npg * PG_BYTES);
        mbar_arrive_expect_tx(&ctl->v_full[st], nkeys * (PG_BYTES / PAGE));
      }
      __syncwarp();
      const auto row_of = [&](int pg, int kv) {
        return static_cast<int>(((static_cast<long long>(bt[j * (KT / PAGE) + pg]) * 2 + kv) * p.nkv + kvh) * PAGE);
      };
      const int pg = lane >> 2, kv = (lane >> 1) & 1, half = lane & 1;
      if (pg < (kv ? nkeys / PAGE : npg))
        tma_load_2d((kv ? vbuf : kbuf) + half * HALF_B + pg * PAGE * 128, &tm, kv ? &ctl->v_full[st] : &ctl->k_full[st],
                    half * 64, row_of(pg, kv));
      if (nkeys % PAGE) load_v_rest(vbuf, &tr, &ctl->v_full[st], row_of(npg - 1, 1), nkeys, lane);
      last = j;
    }
    if (!ok && lane == 0) {
      record_error(nullptr, ERR_TIMEOUT_PRODUCER);
      *abort_flag = 1;
      // the copies already issued must land before the CTA's shared memory is released (bounded waits)
      for (int j = last > 0 ? last - 1 : 0; j <= last; ++j) {
        mbar_wait(&ctl->k_full[j & 1], (j >> 1) & 1u, nullptr);
        mbar_wait(&ctl->v_full[j & 1], (j >> 1) & 1u, nullptr);
      }
    }
  } else if (warp == 1 && ntiles > 0) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      bool ok = mbar_wait(&ctl->q_ready, 0, abort_flag);
      const uint32_t idesc_s = idesc_bf16_f32(128, KT);
      const uint32_t idesc_o = idesc_bf16_f32(128, D) | (1u << 16);     // B (V) MN-major
      const uint32_t qa = smem_u32(sm + OFF_Q), pa = smem_u32(sm + OFF_P);
      for (int j = 0; j <= ntiles && ok; ++j) {
        if (j < ntiles) {
          const int st = j & 1;
          const uint32_t par = (j >> 1) & 1u;
          ok = mbar_wait(&ctl->k_full[st], par, abort_flag) && mbar_wait(&ctl->s_empty[st], par ^ 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ka = smem_u32(sm + OFF_K + st * TILE_B);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = (ks >> 2) * HALF_B + (ks & 3) * 32;
            umma_f16(tmem + st * KT, umma_desc_sw128(qa + off), umma_desc_sw128(ka + off), idesc_s, ks ? 1u : 0u);
          }
          umma_commit(&ctl->s_full[st]);
        }
        if (j >= 1) {
          const int jj = j - 1, st = jj & 1;
          ok = mbar_wait(&ctl->p_full, jj & 1u, abort_flag) && mbar_wait(&ctl->v_full[st], (jj >> 1) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t va = smem_u32(sm + OFF_V + st * TILE_B);
#pragma unroll
          for (int ks = 0; ks < KT / 16; ++ks) {
            const uint64_t ad = umma_desc_sw128(pa + (ks >> 2) * HALF_B + (ks & 3) * 32);
            const uint64_t bd = umma_desc_sw128_mn(va + ks * 2048, HALF_B, 1024);
            umma_f16(tmem + 2 * KT, ad, bd, idesc_o, (jj > 0 || ks > 0) ? 1u : 0u);
          }
          umma_commit(&ctl->pv_done);
          umma_commit(&ctl->kv_empty[st]);
        }
      }
      if (!ok) {
        record_error(nullptr, ERR_TIMEOUT_MMA);
        *abort_flag = 1;
        umma_commit(&ctl->drain);           // let the issued MMAs land before TMEM is released
        mbar_wait(&ctl->drain, 0, nullptr);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax / output: thread = (row, half)
    // warpgroup gi takes keys [64 gi, 64 gi + 64) of every tile and dims [64 gi, 64 gi + 64) of O; the two
    // halves of a row agree on the maximum through shared memory, so both take the same rescale decisions
    const int gi = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int tok = ctl->tok[r];
    const int pos = ctl->pos[r];
    const int head = kvh * G + (r % G);
    // Q row, this warpgroup's dims half -> shared memory (128-byte swizzle)
    {
      uint8_t* qd = sm + OFF_Q + gi * HALF_B;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (static_cast<long long>(tok < 0 ? 0 : tok) * p.nq + head) * D +
                                                        gi * 64);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 v = tok >= 0 ? src[c] : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(qd + r * 128 + ((c ^ (r & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      mbar_arrive(&ctl->q_ready);
    }
    float m_use = NO_SCORE, l = 0.f;
    bool stop = false;
    for (int j = 0; j < ntiles; ++j) {
      const int st = j & 1;
      const bool got = mbar_wait(&ctl->s_full[st], (j >> 1) & 1u, abort_flag);
      if (named_bar_or(1, SOFT, !got)) {
        *abort_flag = 1;
        stop = true;
        break;
      }
      tc_fence_after();
      const uint32_t sa = tmem + st * KT + gi * 64 + lane_off;
      const int kbase = j * KT + gi * 64;
      // pass 1: masked maximum of this half, then of the row
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(sa + c * 32, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (kbase + c * 32 + i <= pos) mx = fmaxf(mx, u32_as_f32(v[i]) * p.scale_log2);
      }
      ctl->xm[j & 1][gi][r] = mx;
      named_bar_sync(2, SOFT);
      mx = fmaxf(ctl->xm[j & 1][0][r], ctl->xm[j & 1][1][r]);
      float alpha = 1.f;
      if (mx > m_use + RESCALE_LOG2) {
        alpha = m_use == NO_SCORE ? 1.f : ex2(m_use - mx);
        l *= alpha;
        m_use = mx;
      }
      // pass 2: weights as bf16, their partial row sum
      uint32_t pk[32];
      float ls = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(sa + c * 32, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const int key = kbase + c * 32 + i;
          const float p0 = key <= pos ? ex2(u32_as_f32(v[i]) * p.scale_log2 - m_use) : 0.f;
          const float p1 = key + 1 <= pos ? ex2(u32_as_f32(v[i + 1]) * p.scale_log2 - m_use) : 0.f;
          const uint32_t w = pack_bf16x2(p0, p1);
          pk[(c * 32 + i) >> 1] = w;
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
          ls += f.x + f.y;
        }
      }
      tc_fence_before();
      mbar_arrive(&ctl->s_empty[st]);
      l += ls;
      if (j >= 1) {
        const bool okp = mbar_wait(&ctl->pv_done, (j - 1) & 1u, abort_flag);
        if (named_bar_or(1, SOFT, !okp)) {
          *abort_flag = 1;
          stop = true;
          break;
        }
        tc_fence_after();
        // rescale this half of O (warp-collective TMEM access; rows that keep their maximum multiply by 1)
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
          const uint32_t oa = tmem + 2 * KT + gi * 64 + lane_off;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tmem_ld32(oa + c * 32, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(u32_as_f32(v[i]) * alpha);
            tmem_st32(oa + c * 32, v);
          }
          tmem_wait_st();
        }
      }
      // P, this key half -> shared memory (A operand of PV, 128-byte swizzle)
      uint8_t* pd = sm + OFF_P + gi * HALF_B;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 v = make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
        *reinterpret_cast<uint4*>(pd + r * 128 + ((c ^ (r & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(&ctl->p_full);
    }
    if (!stop && ntiles > 0) {
      const bool okp = mbar_wait(&ctl->pv_done, (ntiles - 1) & 1u, abort_flag);
      if (named_bar_or(1, SOFT, !okp)) {
        *abort_flag = 1;
        stop = true;
      }
    }
    if (!stop) {                          // (a row without keys is zeros)
      tc_fence_after();
      ctl->xl[gi][r] = l;
      named_bar_sync(2, SOFT);
      const float lt = ctl->xl[0][r] + ctl->xl[1][r];
      const float inv = 1.f / lt;         // a row with keys and no weight (scores of -inf alone): 0 / 0
      const uint32_t oa = tmem + 2 * KT + gi * 64 + lane_off;
      __nv_bfloat16* orow = p.o + (static_cast<long long>(tok < 0 ? 0 : tok) * p.nq + head) * D + gi * 64;
      float sq = 0.f;
      int bad = -1;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(oa + c * 32, v);
        tmem_wait_ld();
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          w[i] = pos >= 0 ? pack_bf16x2(u32_as_f32(v[2 * i]) * inv, u32_as_f32(v[2 * i + 1]) * inv) : 0u;
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
          sq = fmaf(f.x, f.x, fmaf(f.y, f.y, sq));
        }
        if (tok >= 0) {
          uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 nv = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            if (p.check == nullptr) {
              dst[i] = nv;
            } else if (bad < 0) {
              const uint4 ov = dst[i];
              const uint32_t a[4] = {nv.x, nv.y, nv.z, nv.w}, b[4] = {ov.x, ov.y, ov.z, ov.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int dd = bf16x2_diff(a[e], b[e]);
                if (bad < 0 && dd >= 0) bad = gi * 64 + c * 32 + i * 8 + e * 2 + dd;
              }
            }
          }
        }
      }
      if (tok >= 0) {
        if (p.check != nullptr && bad >= 0)
          report_replay_mismatch(p.check, static_cast<unsigned long long>(tok) * p.nq * D + head * D + bad);
        if (p.check == nullptr && p.row_sq != nullptr) atomicAdd(p.row_sq + tok, sq);
      }
    }
    if (p.check != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && r == 0 && gi == 0) atomicAdd(p.check + 2, 1ull);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------- prefill, ping-pong
// Two query tiles at a time that share their key / value tiles (consecutive tiles of one request, so they attend to
// the same keys), so the tensor pipe always has one tile's MMAs to run while the other tile's softmax runs. A CTA goes
// through pairs until none is left: it takes over those of CTAs that have not started.
//   warps 0, 2  TMA: K and V pages of each 128-key tile into one of two stages (shared by both query tiles);
//   warp 1      MMA, in the order PV0(j-1), S0(j), PV1(j-1), S1(j) for key tile j: S_x = Q_x K_j^T into TMEM,
//               O_x += P_x V_{j-1} with P_x read from TMEM (the A operand of a tcgen05 MMA may live in tensor
//               memory), so P never goes through shared memory;
//   warp 3      the next pair: which it is, its rows' tokens and positions, its Q tiles by TMA;
//   warps 4-11  softmax of query tile 0, warps 12-19 of query tile 1: two threads per row, of warps w and w + 4, each
//               with half of the key tile: masked maximum (exchanged), conditional rescale of O (only when the
//               reference maximum moves by more than 2^8), P = exp2(S - max) rounded to bf16 and written back
//               over the last 64 columns of S_x, the row sum of those bf16 weights (in one order: the second thread
//               goes on from the first's sum while the MMAs run); at the end O / l,
//               zeros for a row without keys
// Bound by the chain of one tile: its softmax (2290 cycles a 128-key tile, 1600 of them the exponentials, which the two
// tiles share the unit for) and the MMAs behind it (1500), against 2048 cycles for the exponentials or the MMAs of both
// tiles alone. 8 x 2048 tokens, 16 / 8 heads: 162 us, 849 TFLOP/s, 0.50 of a dense bf16 product's rate; 32 x 1024 210 us,
// 16 x 512 43 us. A CTA for each pair took 182, 244 and 53 us: its start, first positions and Q took 10000 cycles. Pairs
// ordered by kv head first, then length: 176, 202, 47. Q through the load units instead of TMA (little of the L1 is left
// beside the shared memory, and a load in flight needs its lines): 190, 260, 57. One softmax thread a row: 193, 257, 54,
// and 37, 517 and 1 tokens behind 301, 0 and 1000 (32 / 8 heads) 26.8 against 23.1. The other way 200, 77 and 130 tokens
// behind 0, 40 and 16 (4 / 1), where there is one pair a CTA: 12.3 against 13.5.
// TMEM: S_0, S_1, O_0, O_1 (128 columns each). S_x(j + 1) overwrites P_x(j) only after PV_x(j) in the MMA order
// (tcgen05 MMAs of one thread run in issue order), and the commit that signals S_x(j) also covers PV_x(j - 1), so
// the softmax may rescale O_x as soon as it sees S_x(j). Every decision is per row and key tiles start at absolute
// multiples of 128, so rows are reproduced bit for bit whatever tile (or pair) they are computed in.
namespace pp {
constexpr int KT = 128;
constexpr int HALF_B = 128 * 128;
constexpr int TILE_B = 2 * HALF_B;
constexpr int OFF_Q = 0, OFF_K = 2 * TILE_B, OFF_V = 4 * TILE_B, OFF_CTL = 6 * TILE_B;
constexpr float RESCALE_LOG2 = 8.f;
constexpr int PG_BYTES = PAGE * D * 2;
// A pair of query tiles, as warp 3 makes it known to the others.
struct Pair {
  int live, bx, kvh, req;
  int nt[2];                                  // key tiles
  int maxpos;
  int tok[2][ROWS], pos[2][ROWS];             // a row's token and position, -1: none
};
struct Ctl {
  uint4 next;                                 // the hardware's answer: the next pair (16-byte aligned)
  uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_done[2], q_full[2], q_empty[2];   // per query tile
  uint64_t pair_full[2], pair_empty[2];
  uint64_t next_full, drain;
  uint32_t tmem_base;
  int abort_flag;
  Pair pair[2];                               // this pair and the next, in turn
  float part_max[2][2][ROWS];                 // [query tile][thread of the row]
  float sum[2][ROWS], sq[2][ROWS];            // passed from a row's first thread to its second
  float l[2][ROWS];                           // and back
  int begin[2][2][ROWS], stop[2][2][ROWS];    // whether waits ran out, at a pair's begin and behind its key tiles
  int bad[2][ROWS];                           // check mode: the first half's first difference
};
constexpr int SMEM = OFF_CTL + static_cast<int>(sizeof(Ctl)) + 1024;
constexpr int THREADS = 128 + 4 * ROWS;   // warpgroup 0: warps 0, 2 TMA, warp 1 TMEM + MMA; warpgroups 1-4: softmax
// (a, b) * s + d in one instruction, each rounded once.
__device__ __forceinline__ float2 fma2(uint32_t a, uint32_t b, float s, float d) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(a), "r"(b), "f"(s), "f"(d));
  return r;
}
// 32 bytes, a whole sector: in one store where the output lies on 32-byte boundaries (`wide`), else in two.
__device__ __forceinline__ void store32(void* p, const uint32_t* w, bool wide) {
  if (!wide) {
    uint4* q = static_cast<uint4*>(p);
    q[0] = make_uint4(w[0], w[1], w[2], w[3]);
    q[1] = make_uint4(w[4], w[5], w[6], w[7]);
    return;
  }
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The two warps that share 32 rows of query tile x (warps w and w + 4).
__device__ __forceinline__ void pair_sync(int x, int quarter) {
  asm volatile("bar.sync %0, 64;" ::"r"(1 + x * 4 + quarter) : "memory");
}
constexpr int P_COL = 64;                 // P_x lives in columns [64, 128) of S_x (bf16 pairs)
}  // namespace pp

// Work of CTAs that have not started yet can be taken over: the hardware cancels such a CTA and names its index.
__device__ __forceinline__ void request_next(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ bool next_index(const uint4* answer, int& x, int& y) {
  uint32_t got, a = 0, b = 0;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t.reg .b32 c;\n\t"
      "ld.shared.b128 h, [%3];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, c, _}, h;\n\t}\n"
      : "=r"(got), "+r"(a), "+r"(b)
      : "r"(smem_u32(answer))
      : "memory");
  x = static_cast<int>(a);
  y = static_cast<int>(b);
  return got != 0;
}
__global__ void __launch_bounds__(pp::THREADS, 1) prefill_pp_kernel(const __grid_constant__ CUtensorMap tm,
                                                                    const __grid_constant__ CUtensorMap tq,
                                                                    const __grid_constant__ CUtensorMap tq1,
                                                                    const __grid_constant__ CUtensorMap tr,
                                                                    const PrefillParams p) {
  pdl_trigger();
  using namespace pp;
  extern __shared__ uint8_t pp_raw[];
  uint8_t* sm = pp_raw + ((1024 - (smem_u32(pp_raw) & 1023)) & 1023);
  Ctl* ctl = reinterpret_cast<Ctl*>(sm + OFF_CTL);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.nq / p.nkv;
  const int tpc = ROWS / G;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->k_full[i], 1);
      mbar_init(&ctl->v_full[i], 1);
      mbar_init(&ctl->k_empty[i], 1);
      mbar_init(&ctl->v_empty[i], 1);
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->p_full[i], 2 * ROWS);
      mbar_init(&ctl->o_done[i], 1);
      mbar_init(&ctl->q_full[i], 1);
      mbar_init(&ctl->q_empty[i], 1);
      mbar_init(&ctl->pair_full[i], 1);
      mbar_init(&ctl->pair_empty[i], THREADS / 32 - 1);
    }
    mbar_init(&ctl->next_full, 1);
    mbar_init(&ctl->drain, 1);
    ctl->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tm);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  volatile int* abort_flag = &ctl->abort_flag;
  // Pair n of this CTA: null where a wait ran out (`live` is 0 behind the last pair).
  const auto pair_of = [&](int n) -> const Pair* {
    return mbar_wait(&ctl->pair_full[n & 1], (n >> 1) & 1, abort_flag) ? &ctl->pair[n & 1] : nullptr;
  };

  if (warp == 3) {
    // ------------------------------------------------------------ pairs: which, their rows, and Q
    // One pair ahead of the others, in the order in which the CTAs would have started.
    bool ok = true;
    int gx = blockIdx.x, gy = blockIdx.y, loads[2] = {0, 0};
    bool live = true;
    for (int n = 0;; ++n) {
      Pair& pr = ctl->pair[n & 1];
      // the launch order, kv heads fastest: the longest pairs of all heads come first
      const int at = gx + static_cast<int>(gridDim.x) * gy, bx = at / p.nkv, kvh = at % p.nkv;
      if (n >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&ctl->pair_empty[n & 1], ((n - 2) >> 1) & 1, abort_flag));
      if (!ok) break;
      int4 tl[2];
      int top = -1;
      if (live) {
        tl[0] = p.tiles[2 * bx];
        tl[1] = p.tiles[2 * bx + 1];
        const int req = tl[0].x;
        for (int x = 0; x < 2; ++x) {
          int tok[4], ps[4], mx = -1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ti = (lane + 32 * i) / G;
            tok[i] = -1;
            if (tl[x].x == req && ti < tl[x].z && ti < tpc) tok[i] = tl[x].w >= 0 ? p.row_idx[tl[x].w + ti] : tl[x].y + ti;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) ps[i] = tok[i] >= 0 ? p.pos[tok[i]] : -1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (ps[i] >= p.limit || ps[i] < 0) ps[i] = -1;
            mx = max(mx, ps[i]);
            pr.tok[x][lane + 32 * i] = tok[i];
            pr.pos[x][lane + 32 * i] = ps[i];
          }
          mx = __reduce_max_sync(0xffffffffu, mx);
          if (lane == 0) pr.nt[x] = mx >= 0 ? mx / KT + 1 : 0;
          top = max(top, mx);
        }
      }
      if (lane == 0) {
        pr.live = live;
        pr.bx = bx;
        pr.kvh = kvh;
        pr.req = live ? tl[0].x : 0;
        pr.maxpos = top;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->pair_full[n & 1]);
      if (!live) break;
      // Q_x once S_x of the pair before is formed. A whole tile of consecutive tokens is one box (G heads of each token) for
      // each half of the dims, else every token has its own; rows without a token keep what was there (they are masked).
      for (int x = 0; x < 2; ++x) {
        if (n >= 1) ok = __all_sync(0xffffffffu, mbar_wait(&ctl->q_empty[x], (n - 1) & 1, abort_flag));
        if (!ok) break;
        const int count = tl[x].x == tl[0].x ? max(0, min(tl[x].z, tpc)) : 0;
        uint8_t* qd = sm + OFF_Q + x * TILE_B;
        if (lane == 0) {
          if (count > 0) mbar_arrive_expect_tx(&ctl->q_full[x], count * G * D * 2);
          else mbar_arrive(&ctl->q_full[x]);
        }
        __syncwarp();
        loads[x] = n + 1;
        if (count == tpc && tl[x].w < 0) {
          if (lane < 2) tma_load_3d(qd + lane * HALF_B, &tq, &ctl->q_full[x], lane * 64, kvh * G, tl[x].y);
        } else {
          for (int i = lane; i < 2 * count; i += 32)
            tma_load_3d(qd + (i & 1) * HALF_B + (i >> 1) * G * 128, &tq1, &ctl->q_full[x], (i & 1) * 64, kvh * G,
                        pr.tok[x][(i >> 1) * G]);
        }
      }
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&ctl->next_full, 16);
        request_next(&ctl->next, &ctl->next_full);
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, mbar_wait(&ctl->next_full, n & 1, nullptr));
      if (!ok) break;
      live = next_index(&ctl->next, gx, gy);
      fence_proxy_async_smem();
      __syncwarp();
    }
    if (!ok && lane == 0) *abort_flag = 1;
    // what is on its way has to land before the CTA ends
    for (int x = 0; x < 2; ++x)
      if (loads[x] > 0) mbar_wait(&ctl->q_full[x], (loads[x] - 1) & 1, nullptr);
  } else if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------ TMA producers (all 32 lanes issue): warp 0 K, warp 2 V
    // K's stage is free once S of both query tiles is formed, a softmax and a product before V's: taken apart, the next
    // K is on its way that much earlier (with one barrier for both, the MMAs waited for K in half of the time)
    pdl_wait();                           // the pages may come from the kernel before (launched with overlap)
    const int kv = warp >> 1;
    uint64_t* full = kv ? ctl->v_full : ctl->k_full;
    uint64_t* empty = kv ? ctl->v_empty : ctl->k_empty;
    bool ok = true;
    int kt = 0;                           // key tiles so far, over all pairs
    for (int n = 0; ok; ++n) {
      const Pair* pr = pair_of(n);
      ok = __all_sync(0xffffffffu, pr != nullptr);
      if (!ok || !pr->live) break;
      const int ntiles = max(pr->nt[0], pr->nt[1]), maxpos = pr->maxpos, kvh = pr->kvh;
      const int* bt = p.block_table + static_cast<long long>(pr->req) * p.max_pages;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->pair_empty[n & 1]);
      for (int j = 0; j < ntiles; ++j, ++kt) {
        const int st = kt & 1;
        bool got = true;
        if (lane == 0) got = mbar_wait(&empty[st], ((kt >> 1) & 1u) ^ 1u, abort_flag);
        if (!__shfl_sync(0xffffffffu, got ? 1 : 0, 0)) {
          ok = false;
          break;
        }
        // whole pages of K (masked scores are not used), of V the keys alone
        const int nkeys = min(KT, maxpos + 1 - j * KT), npg = kv ? nkeys / PAGE : (nkeys + PAGE - 1) / PAGE;
        uint8_t* buf = sm + (kv ? OFF_V : OFF_K) + st * TILE_B;
        if (kv && nkeys < KT) clear_v(buf, nkeys, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&full[st], kv ? nkeys * (PG_BYTES / PAGE) : npg * PG_BYTES);
        __syncwarp();
        const auto row_of = [&](int pg) {
          return static_cast<int>(((static_cast<long long>(bt[j * (KT / PAGE) + pg]) * 2 + kv) * p.nkv + kvh) * PAGE);
        };
        if (lane < 2 * npg) {
          const int pg = lane >> 1, half = lane & 1;
          tma_load_2d(buf + half * HALF_B + pg * PAGE * 128, &tm, &full[st], half * 64, row_of(pg));
        }
        if (kv && nkeys % PAGE) load_v_rest(buf, &tr, &full[st], row_of(npg), nkeys, lane);
      }
    }
    if (!ok) {
      if (lane == 0) *abort_flag = 1;
      for (int j = kt > 1 ? kt - 2 : 0; j < kt; ++j) mbar_wait(&full[j & 1], (j >> 1) & 1u, nullptr);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      bool ok = true;
      const uint32_t idesc_s = idesc_bf16_f32(128, KT);
      const uint32_t idesc_o = idesc_bf16_f32(128, D) | (1u << 16);     // B (V) MN-major
      int kt = 0, turn[2] = {0, 0};       // key tiles before this pair, turns of P_x so far
      for (int n = 0; ok; ++n) {
        const Pair* pr = pair_of(n);
        ok = pr != nullptr;
        if (!ok || !pr->live) break;
        const int nt[2] = {pr->nt[0], pr->nt[1]};
        const int ntiles = max(nt[0], nt[1]);
        mbar_arrive(&ctl->pair_empty[n & 1]);
        for (int x = 0; x < 2 && ok; ++x) {
          ok = mbar_wait(&ctl->q_full[x], n & 1, abort_flag);
          if (ok && nt[x] == 0) mbar_arrive(&ctl->q_empty[x]);
        }
        for (int j = 0; j <= ntiles && ntiles > 0 && ok; ++j) {
          const int now = kt + j, was = kt + j - 1;
          if (j < ntiles) ok = mbar_wait(&ctl->k_full[now & 1], (now >> 1) & 1u, abort_flag);
          if (ok && j >= 1) ok = mbar_wait(&ctl->v_full[was & 1], (was >> 1) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          for (int x = 0; x < 2 && ok; ++x) {
            const uint32_t s_col = tmem + x * KT, o_col = tmem + 2 * KT + x * D;
            if (j >= 1 && j - 1 < nt[x]) {
              // O_x += P_x(j-1) V(j-1): P_x in columns [64, 128) of S_x (bf16 pairs), 8 columns per K = 16 step
              ok = mbar_wait(&ctl->p_full[x], turn[x]++ & 1u, abort_flag);
              if (!ok) break;
              tc_fence_after();
              const uint32_t va = smem_u32(sm + OFF_V + (was & 1) * TILE_B);
#pragma unroll
              for (int ks = 0; ks < KT / 16; ++ks) {
                const uint64_t bd = umma_desc_sw128_mn(va + ks * 2048, HALF_B, 1024);
                umma_f16_tmem_a(o_col, s_col + P_COL + ks * 8, bd, idesc_o, (j - 1 > 0 || ks > 0) ? 1u : 0u);
              }
              if (j - 1 == nt[x] - 1) umma_commit(&ctl->o_done[x]);
            }
            if (j < nt[x]) {
              const uint32_t qa = smem_u32(sm + OFF_Q + x * TILE_B);
              const uint32_t ka = smem_u32(sm + OFF_K + (now & 1) * TILE_B);
#pragma unroll
              for (int ks = 0; ks < D / 16; ++ks) {
                const uint32_t off = (ks >> 2) * HALF_B + (ks & 3) * 32;
                umma_f16(s_col, umma_desc_sw128(qa + off), umma_desc_sw128(ka + off), idesc_s, ks ? 1u : 0u);
              }
              umma_commit(&ctl->s_full[x]);
              if (j == nt[x] - 1) umma_commit(&ctl->q_empty[x]);
            }
          }
          if (ok && j < ntiles) umma_commit(&ctl->k_empty[now & 1]);
          if (ok && j >= 1) umma_commit(&ctl->v_empty[was & 1]);
        }
        kt += ntiles;
      }
      if (!ok) {
        record_error(nullptr, ERR_TIMEOUT_MMA);
        *abort_flag = 1;
        umma_commit(&ctl->drain);
        mbar_wait(&ctl->drain, 0, nullptr);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax / output: two threads a row of tile x
    // part 0: keys [64, 128) of each key tile and dims [0, 64) of O; part 1: keys [0, 64), dims [64, 128). Both threads
    // of a row go through every pair_sync, whatever fails: a wait that ran out sets the abort flag and goes on.
    const int x = (warp - 4) >> 3, part = ((warp >> 2) & 1) ^ 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_col = tmem + x * KT + lane_off, o_col = tmem + 2 * KT + x * D + lane_off;
    const int key0 = (1 - part) * 64;
    const bool wide = (reinterpret_cast<uintptr_t>(p.o) & 31) == 0;
    int turn = 0, outs = 0;               // turns of S_x and O_x so far
    for (int n = 0;; ++n) {
      const Pair* pr = pair_of(n);
      bool stop = pr == nullptr;
      if (stop) *abort_flag = 1;
      // both warps give up, or neither
      ctl->begin[x][part][r] = stop;
      pair_sync(x, quarter);
      if (__any_sync(0xffffffffu, stop || ctl->begin[x][part ^ 1][r])) break;
      pr = &ctl->pair[n & 1];
      if (!pr->live) break;
      const int pos = pr->pos[x][r], my_tiles = pr->nt[x];
      float m_use = NO_SCORE, l = 0.f;    // l: part 1's
      for (int j = 0; j < my_tiles; ++j) {
        if (!mbar_wait(&ctl->s_full[x], turn++ & 1u, abort_flag)) {
          *abort_flag = 1;
          stop = true;
        }
        __syncwarp();
        tc_fence_after();
        // This half of the S row, and the maximum over both. P (bf16 pairs) goes to columns [64, 128): the weights of keys
        // [64, 128) over columns [96, 128) and those of keys [0, 64) over [64, 96), written after part 0 read the S
        // values under them (pair_sync).
        const int lim = pos - j * KT - key0;      // keys [0, lim] of this half are visible to the row
        // every key visible to every row of the warp (all but a prompt's last tiles): no masks, the same values
        const bool full = __all_sync(0xffffffffu, lim >= 63);
        uint32_t v[2][32];
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // (a maximum does not depend on the order)
        tmem_ld32(s_col + key0, v[0]);
        tmem_ld32(s_col + key0 + 32, v[1]);
        tmem_wait_ld();
        if (full) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], u32_as_f32(v[c][i]), u32_as_f32(v[c][i + 1]));
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i <= lim) mx4[i & 3] = fmaxf(mx4[i & 3], u32_as_f32(v[c][i]));
        }
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        ctl->part_max[x][part][r] = mx;
        tc_fence_before();
        pair_sync(x, quarter);
        tc_fence_after();
        mx = fmaxf(mx, ctl->part_max[x][part ^ 1][r]);
        mx *= p.scale_log2;                // scale > 0: the maximum commutes with it
        float alpha = 1.f;
        if (mx > m_use + RESCALE_LOG2) {
          alpha = m_use == NO_SCORE ? 1.f : ex2(m_use - mx);
          l *= alpha;
          m_use = mx;
        }
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
          // PV_x(j-1) is complete (the commit of S_x(j) covers it): rescale this half of the row of O_x
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t o[16];
            tmem_ld16(o_col + part * 64 + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(u32_as_f32(o[i]) * alpha);
            tmem_st16(o_col + part * 64 + c * 16, o);
          }
        }
        uint32_t pk[2][16];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (full) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 e = fma2(v[c][i], v[c][i + 1], p.scale_log2, -m_use);
              pk[c][i >> 1] = pack_bf16x2(ex2(e.x), ex2(e.y));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const int key = c * 32 + i;
              const float p0 = key <= lim ? ex2(u32_as_f32(v[c][i]) * p.scale_log2 - m_use) : 0.f;
              const float p1 = key + 1 <= lim ? ex2(u32_as_f32(v[c][i + 1]) * p.scale_log2 - m_use) : 0.f;
              pk[c][i >> 1] = pack_bf16x2(p0, p1);
            }
          }
          tmem_st16(s_col + P_COL + (1 - part) * 32 + c * 16, pk[c]);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->p_full[x]);
        // the row's sum over keys [64, 128), then [0, 64), one order whoever holds them
        const auto add = [&](float s) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) s += u32_as_f32(pk[c][i] << 16) + u32_as_f32(pk[c][i] & 0xffff0000u);
          return s;
        };
        if (part == 0) ctl->sum[x][r] = add(0.f);
        pair_sync(x, quarter);
        if (part == 1) l += add(ctl->sum[x][r]);
      }
      if (my_tiles > 0 && !mbar_wait(&ctl->o_done[x], outs++ & 1u, abort_flag)) {
        *abort_flag = 1;
        stop = true;
      }
      ctl->stop[x][part][r] = stop;
      if (part == 1) ctl->l[x][r] = l;
      pair_sync(x, quarter);
      stop = __any_sync(0xffffffffu, stop || ctl->stop[x][part ^ 1][r]);
      const int bx = pr->bx, kvh = pr->kvh, tok = pr->tok[x][r];
      // a row without keys is zeros, whether or not others of its tile have some
      if (!stop && __any_sync(0xffffffffu, tok >= 0)) {
        const int head = kvh * G + (r % G);
        tc_fence_after();
        l = ctl->l[x][r];
        const float inv = 1.f / l;        // a row with keys and no weight (scores of -inf alone): 0 / 0
        __nv_bfloat16* orow = p.o + (static_cast<long long>(tok < 0 ? 0 : tok) * p.nq + head) * D;
        int bad = -1;
        uint32_t w[2][16];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[32];
          tmem_ld32(o_col + part * 64 + c * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) w[c][i] = pack_bf16x2(u32_as_f32(v[2 * i]) * inv, u32_as_f32(v[2 * i + 1]) * inv);
          if (pos < 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[c][i] = 0u;
          }
          if (p.check == nullptr) {
            if (tok >= 0) {
              store32(orow + part * 64 + c * 32, &w[c][0], wide);
              store32(orow + part * 64 + c * 32 + 16, &w[c][8], wide);
            }
          } else if (tok >= 0) {
            uint4* dst = reinterpret_cast<uint4*>(orow + part * 64 + c * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 nv = make_uint4(w[c][4 * i], w[c][4 * i + 1], w[c][4 * i + 2], w[c][4 * i + 3]);
              if (bad < 0) {
                const uint4 ov = dst[i];
                const uint32_t a[4] = {nv.x, nv.y, nv.z, nv.w}, b[4] = {ov.x, ov.y, ov.z, ov.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int dd = bf16x2_diff(a[e], b[e]);
                  if (bad < 0 && dd >= 0) bad = part * 64 + c * 32 + i * 8 + e * 2 + dd;
                }
              }
            }
          }
        }
        const auto squares = [&](float sq) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[c][i]));
              sq = fmaf(f.x, f.x, fmaf(f.y, f.y, sq));
            }
          return sq;
        };
        if (p.check != nullptr || p.row_sq != nullptr) {
          if (part == 0) {
            ctl->sq[x][r] = squares(0.f);
            ctl->bad[x][r] = bad;
          }
          pair_sync(x, quarter);
          if (tok >= 0) {
            if (p.check != nullptr && bad >= 0 && (part == 0 || ctl->bad[x][r] < 0))      // the row's first difference
              report_replay_mismatch(p.check, static_cast<unsigned long long>(tok) * p.nq * D + head * D + bad);
            if (part == 1 && p.check == nullptr) atomicAdd(p.row_sq + tok, squares(ctl->sq[x][r]));
          }
        }
      }
      if (p.check != nullptr && bx == 0 && kvh == 0 && r == 0 && x == 0 && part == 0) atomicAdd(p.check + 2, 1ull);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->pair_empty[n & 1]);
      if (stop) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------- decode
// Split-KV decode ("flash decoding"): the keys of each (sequence, kv head) are cut into chunks of SPLIT keys at
// absolute multiples of SPLIT, and the chunks into segments of SEG chunks. One CTA takes a whole segment: it
// merges the segment's chunks in order with the running-maximum softmax and writes one record (the segment's
// softmax statistics and unnormalised output); a combine kernel merges the segments of a row in a fixed order.
// Chunk and segment boundaries and every reduction order depend only on the row, so a replay of any subset of
// sequences reproduces their outputs bit for bit. (One record per segment instead of one per chunk cuts the
// record traffic of both kernels by SEG.)
//
// Memory path: decode reads every K and V byte of the context once, so the kernel is bound by HBM. A CTA owns
// one (sequence, kv head) and every gridDim.z-th chunk of it; TMA copies each chunk's pages (one 16-row x
// 128-byte box per page, half head dim and K or V, with the 128-byte swizzle) into one of two buffers, so the
// copies of the next chunk are in flight while the current chunk is computed. The sequence's block-table row
// is read once into shared memory.
// Arithmetic on tensor cores (mma.m16n8k16, bf16 in, fp32 accumulate): the G query heads of the kv head are
// the rows of the A operand (rows G..15 are zero); each warp takes 16 keys of the chunk: S = Q K^T from
// swizzle-conflict-free ldmatrix loads of K, the chunk's softmax statistics across the four warps through
// shared memory, then O_w = P V with P kept in registers as the A operand. The chunk record is the sum of the
// four warps' O in a fixed order, so it depends only on the chunk, not on which CTA computed it.
constexpr int SPLIT = 64;                  // keys per chunk (4 pages)
constexpr int SEG = 4;                     // chunks per segment (one partial record each)
constexpr int SEG_KEYS = SPLIT * SEG;
constexpr int REC = D + 4;                 // floats per partial record: o[D], m, l, pad
constexpr int PAGE_BYTES = PAGE * D * 2;   // 4 KB: one page of K (or V) of one kv head

struct DecodeParams {
  const __nv_bfloat16* q;     // [B, nq, D] (one new token per sequence)
  __nv_bfloat16* o;           // [B, nq, D]
  const __nv_bfloat16* cache;
  const int* block_table;     // [R, max_pages]
  int max_pages;
  const int* seq_req;         // [B] request (block-table row) of each sequence
  const int* ctx;             // [B] keys to attend (including the new token)
  const int* seq_idx;         // optional list of sequences to run (replay); null = all
  int nq, nkv;
  int max_splits;             // segments per sequence the partial buffer holds
  float scale_log2;
  float* part;                // [B][nkv][max_splits][G][REC] scratch
  float* row_sq;
  int* err;                   // error word (bounded waits), or null
  unsigned long long* check;  // check mode (replay): compare with o instead of writing (state row), or null
};

constexpr int MAX_BT = 512;                // block-table entries staged per sequence (8192 tokens)
constexpr int HALF_BYTES = SPLIT * 128;    // one half (64 dims) of the chunk's K or V rows: 8 KB

template <int G>
struct DecodeSmem {
  uint8_t k[2][2 * HALF_BYTES];         // [buffer][half][key][128 B, swizzled]; reused for per-warp O partials
  uint8_t v[2][2 * HALF_BYTES];
  float red[4][8];                      // per-warp row maxima
  float red2[4][8];                     // per-warp row sums (of the segment, at its end)
  float segm[8];                        // row maxima of the segment, at its end
  int bt[MAX_BT];
  uint64_t bar[2][2];                   // [buffer][K, V]
};

// byte offset of 16-byte chunk j (0..15 over the head dim) of row `key` in a [half][key][128 B] swizzled buffer
__device__ __forceinline__ uint32_t kv_off(int key, int j) {
  return static_cast<uint32_t>((j >> 3) * HALF_BYTES + key * 128 + (((j & 7) ^ (key & 7)) << 4));
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* gsrc, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(smem_dst)),
               "l"(gsrc), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void bf8_to_f32(const uint4& u, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = __bfloat1622float2(h[j]);
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
  }
}

template <int G>
__device__ __forceinline__ void decode_issue(DecodeSmem<G>& sm, const CUtensorMap* tm, const DecodeParams& p, int buf,
                                             int sp, int n, int kvh, int lane) {
  const int k0 = sp * SPLIT;
  const int npages = (min(SPLIT, n - k0) + PAGE - 1) / PAGE;
  if (lane == 0) {
    mbar_arrive_expect_tx(&sm.bar[buf][0], npages * PAGE_BYTES);
    mbar_arrive_expect_tx(&sm.bar[buf][1], npages * PAGE_BYTES);
  }
  __syncwarp();
  if (lane < 4 * npages) {            // lane -> (page, K/V, half)
    const int pg = lane % npages, w = lane / npages, kv = w >> 1, half = w & 1;
    const long long blk = sm.bt[k0 / PAGE + pg];
    const int row = static_cast<int>(((blk * 2 + kv) * p.nkv + kvh) * PAGE);
    uint8_t* dst = (kv ? sm.v[buf] : sm.k[buf]) + half * HALF_BYTES + pg * PAGE * 128;
    tma_load_2d(dst, tm, &sm.bar[buf][kv], half * 64, row);
  }
}

// Merges the segments of each (sequence, kv head) in segment order; one CTA of 128 threads. The segment maxima
// and weights are computed in parallel over segments, then thread d sums dimension d over them in order.
constexpr int MAX_SPLITS = MAX_BT * PAGE / SEG_KEYS;

template <int G>
__device__ __forceinline__ void combine_row(const DecodeParams& p, int b, int kvh) {
  __shared__ float wsh[G][MAX_SPLITS];
  __shared__ float Lsh[G];
  __shared__ float msh[4][G];
  const int d = threadIdx.x, lane = d & 31, warp = d >> 5;
  const int n = p.ctx[b];
  const int ns = (n + SEG_KEYS - 1) / SEG_KEYS;
  const float* base = p.part + (static_cast<long long>(b) * p.nkv + kvh) * p.max_splits * G * REC;
  float m[G];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    float v = -INFINITY;
    for (int s = d; s < ns; s += 128) v = fmaxf(v, base[(s * G + h) * REC + D]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, k));
    if (lane == 0) msh[warp][h] = v;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < G; ++h) {
    m[h] = fmaxf(fmaxf(msh[0][h], msh[1][h]), fmaxf(msh[2][h], msh[3][h]));
    for (int s = d; s < ns; s += 128) wsh[h][s] = ex2(base[(s * G + h) * REC + D] - m[h]);
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float l = 0.f;
      for (int s = lane; s < ns; s += 32) l = fmaf(base[(s * G + h) * REC + D + 1], wsh[h][s], l);
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
      if (lane == 0) Lsh[h] = l;
    }
  }
  __syncthreads();
  float sqsum = 0.f;
#pragma unroll
  for (int h = 0; h < G; ++h) {
    float acc = 0.f;
    const float* r = base + h * REC + d;
#pragma unroll 8
    for (int s = 0; s < ns; ++s) acc = fmaf(r[s * G * REC], wsh[h][s], acc);
    const __nv_bfloat16 ob = __float2bfloat16(acc / Lsh[h]);
    __nv_bfloat16* dst = p.o + (static_cast<long long>(b) * p.nq + kvh * G + h) * D + d;
    if (p.check == nullptr) {
      *dst = ob;
    } else {
      const float x = __bfloat162float(ob), y = __bfloat162float(*dst);
      if (!(x == y) && !(x != x && y != y))
        report_replay_mismatch(p.check, static_cast<unsigned long long>(b) * p.nq * D + (kvh * G + h) * D + d);
    }
    const float f = __bfloat162float(ob);
    sqsum = fmaf(f, f, sqsum);
  }
  if (p.check != nullptr) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && d == 0) atomicAdd(p.check + 2, 1ull);
    return;
  }
  if (p.row_sq != nullptr) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sqsum += __shfl_xor_sync(0xffffffffu, sqsum, m);
    if (lane == 0) atomicAdd(p.row_sq + b, sqsum);
  }
}

template <int G>
__global__ void __launch_bounds__(128) decode_split_kernel(const __grid_constant__ CUtensorMap tm, const DecodeParams p) {
  pdl_trigger();   // a dependent GEMM may start its prologue and weight loads now
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  // the swizzled buffers need 1024-byte alignment
  unsigned char* base = dsm_raw + ((1024 - (smem_u32(dsm_raw) & 1023)) & 1023);
  DecodeSmem<G>& sm = *reinterpret_cast<DecodeSmem<G>*>(base);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;          // mma fragment row (head) and column pair
  const int b = p.seq_idx ? p.seq_idx[blockIdx.x] : blockIdx.x;
  const int kvh = blockIdx.y;
  const int n = p.ctx[b];
  if (static_cast<int>(blockIdx.z) * SEG_KEYS >= n) return;
  if (tid == 0) {
    tma_prefetch_desc(&tm);
    mbar_init(&sm.bar[0][0], 1);
    mbar_init(&sm.bar[0][1], 1);
    mbar_init(&sm.bar[1][0], 1);
    mbar_init(&sm.bar[1][1], 1);
    fence_mbar_init();
  }
  const int npg_all = min((n + PAGE - 1) / PAGE, MAX_BT);
  const int* btrow = p.block_table + static_cast<long long>(p.seq_req[b]) * p.max_pages;
  for (int i = tid; i < npg_all; i += 128) sm.bt[i] = btrow[i];
  // Q as mma A fragments (rows = heads of this kv head, zero beyond G): a0 = (g, 16 ks + 2t), a2 = (g, +8)
  uint32_t qa[8][2];
  {
    const __nv_bfloat16* qrow = p.q + (static_cast<long long>(b) * p.nq + kvh * G + g) * D;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      qa[ks][0] = g < G ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 2 * t) : 0u;
      qa[ks][1] = g < G ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8 + 2 * t) : 0u;
    }
  }
  __syncthreads();
  if (warp == 0) decode_issue(sm, &tm, p, 0, static_cast<int>(blockIdx.z) * SEG, n, kvh, lane);
  bool ok = true;
  const int mi = lane >> 3, rr = lane & 7;        // ldmatrix: matrix index and row of this lane's address
  int it = 0;
  // running statistics of the current segment (row g of this warp's fragments): max (common to the four warps),
  // this warp's weight sum, this warp's unnormalised output
  float m_run = -INFINITY, l_run = 0.f;
  float o[16][4];
#pragma unroll
  for (int dt = 0; dt < 16; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[dt][e] = 0.f;
  for (int sp = static_cast<int>(blockIdx.z) * SEG; sp * SPLIT < n; ++it) {
    const int buf = it & 1;
    const uint32_t par = (it >> 1) & 1;
    const bool seg_end = (sp + 1) % SEG == 0 || (sp + 1) * SPLIT >= n;
    // the next chunk of this CTA: the next one of the segment, or the first of its next segment
    const int nsp = (sp + 1) % SEG != 0 ? sp + 1 : sp + 1 + (static_cast<int>(gridDim.z) - 1) * SEG;
    if (warp == 0 && nsp * SPLIT < n) decode_issue(sm, &tm, p, buf ^ 1, nsp, n, kvh, lane);   // next chunk
    const int nk = min(SPLIT, n - sp * SPLIT);
    ok = mbar_wait(&sm.bar[buf][0], par, nullptr) && ok;
    // S = Q K^T for keys [16 warp, 16 warp + 16): two n-tiles of 8 keys
    float sc[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = 0.f;
    {
      const uint32_t kb = smem_u32(sm.k[buf]);
      const int key = warp * 16 + (mi >> 1) * 8 + rr;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(kb + kv_off(key, 2 * ks + (mi & 1)), b0, b1, b2, b3);
        mma_bf16(sc[0], qa[ks][0], 0u, qa[ks][1], 0u, b0, b1);
        mma_bf16(sc[1], qa[ks][0], 0u, qa[ks][1], 0u, b2, b3);
      }
    }
    // scores of row g: keys 16 warp + 8 nt + 2 t + e (e = 0, 1); rows g + 8 are padding
    float x[2][2];
    float mx = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int kk = warp * 16 + nt * 8 + 2 * t + e;
        x[nt][e] = (kk < nk && g < G) ? sc[nt][e] * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, x[nt][e]);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (t == 0) sm.red[warp][g] = mx;
    __syncthreads();      // (A) red[] complete; every warp is done reading k[buf]
    const float Mc = fmaxf(fmaxf(sm.red[0][g], sm.red[1][g]), fmaxf(sm.red[2][g], sm.red[3][g]));
    const float M = fmaxf(m_run, Mc);
    const float alpha = m_run == -INFINITY ? 0.f : ex2(m_run - M);   // rescales the segment so far
    m_run = M;
    uint32_t pa[2];
    float lsum = 0.f;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const float p0 = x[nt][0] == -INFINITY ? 0.f : ex2(x[nt][0] - M);
      const float p1 = x[nt][1] == -INFINITY ? 0.f : ex2(x[nt][1] - M);
      pa[nt] = pack_bf16x2(p0, p1);
      const float2 r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&pa[nt]));
      lsum += r.x + r.y;                    // the row sum of the weights the MMA uses
    }
    lsum += __shfl_xor_sync(0xffffffffu, lsum, 1);
    lsum += __shfl_xor_sync(0xffffffffu, lsum, 2);
    l_run = fmaf(l_run, alpha, lsum);
    ok = mbar_wait(&sm.bar[buf][1], par, nullptr) && ok;
    if (nk < SPLIT) {
      // the last chunk of the sequence: V behind its end has weights of zero, but what its last page holds there, or the
      // shared memory of pages that were not loaded, may be NaN; clear it
      for (int i = tid; i < (SPLIT - nk) * 16; i += 128) {
        const int r = nk + (i >> 4), c = i & 15;
        *reinterpret_cast<uint4*>(sm.v[buf] + (c >> 3) * HALF_BYTES + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
    }
    // O_w = alpha O_w + P V: 16 n-tiles of 8 dims
#pragma unroll
    for (int dt = 0; dt < 16; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[dt][e] *= alpha;
    {
      const uint32_t vb = smem_u32(sm.v[buf]);
      const int key = warp * 16 + (mi & 1) * 8 + rr;
#pragma unroll
      for (int pr = 0; pr < 8; ++pr) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(vb + kv_off(key, 2 * pr + (mi >> 1)), b0, b1, b2, b3);
        mma_bf16(o[2 * pr], pa[0], 0u, pa[1], 0u, b0, b1);
        mma_bf16(o[2 * pr + 1], pa[0], 0u, pa[1], 0u, b2, b3);
      }
    }
    if (seg_end) {
      // per-warp partials (rows < G) go where this chunk's K was (no warp reads k[buf] after barrier A)
      float* wpart = reinterpret_cast<float*>(sm.k[buf]);     // [4][G][D]
      if (g < G) {
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
          *reinterpret_cast<float2*>(wpart + (warp * G + g) * D + dt * 8 + 2 * t) = make_float2(o[dt][0], o[dt][1]);
        if (t == 0) {
          sm.red2[warp][g] = l_run;
          if (warp == 0) sm.segm[g] = m_run;
        }
      }
      __syncthreads();      // (C) wpart, red2[] and segm[] complete
      float* rec = p.part + ((static_cast<long long>(b) * p.nkv + kvh) * p.max_splits + sp / SEG) * G * REC;
      for (int i = tid; i < G * D; i += 128) {
        const int h = i / D, d = i % D;
        rec[h * REC + d] = (wpart[(0 * G + h) * D + d] + wpart[(1 * G + h) * D + d]) +
                           (wpart[(2 * G + h) * D + d] + wpart[(3 * G + h) * D + d]);
      }
      if (tid < G) {
        rec[tid * REC + D] = sm.segm[tid];
        rec[tid * REC + D + 1] = (sm.red2[0][tid] + sm.red2[1][tid]) + (sm.red2[2][tid] + sm.red2[3][tid]);
      }
      m_run = -INFINITY;
      l_run = 0.f;
#pragma unroll
      for (int dt = 0; dt < 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][e] = 0.f;
    }
    fence_proxy_async_smem();   // this buffer's generic writes (partials, cleared rows) before its next TMA fill
    __syncthreads();      // (D) buffer buf and red[], red2[], segm[] free for later chunks
    sp = nsp;
  }
  if (!ok && tid == 0) record_error(p.err, ERR_TIMEOUT_PEER);
  if (gridDim.z == 1) {   // this CTA wrote every segment of the row: merge them here, no combine launch
    __syncthreads();
    combine_row<G>(p, b, kvh);
  }
}



// The merge of one (sequence b, kv head) by the 128 threads of a CTA (the combine kernel, or the split kernel
// itself when one CTA held every segment of the row): the same arithmetic either way, so replays stay exact.
template <int G>
__global__ void __launch_bounds__(128) decode_combine_kernel(const DecodeParams p) {
  pdl_trigger();   // a dependent GEMM may start its prologue and weight loads now
  combine_row<G>(p, p.seq_idx ? p.seq_idx[blockIdx.x] : blockIdx.x, blockIdx.y);
}

}  // namespace attn
}  // namespace sdc

using namespace sdc::attn;

template <int G>
static int launch_decode(const DecodeParams& p, const CUtensorMap& tm, dim3 grid, dim3 grid2, cudaStream_t st) {
  static bool attr_set = false;      // per process; the attribute applies to every device
  const int smem = static_cast<int>(sizeof(DecodeSmem<G>)) + 1024;   // + room to align the buffers to 1 KB
  if (!attr_set) {
    cudaError_t e = cudaFuncSetAttribute(decode_split_kernel<G>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    attr_set = true;
  }
  decode_split_kernel<G><<<grid, 128, smem, st>>>(tm, p);
  if (grid.z > 1) decode_combine_kernel<G><<<grid2, 128, 0, st>>>(p);   // z == 1: merged by the split kernel
  return static_cast<int>(cudaGetLastError());
}

static int launch_prefill(const void* q, void* o, const void* cache, long long num_blocks, const int* block_table,
                          int max_pages, const int* pos, int limit, const void* tiles, int ntiles, const int* row_idx,
                          int nq, int nkv, int head_dim, float scale, void* row_sq, void* check, bool overlap,
                          cudaStream_t stream) {
  if (ntiles <= 0) return 0;
  if (head_dim != D || nq % nkv || (ROWS % (nq / nkv))) return -1;
  PrefillParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.o = static_cast<__nv_bfloat16*>(o);
  p.cache = static_cast<const __nv_bfloat16*>(cache);
  p.block_table = block_table;
  p.max_pages = max_pages;
  p.pos = pos;
  p.limit = limit;
  p.tiles = static_cast<const int4*>(tiles);
  p.row_idx = row_idx;
  p.nq = nq;
  p.nkv = nkv;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.row_sq = static_cast<float*>(row_sq);
  p.check = static_cast<unsigned long long*>(check);
  if (p.check != nullptr && row_idx == nullptr) return -1;
  CUtensorMap tm, tr;
  if (!make_map_bf16_sw128(&tm, cache, num_blocks * 2 * nkv * PAGE, D, D, 64, PAGE) ||
      !make_map_bf16_sw128(&tr, cache, num_blocks * 2 * nkv * PAGE, D, D, 64, 1))
    return -2;
  // Q by token: the tiles say which tokens there are
  CUtensorMap tq, tq1;
  const int G = nq / nkv;
  if (!make_map3_bf16_sw128(&tq, q, 1ll << 31, nq, D, 64, G, ROWS / G) ||
      !make_map3_bf16_sw128(&tq1, q, 1ll << 31, nq, D, 64, G, 1))
    return -2;
  // the attributes belong to a device; one bit for each that has them (setting them twice does no harm)
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev > 63 || !(ready.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(prefill_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pf::SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(prefill_pp_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pp::SMEM);
    if (e == cudaSuccess && dev <= 63) ready.fetch_or(1ull << dev);
  }
  if (e != cudaSuccess) return static_cast<int>(e);
  static const bool pingpong = [] {
    const char* v = std::getenv("SDCGUARD_PREFILL_PINGPONG");
    return v == nullptr || v[0] != '0';
  }();
  // with ping-pong, tiles come in pairs of one request (entries 2i and 2i + 1; an odd count is padded by the caller)
  if (pingpong && ntiles % 2) return -3;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(pingpong ? ntiles / 2 : ntiles, nkv);
  cfg.blockDim = dim3(pingpong ? pp::THREADS : 128 + pf::SOFT);
  cfg.dynamicSmemBytes = pingpong ? pp::SMEM : pf::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = overlap ? 1 : 0;
  return static_cast<int>(pingpong ? cudaLaunchKernelEx(&cfg, prefill_pp_kernel, tm, tq, tq1, tr, p)
                                   : cudaLaunchKernelEx(&cfg, prefill_tc_kernel, tm, tr, p));
}

extern "C" {

int sdc_attn_prefill(const void* q, void* o, const void* cache, long long num_blocks, const int* block_table,
                     int max_pages, const int* pos, const void* tiles, int ntiles, const int* row_idx, int nq, int nkv,
                     int head_dim, float scale, void* row_sq, void* check, void* stream) {
  return launch_prefill(q, o, cache, num_blocks, block_table, max_pages, pos, 0x7fffffff, tiles, ntiles, row_idx, nq, nkv,
                        head_dim, scale, row_sq, check, false, static_cast<cudaStream_t>(stream));
}

// The prefill over pages that the kernel before it in the stream writes (sdc_kv8_expand): it starts while that one runs
// and waits for it before its first page. Positions beyond the block table's rows (max_pages * 16) are rows without keys.
struct AttnPrefillArgs {
  const void* q;
  void* o;
  const void* cache;
  long long num_blocks;
  const int* block_table;
  int max_pages;
  const int* pos;
  const void* tiles;
  int ntiles;
  const int* row_idx;
  int nq;
  int nkv;
  float scale;
  void* row_sq;
  void* check;
  void* stream;
};
int sdc_attn_prefill_expanded(const AttnPrefillArgs* a) {
  return launch_prefill(a->q, a->o, a->cache, a->num_blocks, a->block_table, a->max_pages, a->pos, a->max_pages * PAGE,
                        a->tiles, a->ntiles, a->row_idx, a->nq, a->nkv, D, a->scale, a->row_sq, a->check, true,
                        static_cast<cudaStream_t>(a->stream));
}

int sdc_attn_decode_splits(int max_ctx) { return (max_ctx + SEG_KEYS - 1) / SEG_KEYS; }

// Scratch: `part` holds nseq_rows x nkv x max_splits x (nq / nkv) x (D + 4) floats, where nseq_rows covers
// every sequence index used (seq_idx entries included) and max_splits = sdc_attn_decode_splits(max_ctx).
int sdc_attn_decode(const void* q, void* o, const void* cache, long long num_blocks, const int* block_table,
                    int max_pages, const int* seq_req, const int* ctx, const int* seq_idx, int nseq, int nq, int nkv,
                    int head_dim, int max_ctx, float scale, void* part, void* row_sq, void* check, void* stream) {
  if (nseq <= 0) return 0;
  if (head_dim != D || nq % nkv || part == nullptr || nq / nkv > 8) return -1;
  // the layer's cache as [num_blocks * 2 * nkv * 16 rows, 128] bf16; one box = one page of K or V, half the dims
  CUtensorMap tm;
  if (!make_map_bf16_sw128(&tm, cache, num_blocks * 2 * nkv * PAGE, D, D, 64, PAGE)) return -2;
  DecodeParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.o = static_cast<__nv_bfloat16*>(o);
  p.cache = static_cast<const __nv_bfloat16*>(cache);
  p.block_table = block_table;
  p.max_pages = max_pages;
  p.seq_req = seq_req;
  p.ctx = ctx;
  p.seq_idx = seq_idx;
  p.nq = nq;
  p.nkv = nkv;
  p.max_splits = sdc_attn_decode_splits(max_ctx);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(part);
  p.row_sq = static_cast<float*>(row_sq);
  p.err = nullptr;
  p.check = static_cast<unsigned long long*>(check);
  if (p.check != nullptr && seq_idx == nullptr) return -1;
  const int G = nq / nkv;
  // CTAs per (sequence, kv head): enough for about four waves of three CTAs per SM over the whole batch
  int z = (148 * 3 * 4 + nseq * nkv - 1) / (nseq * nkv);
  z = z < 1 ? 1 : (z > p.max_splits ? p.max_splits : z);
  if (max_ctx > MAX_BT * PAGE) return -1;
  dim3 grid(nseq, nkv, z), grid2(nseq, nkv);
  auto st = static_cast<cudaStream_t>(stream);
  switch (G) {
    case 1: return launch_decode<1>(p, tm, grid, grid2, st);
    case 2: return launch_decode<2>(p, tm, grid, grid2, st);
    case 4: return launch_decode<4>(p, tm, grid, grid2, st);
    case 8: return launch_decode<8>(p, tm, grid, grid2, st);
    default:
      return -1;
  }
}

}  // extern "C"

// run-time wait limit of this unit (see common.cuh)
SDC_WAIT_LIMIT_SETTER(attention)
