// A whole MoE layer for up to 16 tokens in two kernels: x -> router logits | top-k, softmax over the selected logits, fc1 + SwiGLU, fc2, sum over
// the selected experts:
//     logits = x Wg + bg,   y_t = sum_j g_tj (SwiGLU(x_t W1_e + b1_e) W2_e + b2_e),   e = the j-th largest logit, g = softmax of the k largest.
//
// What bounds it: the active experts' packed weights, 13 MB per expert of 2880 x 2880, read once, and below some four tokens the latency of the
// steps that depend on one another.  Hence two kernels, and few waits in the second:
//  1. moe_tokens_router_kernel, a CTA per expert: its logit of every token, on CUDA cores (an expert's row of Wg is 6 KB: nothing to tile).
//  2. moe_tokens_kernel, one CTA per SM, launched cooperatively.  Every CTA selects the k best of every token for itself (a warp per token), so that the
//     list of active experts needs no exchange.  Weights are cut into units of 32 rows over all of k; a unit is streamed in stages of 512 k (one
//     TMA box of values, one of scales) by one thread through a ring that takes what shared memory is left.  fc1's units are dealt out evenly, and fc2's
//     stages, whose sums may be cut anywhere.  fc2 reads all of fc1's outputs of an expert: a counter per expert in global memory says when they are
//     there, and the ring goes on filling with fc2's weights meanwhile (one token of four experts: all of them).
//     fc2's partial sums go to the workspace; a counter per 32 output columns tells the CTA whose contribution completes them, which adds them up in
//     a fixed order (slots, then parts along k): the result does not depend on who comes last.
//
// Arithmetic: a code converts to fp16 exactly (two codes an instruction), tokens are fp16 scaled by a power of two per row that puts the largest
// finite element in [2^11, 2^12): elements down to 2^-25 of it keep all of bf16's bits.  mma.sync m16n8k16 sums one scale group of 32 k in fp32, which
// is multiplied by the group's scale and added up in fp32.  The legacy tensor path is far more than 16 tokens need, and its fragments come straight
// from the packed words.  SwiGLU outputs stay fp32 in the workspace; as operand they are fp16 of the row's scale, 2^-12 of a value off, in two terms
// (2^-23) where the expert has at most half as many tokens as there are columns.
#include "gemm_tc_common.cuh"
#include "topk_select.cuh"
#include <cuda_fp16.h>

namespace {

constexpr int MT_MAX_TOKENS = 16;
constexpr int MT_MAX_K = 16;              // picks per token
constexpr int MT_MAX_EXPERTS = 256;
constexpr int MT_WARPS = 16;              // consumer warps: 8 shares of k times 2 slabs of 16 weight rows
constexpr int MT_CONSUMERS = MT_WARPS * 32;
constexpr int MT_THREADS = MT_CONSUMERS + 32;
constexpr int MT_UNIT = 32;               // weight rows of a unit
constexpr int MT_STAGE_KT = 4;            // 128-k tiles of a stage
constexpr int MT_STAGE_VALUES = MT_STAGE_KT * 4 * MT_UNIT * 16;
constexpr int MT_STAGE_BYTES = MT_STAGE_VALUES + MT_STAGE_KT * MT_UNIT * 4;
constexpr int MT_MAX_STAGES = 24;
constexpr int MT_COUNTERS = 256;          // words of each of the three counter arrays
constexpr int MT_ROUTER_THREADS = 256;

struct TokensParams {
  const void* x; int x_dtype; int64_t ld_x;
  int T, d, ff, E, k;
  const void* b1; int b1_dtype; int64_t ld_b1;
  const void* b2; int b2_dtype; int64_t ld_b2;
  float alpha, limit; int has_limit;
  void* y; int64_t ld_y; int y_dtype;
  // workspace
  float* logits; float* xmax;
  int32_t* done1; int32_t* done2; uint32_t* hmax;       // units of fc1 per expert, stages of fc2 per 32 columns, largest |h| per entry
  float* h; float* part;
  int stages, tok_bytes;                // of the ring; shared memory of the staged tokens
  int32_t* status;
};
struct TokensMaps { CUtensorMap v1, s1, v1t, s1t, v2, s2, v2t, s2t; };     // values and scales of whole and of last stages

// ---- router ----------------------------------------------------------------------------------------------------
template <typename TX> __device__ __forceinline__ void load8(const TX* p, float (&f)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const TX* e = reinterpret_cast<const TX*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<TX>(e[i]);
}

// TP: tokens rounded up to a power of two.  A thread takes every 256th chunk of eight k of all tokens.
template <typename TX, int TP>
__global__ void __launch_bounds__(MT_ROUTER_THREADS)
moe_tokens_router_kernel(const TX* x, int64_t ld_x, int T, int d, const __nv_bfloat16* wg, int64_t ld_wg, const void* bg, int bg_dtype, int E,
                         float* logits, float* xmax, int32_t* counters) {
  __shared__ float s_sum[MT_ROUTER_THREADS / 32][TP];
  const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_begin();
  if (e == 0)
    for (int i = threadIdx.x; i < 3 * MT_COUNTERS; i += MT_ROUTER_THREADS) counters[i] = 0;
  float acc[TP];
#pragma unroll
  for (int t = 0; t < TP; ++t) acc[t] = 0.0f;
  for (int c = threadIdx.x; c < d / 8; c += MT_ROUTER_THREADS) {
    float w[8];
    load8(wg + e * ld_wg + c * 8, w);
#pragma unroll
    for (int t = 0; t < TP; ++t)
      if (t < T) {
        float v[8];
        load8(x + t * ld_x + c * 8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[t] = fmaf(w[i], v[i], acc[t]);
      }
  }
#pragma unroll
  for (int t = 0; t < TP; ++t) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) acc[t] += __shfl_xor_sync(0xFFFFFFFFu, acc[t], o);
    if (lane == 0) s_sum[warp][t] = acc[t];
  }
  __syncthreads();
  if (threadIdx.x < T) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < MT_ROUTER_THREADS / 32; ++w) v += s_sum[w][threadIdx.x];
    if (bg) v += load_bias(bg, bg_dtype, e);
    logits[threadIdx.x * E + e] = v;
  }
  // largest finite element of a token's row, which the second kernel scales by
  for (int t = e; t < T; t += E) {
    float mx = 0.0f;
    for (int c = threadIdx.x; c < d / 8; c += MT_ROUTER_THREADS) {
      float v[8];
      load8(x + t * ld_x + c * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]);
        if (a < __int_as_float(0x7F800000)) mx = fmaxf(mx, a);
      }
    }
    const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(mx));
    __syncthreads();                                           // (s_sum is free; uniform: e and T are the block's)
    if (lane == 0) s_sum[warp][0] = __uint_as_float(m);
    __syncthreads();
    if (threadIdx.x == 0) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < MT_ROUTER_THREADS / 32; ++w) v = fmaxf(v, s_sum[w][0]);
      xmax[t] = v;
    }
  }
}

// ---- layer -----------------------------------------------------------------------------------------------------
// e2m1 codes of a word -> fp16 pairs: byte b holds k = (0, 2), (4, 6), (1, 3), (5, 7) of its eight
__device__ __forceinline__ void e2m1_word(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// e8m0 byte -> 2^(byte - 127): byte 0 is 0.0 and byte 255 is NaN, as the dequantiser has them
__device__ __forceinline__ float e8m0_f32(uint32_t b) { return __uint_as_float((b << 23) | ((b + 1u) >> 8)); }
// power of two that puts the largest finite element of a row in [2^11, 2^12)
__device__ __forceinline__ int row_exponent(float mx) { return max(-126, min(116, (int)(__float_as_uint(mx) >> 23) - 127 - 11)); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// eight consecutive k of a token as the B fragments of their two MMAs
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(half2_bits(v[0], v[2]), half2_bits(v[4], v[6]), half2_bits(v[1], v[3]), half2_bits(v[5], v[7]));
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ int ld_acquire(const int32_t* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void consumer_bar() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
static_assert(MT_CONSUMERS == 512, "consumer_bar");

struct TokensShared {                   // beside ring, staged tokens and partial sums
  uint64_t full[MT_MAX_STAGES], empty[MT_MAX_STAGES];
  int abort;
  int n_active;
  int counts[8];
  int act[MT_MAX_EXPERTS];              // active experts in ascending order
  uint16_t rank[MT_MAX_EXPERTS];        // place of an expert in that list
  uint16_t tokens[MT_MAX_EXPERTS];      // its tokens, a bit each
  alignas(16) uint8_t slot[MT_MAX_EXPERTS][MT_MAX_TOKENS];     // which pick of the token it is
  uint8_t sel[MT_MAX_TOKENS][MT_MAX_K];
  float gate[MT_MAX_TOKENS][MT_MAX_K];
  float undo[MT_MAX_TOKENS];            // 2^exponent of the staged rows
  int n_done;
  int done[MT_COUNTERS];
};

// A warp selects the k largest logits of token t, ties to the lower expert, and their softmax
__device__ __forceinline__ void select_token(const TokensParams& p, TokensShared& s, int t, int lane) {
  uint32_t key[MT_MAX_EXPERTS / 32];
#pragma unroll
  for (int i = 0; i < MT_MAX_EXPERTS / 32; ++i) {
    const int e = lane + 32 * i;
    key[i] = e < p.E ? sel_float_key(__ldcg(p.logits + t * p.E + e)) : 0u;
  }
  float first = 0.0f, sum = 0.0f, mine = 0.0f;
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = 0u;
    int at = MT_MAX_EXPERTS;
#pragma unroll
    for (int i = 0; i < MT_MAX_EXPERTS / 32; ++i)
      if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
    const int e = __reduce_min_sync(0xFFFFFFFFu, best == top ? at : MT_MAX_EXPERTS);
#pragma unroll
    for (int i = 0; i < MT_MAX_EXPERTS / 32; ++i)
      if (lane + 32 * i == e) key[i] = 0u;
    const float v = sel_key_float(top);
    if (j == 0) first = v;
    const float w = expf(v - first);
    sum += w;
    if (lane == j) mine = w;
    if (lane == 0) s.sel[t][j] = (uint8_t)e;
  }
  if (lane < p.k) s.gate[t][lane] = __fdiv_rn(mine, sum);
}

template <int NBLK>                     // blocks of eight token columns
__global__ void __launch_bounds__(MT_THREADS, 1) moe_tokens_kernel(const TokensParams p, const __grid_constant__ TokensMaps maps) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 127) & ~(uintptr_t)127);
  __shared__ TokensShared s;
  __shared__ __align__(16) float s_red[2][8][2 * NBLK * 128];          // [buffer][share of k][slab, block, lane, 4]
  const uint32_t ring = smem_u32(smem), toks = ring + (uint32_t)(p.stages * MT_STAGE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto FULL = [&](int i) { return smem_u32(&s.full[i]); };
  auto EMPTY = [&](int i) { return smem_u32(&s.empty[i]); };
  const Ctl ctl{&s.abort, p.status};

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(FULL(i), 1);
      mbar_init(EMPTY(i), MT_WARPS);
    }
    s.abort = 0;
    s.n_done = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < MT_MAX_EXPERTS) *reinterpret_cast<uint4*>(s.slot[threadIdx.x]) = make_uint4(~0u, ~0u, ~0u, ~0u);
  if (warp < p.T) select_token(p, s, warp, lane);
  __syncthreads();
  if (threadIdx.x < p.T * p.k) {
    const int t = threadIdx.x / p.k, j = threadIdx.x - t * p.k;
    s.slot[s.sel[t][j]][t] = (uint8_t)j;
  }
  __syncthreads();
  {
    uint32_t mask = 0;
    const int e = threadIdx.x;
    if (e < MT_MAX_EXPERTS) {
#pragma unroll
      for (int t = 0; t < MT_MAX_TOKENS; ++t) mask |= (s.slot[e][t] != 0xFF ? 1u : 0u) << t;
      s.tokens[e] = (uint16_t)mask;
    }
    const uint32_t live = __ballot_sync(0xFFFFFFFFu, mask != 0);
    if (e < MT_MAX_EXPERTS && lane == 0) s.counts[warp] = __popc(live);
    __syncthreads();
    if (e < MT_MAX_EXPERTS) {
      int at = __popc(live & ((1u << lane) - 1u));
      for (int w = 0; w < warp; ++w) at += s.counts[w];
      if (mask) { s.act[at] = e; s.rank[e] = (uint16_t)at; }
      if (e == MT_MAX_EXPERTS - 1) s.n_active = at + (mask ? 1 : 0);
    }
    __syncthreads();
  }

  const int A = s.n_active, G = gridDim.x, c = blockIdx.x;
  const int KT1 = (p.d + 127) >> 7, KT2 = (p.ff + 127) >> 7, KS1 = (KT1 + MT_STAGE_KT - 1) / MT_STAGE_KT, KS2 = (KT2 + MT_STAGE_KT - 1) / MT_STAGE_KT;
  const int NB1 = 2 * p.ff / MT_UNIT, NB2 = p.d / MT_UNIT;
  const int U1 = A * NB1;
  const int64_t S2 = (int64_t)A * NB2 * KS2;
  const int u_begin = (int)((int64_t)U1 * c / G), u_end = (int)((int64_t)U1 * (c + 1) / G);
  const int64_t s_begin = S2 * c / G, s_end = S2 * (c + 1) / G;

  if (warp == MT_WARPS) {
    // ================================= weights =================================================================
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      auto stage = [&](const CUtensorMap* v, const CUtensorMap* sc, int tiles, int nb, int64_t tile) {
        const int i = it % p.stages;
        ok = mbar_wait(EMPTY(i), ((it / p.stages) & 1u) ^ 1u, ctl, 1001);
        if (!ok) return;
        const uint32_t dst = ring + (uint32_t)(i * MT_STAGE_BYTES);
        mbar_expect_tx(FULL(i), (uint32_t)(tiles * MT_UNIT * 68));
        tma_tile_2d(dst, v, (nb & 3) * 128, (int)(tile * 4), FULL(i));
        tma_tile_2d(dst + MT_STAGE_VALUES, sc, (nb & 3) * 32, (int)tile, FULL(i));
        ++it;
      };
      const int NT1 = (2 * p.ff + 127) >> 7, NT2 = (p.d + 127) >> 7;
      const int tail1 = KT1 - (KS1 - 1) * MT_STAGE_KT, tail2 = KT2 - (KS2 - 1) * MT_STAGE_KT;
      for (int u = u_begin; u < u_end && ok; ++u) {
        const int a = u / NB1, nb = u - a * NB1;
        const int64_t tile = ((int64_t)s.act[a] * NT1 + (nb >> 2)) * KT1;
        for (int js = 0; js < KS1 && ok; ++js) {
          if (js < KS1 - 1) stage(&maps.v1, &maps.s1, MT_STAGE_KT, nb, tile + js * MT_STAGE_KT);
          else stage(&maps.v1t, &maps.s1t, tail1, nb, tile + js * MT_STAGE_KT);
        }
      }
      for (int64_t q = s_begin; q < s_end && ok; ++q) {
        const int u = (int)(q / KS2), js = (int)(q - (int64_t)u * KS2), a = u / NB2, nb = u - a * NB2;
        const int64_t tile = ((int64_t)s.act[a] * NT2 + (nb >> 2)) * KT2;
        if (js < KS2 - 1) stage(&maps.v2, &maps.s2, MT_STAGE_KT, nb, tile + js * MT_STAGE_KT);
        else stage(&maps.v2t, &maps.s2t, tail2, nb, tile + js * MT_STAGE_KT);
      }
      if (!ok) {                                              // copies in flight land before the block's shared memory goes
        const uint32_t lo = it > (uint32_t)p.stages ? it - p.stages : 0;
        for (uint32_t j = lo; j < it; ++j)
          for (uint32_t t = 0; t < (1u << 16) && !mbar_test(FULL(j % p.stages), (j / p.stages) & 1u); ++t) __nanosleep(64);
      }
    }
    return;
  }

  // ================================= consumers =================================================================
  const int wk = warp & 7, slab = warp >> 3, qrow = lane >> 2, c4 = lane & 3;
  const int tid = threadIdx.x;
  bool dead = false;                    // a wait ran out: the rest is gone through without waiting, its results are void
  uint32_t it = 0, buf = 0;
  float acc[NBLK][4];

  // staged token column col, eight k from 8 * k8 on
  auto tok_at = [&](int col, int k8) { return toks + (uint32_t)((((k8 >> 2) * NBLK + (col >> 3)) * 8 + (col & 7)) * 64 + (k8 & 3) * 16); };
  auto red_at = [&](int row, int col) {
    return (((row >> 4) * NBLK + (col >> 3)) * 32 + (row & 7) * 4 + ((col & 7) >> 1)) * 4 + ((row >> 3) & 1) * 2 + (col & 1);
  };
  // one stage of a unit: groups wk and wk + 8 of its up to sixteen
  auto multiply = [&](int tiles, int group0, uint32_t blocks) {
    const int i = it % p.stages;
    if (!dead) dead = !__all_sync(0xFFFFFFFFu, mbar_wait(FULL(i), (it / p.stages) & 1u, ctl, 1002));
    const uint32_t st = ring + (uint32_t)(i * MT_STAGE_BYTES), row = (uint32_t)(slab * 16 + qrow);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int g = wk + 8 * hf;
      if (g < tiles * 4) {
        const uint32_t wl = lds32(st + g * 512 + row * 16 + c4 * 4), wh = lds32(st + g * 512 + row * 16 + 128 + c4 * 4);
        const uint32_t sc = st + MT_STAGE_VALUES + (g >> 2) * 128 + row * 4 + (g & 3);
        const float fl = e8m0_f32(lds8(sc)), fh = e8m0_f32(lds8(sc + 32));
        uint32_t lo[4], hi[4];
        e2m1_word(wl, lo);
        e2m1_word(wh, hi);
#pragma unroll
        for (int b = 0; b < NBLK; ++b)
          if (NBLK == 1 || (blocks >> b & 1)) {
            const uint4 xb = lds128(toks + (uint32_t)((((group0 + g) * NBLK + b) * 8 + qrow) * 64 + c4 * 16));
            float dd[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_f16(dd, lo[0], hi[0], lo[1], hi[1], xb.x, xb.y);
            mma_f16(dd, lo[2], hi[2], lo[3], hi[3], xb.z, xb.w);
            acc[b][0] = fmaf(fl, dd[0], acc[b][0]);
            acc[b][1] = fmaf(fl, dd[1], acc[b][1]);
            acc[b][2] = fmaf(fh, dd[2], acc[b][2]);
            acc[b][3] = fmaf(fh, dd[3], acc[b][3]);
          }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(EMPTY(i));
    ++it;
  };
  auto clear = [&]() {
#pragma unroll
    for (int b = 0; b < NBLK; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[b][j] = 0.0f;
  };
  // the eight shares of k meet; the buffers alternate, so that a warp may be a unit ahead of those that still add
  auto meet = [&]() {
    buf ^= 1u;
#pragma unroll
    for (int b = 0; b < NBLK; ++b)
      *reinterpret_cast<float4*>(&s_red[buf][wk][((slab * NBLK + b) * 32 + lane) * 4]) = make_float4(acc[b][0], acc[b][1], acc[b][2], acc[b][3]);
    consumer_bar();
  };
  auto summed = [&](int row, int col) {
    const int at = red_at(row, col);
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += s_red[buf][w][at];
    return v;
  };

  // ---- tokens as the columns of fc1, in their order ----
  for (int i = tid; i < p.T * KT1 * 16; i += MT_CONSUMERS) {
    const int t = i / (KT1 * 16), k8 = i - t * (KT1 * 16);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (k8 * 8 < p.d) {
      if (p.x_dtype == MOE_F16) load8((const __half*)p.x + t * p.ld_x + k8 * 8, v);
      else load8((const __nv_bfloat16*)p.x + t * p.ld_x + k8 * 8, v);
    }
    const float down = pow2(-row_exponent(__ldcg(p.xmax + t)));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= down;
    sts128(tok_at(t, k8), pack8(v));
  }
  if (tid < p.T) s.undo[tid] = pow2(row_exponent(__ldcg(p.xmax + tid)));
  consumer_bar();

  // ---- fc1 ----
  for (int u = u_begin; u < u_end; ++u) {
    const int a = u / NB1, nb = u - a * NB1, e = s.act[a];
    const uint32_t mask = s.tokens[e];
    const uint32_t blocks = (mask & 0xFFu ? 1u : 0u) | (mask >> 8 ? 2u : 0u);
    clear();
    for (int js = 0; js < KS1; ++js) multiply(min(MT_STAGE_KT, KT1 - js * MT_STAGE_KT), js * 16, blocks);
    meet();
    const int n = __popc(mask);
    if ((tid & ~31) < n * 16) {                               // sixteen outputs of a token by half a warp
      const bool live = tid < n * 16;
      const int t = __fns(mask, 0, live ? (tid >> 4) + 1 : n), i = tid & 15, o = nb * 16 + i;
      float g = summed(2 * i, t) * s.undo[t], l = summed(2 * i + 1, t) * s.undo[t];
      if (p.b1) {
        g += load_bias(p.b1, p.b1_dtype, e * p.ld_b1 + 2 * o);
        l += load_bias(p.b1, p.b1_dtype, e * p.ld_b1 + 2 * o + 1);
      }
      if (p.has_limit) {
        g = min_nan(g, p.limit);
        l = max_nan(min_nan(l, p.limit), -p.limit);
      }
      const float sg = __fdividef(g, 1.0f + gemm_ex2(-p.alpha * g * 1.4426950408889634f)), v = fmaf(sg, l, sg);
      const int entry = t * p.k + s.slot[e][t];
      if (live) __stcg(p.h + (int64_t)entry * p.ff + o, v);
      float m = fabsf(v) < __int_as_float(0x7F800000) ? fabsf(v) : 0.0f;
#pragma unroll
      for (int x = 8; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
      if (live && i == 0) atomicMax(p.hmax + entry, __float_as_uint(m));
    }
    if (u + 1 == u_end || nb + 1 == NB1) {                    // the last of this expert's units here
      consumer_bar();
      if (tid == 0) {
        __threadfence();
        atomicAdd(p.done1 + e, min(nb + 1, u + 1 - u_begin));
      }
    }
  }

  // ---- fc2 ----
  int have = -1, n = 0, cols = 0;       // expert whose rows are staged, its tokens, columns they take
  for (int64_t q = s_begin; q < s_end;) {
    const int u = (int)(q / KS2), js0 = (int)(q - (int64_t)u * KS2), a = u / NB2, e = s.act[a];
    const int js1 = (int)min((int64_t)KS2, js0 + (s_end - q));
    const uint32_t mask = s.tokens[e];
    if (e != have) {
      if (tid == 0 && !dead) {
        const long long t0 = clock64();
        while (ld_acquire(p.done1 + e) < NB1) {
          if (s.abort) break;
          if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
            s.abort = 1;
            if (p.status) atomicExch(p.status, 1003);
            break;
          }
        }
      }
      consumer_bar();                                         // fc1's rows are there, and the staged ones have been read
      n = __popc(mask);
      const bool two = 2 * n <= 8 * NBLK;
      cols = two ? 2 * n : n;
      for (int i = tid; i < n * KT2 * 16; i += MT_CONSUMERS) {
        const int r = i / (KT2 * 16), k8 = i - r * (KT2 * 16), t = __fns(mask, 0, r + 1), entry = t * p.k + s.slot[e][t];
        const float down = pow2(-row_exponent(__uint_as_float(__ldcg(p.hmax + entry))));
        float v[8], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        if (k8 * 8 < p.ff) {
          const float4* src = reinterpret_cast<const float4*>(p.h + (int64_t)entry * p.ff + k8 * 8);
          const float4 v0 = __ldcg(src), v1 = __ldcg(src + 1);
          v[0] = v0.x; v[1] = v0.y; v[2] = v0.z; v[3] = v0.w; v[4] = v1.x; v[5] = v1.y; v[6] = v1.z; v[7] = v1.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] *= down;
          const float left = v[j] - __half2float(__float2half_rn(v[j]));
          w[j] = isfinite(left) ? left : 0.0f;                // (infinities and NaN are the first term's)
        }
        sts128(tok_at(r, k8), pack8(v));
        if (two) sts128(tok_at(n + r, k8), pack8(w));
      }
      if (tid < n) {
        const int t = __fns(mask, 0, tid + 1);
        s.undo[tid] = pow2(row_exponent(__uint_as_float(__ldcg(p.hmax + t * p.k + s.slot[e][t]))));
      }
      consumer_bar();
      have = e;
    }
    clear();
    for (int js = js0; js < js1; ++js) multiply(min(MT_STAGE_KT, KT2 - js * MT_STAGE_KT), js * 16, cols > 8 ? 3u : 1u);
    meet();
    if (tid < n * MT_UNIT) {
      const int r = tid >> 5;
      float v = summed(lane, r);
      if (cols > n) v += summed(lane, n + r);
      __stcg(p.part + ((int64_t)(u + c) * p.T + r) * MT_UNIT + lane, v * s.undo[r]);
    }
    q += js1 - js0;
  }

  // ---- whoever completes 32 output columns adds them up ----
  consumer_bar();
  const int first = (int)(s_begin / KS2), n_parts = s_end > s_begin ? (int)((s_end - 1) / KS2) - first + 1 : 0;
  for (int i = tid; i < n_parts; i += MT_CONSUMERS) {
    const int u = first + i, nb = u % NB2;
    const int mine = (int)(min(s_end, (int64_t)(u + 1) * KS2) - max(s_begin, (int64_t)u * KS2));
    __threadfence();
    if (atomicAdd(p.done2 + nb, mine) + mine == A * KS2) s.done[atomicAdd(&s.n_done, 1)] = nb;
  }
  consumer_bar();
  const int n_done = s.n_done;
  if (n_done == 0) return;
  __threadfence();
  for (int i = tid; i < n_done * p.T * MT_UNIT; i += MT_CONSUMERS) {
    const int w = i >> 5, nb = s.done[w / p.T], t = w % p.T, o = nb * MT_UNIT + lane;
    float y = 0.0f;
    for (int j = 0; j < p.k; ++j) {
      const int e = s.sel[t][j], u = (int)s.rank[e] * NB2 + nb, r = __popc(s.tokens[e] & ((1u << t) - 1u));
      // the CTAs whose ranges the unit's stages are in (those between with nothing to do where there are fewer stages than CTAs)
      const int c0 = (int)((((int64_t)u * KS2 + 1) * G - 1) / S2), c1 = (int)((((int64_t)(u + 1) * KS2) * G - 1) / S2);
      float v = p.b2 ? load_bias(p.b2, p.b2_dtype, e * p.ld_b2 + o) : 0.0f;
      for (int cc = c0; cc <= c1; ++cc)
        if (S2 * cc / G < S2 * (cc + 1) / G) v += __ldcg(p.part + ((int64_t)(u + cc) * p.T + r) * MT_UNIT + lane);
      y = fmaf(s.gate[t][j], v, y);
    }
    if (p.y_dtype == MOE_F16) ((__half*)p.y)[t * p.ld_y + o] = __float2half_rn(y);
    else ((__nv_bfloat16*)p.y)[t * p.ld_y + o] = __float2bfloat16_rn(y);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------
// tiles as a matrix of 32-bit words: `words` per row, boxes of `box_w` words and `box_h` rows
int mt_map(const void* base, uint64_t words, uint64_t rows, uint32_t box_w, uint32_t box_h, CUtensorMap* map) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  static std::mutex mu;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!encode) {
      void* fn = nullptr;
      cudaDriverEntryPointQueryResult qr;
      MOE_CHECK_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &qr));
      if (qr != cudaDriverEntryPointSuccess || !fn) {
        moe_set_error("moe_layer_tokens: the driver does not provide cuTensorMapEncodeTiled");
        return MOE_ERR_UNSUPPORTED;
      }
      encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }
  }
  const cuuint64_t dims[2] = {words, rows}, strides[1] = {words * 4};
  const cuuint32_t box[2] = {box_w, box_h}, estr[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    moe_set_error("moe_layer_tokens: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return MOE_ERR_CUDA;
  }
  return MOE_OK;
}
int mt_weight_maps(const void* values, const void* scales, int E, int K, int N, CUtensorMap* v, CUtensorMap* sc, CUtensorMap* vt, CUtensorMap* st) {
  const uint64_t KT = (uint64_t)cdiv64(K, 128), tiles = (uint64_t)E * (uint64_t)cdiv64(N, 128) * KT;
  const uint32_t tail = (uint32_t)(KT - (cdiv64(KT, MT_STAGE_KT) - 1) * MT_STAGE_KT);
  if (int rc = mt_map(values, 512, tiles * 4, 128, MT_STAGE_KT * 4, v)) return rc;
  if (int rc = mt_map(scales, 128, tiles, 32, MT_STAGE_KT, sc)) return rc;
  if (int rc = mt_map(values, 512, tiles * 4, 128, tail * 4, vt)) return rc;
  return mt_map(scales, 128, tiles, 32, tail, st);
}

struct TokensWorkspace { size_t logits, xmax, counters, h, part, bytes; };
TokensWorkspace mt_workspace(const MoeTokensArgs& a) {
  TokensWorkspace w;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
  const int64_t n = (int64_t)a.T * a.k, active = n < a.E ? n : a.E;
  w.counters = take(3 * MT_COUNTERS * 4);
  w.logits = take((size_t)a.T * a.E * 4);
  w.xmax = take((size_t)a.T * 4);
  w.h = take((size_t)(n * a.ff) * 4);
  w.part = take((size_t)((active * (a.d / MT_UNIT) + moe_sm_count()) * a.T) * MT_UNIT * 4);
  w.bytes = at;
  return w;
}

// the shared memory that is left for the ring, whole stages
constexpr int MT_SMEM = 232448;
template <int NBLK> int mt_static_smem() {
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, moe_tokens_kernel<NBLK>) != cudaSuccess) return MT_SMEM;
  return (int)at.sharedSizeBytes;
}

int mt_check(const MoeTokensArgs* a) {
  MOE_CHECK_ARG(a, "moe_layer_tokens: NULL argument");
  MOE_CHECK_ARG(a->T >= 0 && a->d > 0 && a->ff > 0 && a->E > 0 && a->k > 0, "moe_layer_tokens: sizes must be positive");
  MOE_CHECK_ARG(a->d % 32 == 0 && a->ff % 32 == 0, "moe_layer_tokens: d and ff must be multiples of 32 (got %d, %d)", a->d, a->ff);
  MOE_CHECK_ARG(a->k <= a->E, "moe_layer_tokens: k = %d of %d experts", a->k, a->E);
  const int width = a->d > a->ff ? a->d : a->ff;
  if (a->T > MT_MAX_TOKENS || a->k > MT_MAX_K || a->E > MT_MAX_EXPERTS || width > (a->T > 8 ? 4096 : 8192)) {
    moe_set_error("moe_layer_tokens: takes at most %d tokens, %d picks of %d experts and widths of 8192 (4096 with more than 8 tokens); got T = %d, "
                  "k = %d, E = %d, d = %d, ff = %d", MT_MAX_TOKENS, MT_MAX_K, MT_MAX_EXPERTS, a->T, a->k, a->E, a->d, a->ff);
    return MOE_ERR_UNSUPPORTED;
  }
  return MOE_OK;
}

template <typename TX> int mt_router(const MoeTokensArgs& a, float* logits, float* xmax, int32_t* counters, cudaStream_t st) {
#define MT_ROUTER(TP)                                                                                                                    \
  MOE_CHECK_CUDA(launch_pdl(moe_tokens_router_kernel<TX, TP>, dim3((unsigned)a.E), dim3(MT_ROUTER_THREADS), (size_t)0, st, (const TX*)a.x, a.ld_x, \
                            a.T, a.d, (const __nv_bfloat16*)a.wg_t, a.ld_wg, a.bg, a.bg_dtype, a.E, logits, xmax, counters))
  if (a.T <= 1) MT_ROUTER(1);
  else if (a.T <= 2) MT_ROUTER(2);
  else if (a.T <= 4) MT_ROUTER(4);
  else if (a.T <= 8) MT_ROUTER(8);
  else MT_ROUTER(16);
#undef MT_ROUTER
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <int NBLK> int mt_launch(TokensParams& p, const TokensMaps& maps, cudaStream_t st) {
  const int width = p.d > p.ff ? p.d : p.ff;
  p.tok_bytes = (int)cdiv64(width, 128) * 4 * 512 * NBLK;
  const int left = MT_SMEM - mt_static_smem<NBLK>() - 128 - p.tok_bytes;
  p.stages = left / MT_STAGE_BYTES < MT_MAX_STAGES ? left / MT_STAGE_BYTES : MT_MAX_STAGES;
  if (p.stages < 2) {
    moe_set_error("moe_layer_tokens: no shared memory left for weights (d = %d, ff = %d)", p.d, p.ff);
    return MOE_ERR_UNSUPPORTED;
  }
  const int smem = p.tok_bytes + p.stages * MT_STAGE_BYTES + 128;
  MOE_CHECK_CUDA(cudaFuncSetAttribute(moe_tokens_kernel<NBLK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)moe_sm_count());
  cfg.blockDim = dim3(MT_THREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;       // CTAs wait on one another: all of them run at once or the launch is refused
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MOE_CHECK_CUDA(cudaLaunchKernelEx(&cfg, moe_tokens_kernel<NBLK>, p, maps));
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

}  // namespace

extern "C" __attribute__((visibility("default"))) size_t moe_layer_tokens_workspace_bytes(const MoeTokensArgs* a) {
  return mt_check(a) == MOE_OK ? mt_workspace(*a).bytes : 0;
}

extern "C" __attribute__((visibility("default"))) int moe_layer_tokens(const MoeTokensArgs* args, void* stream) {
  if (int rc = mt_check(args)) return rc;
  const MoeTokensArgs& a = *args;
  if (a.T == 0) return MOE_OK;
  MOE_CHECK_ARG(a.x && a.wg_t && a.w1 && a.w1_scale && a.w2 && a.w2_scale && a.y, "moe_layer_tokens: NULL argument");
  MOE_CHECK_ARG(a.x_dtype == MOE_BF16 || a.x_dtype == MOE_F16, "moe_layer_tokens: x is bf16 or fp16");
  MOE_CHECK_ARG(a.y_dtype == MOE_BF16 || a.y_dtype == MOE_F16, "moe_layer_tokens: y is bf16 or fp16");
  MOE_CHECK_ARG(a.ld_x % 8 == 0 && a.ld_wg % 8 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.wg_t % 16 == 0,
                "moe_layer_tokens: rows of x and Wg^T must be 16-byte aligned");
  MOE_CHECK_ARG((uintptr_t)a.w1 % 16 == 0 && (uintptr_t)a.w1_scale % 16 == 0 && (uintptr_t)a.w2 % 16 == 0 && (uintptr_t)a.w2_scale % 16 == 0,
                "moe_layer_tokens: weight tiles must be 16-byte aligned");
  const TokensWorkspace w = mt_workspace(a);
  MOE_CHECK_ARG(a.workspace && (uintptr_t)a.workspace % 256 == 0 && a.workspace_bytes >= w.bytes,
                "moe_layer_tokens: needs a 256-byte aligned workspace of %zu bytes", w.bytes);
  cudaStream_t st = (cudaStream_t)stream;
  uint8_t* ws = (uint8_t*)a.workspace;
  int32_t* counters = (int32_t*)(ws + w.counters);
  TokensParams p = {};
  p.x = a.x; p.x_dtype = a.x_dtype; p.ld_x = a.ld_x;
  p.T = a.T; p.d = a.d; p.ff = a.ff; p.E = a.E; p.k = a.k;
  p.b1 = a.b1; p.b1_dtype = a.b1_dtype; p.ld_b1 = a.ld_b1;
  p.b2 = a.b2; p.b2_dtype = a.b2_dtype; p.ld_b2 = a.ld_b2;
  p.alpha = a.act_alpha; p.limit = a.act_limit; p.has_limit = a.act_has_limit;
  p.y = a.y; p.ld_y = a.ld_y; p.y_dtype = a.y_dtype;
  p.logits = (float*)(ws + w.logits); p.xmax = (float*)(ws + w.xmax);
  p.done1 = counters; p.done2 = counters + MT_COUNTERS; p.hmax = (uint32_t*)(counters + 2 * MT_COUNTERS);
  p.h = (float*)(ws + w.h); p.part = (float*)(ws + w.part);
  p.status = a.status;
  TokensMaps maps;
  if (int rc = mt_weight_maps(a.w1, a.w1_scale, a.E, a.d, 2 * a.ff, &maps.v1, &maps.s1, &maps.v1t, &maps.s1t)) return rc;
  if (int rc = mt_weight_maps(a.w2, a.w2_scale, a.E, a.ff, a.d, &maps.v2, &maps.s2, &maps.v2t, &maps.s2t)) return rc;
  if (int rc = a.x_dtype == MOE_F16 ? mt_router<__half>(a, p.logits, p.xmax, counters, st) : mt_router<__nv_bfloat16>(a, p.logits, p.xmax, counters, st))
    return rc;
  return a.T > 8 ? mt_launch<2>(p, maps, st) : mt_launch<1>(p, maps, st);
}
