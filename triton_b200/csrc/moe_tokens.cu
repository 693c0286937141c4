// A whole MoE layer for up to 16 tokens in two kernels: x -> router logits | top-k, softmax over the selected logits, fc1 + SwiGLU, fc2, sum over
// the selected experts:
//     logits = x Wg + bg,   y_t = sum_j g_tj (SwiGLU(x_t W1_e + b1_e) W2_e + b2_e),   e = the j-th largest logit, g = softmax of the k largest.
//
// What bounds it: the active experts' packed weights, 13 MB per expert of 2880 x 2880, read once, and below some four tokens the latency of the
// steps that depend on one another.  Hence two kernels, and few waits in the second:
//  1. moe_tokens_router_kernel, a CTA per expert and eight tokens: logits on CUDA cores (an expert's row of Wg is 6 KB: nothing to tile).
//  2. moe_tokens_kernel, one CTA per SM, launched cooperatively.  Every CTA selects the k best of every token for itself (a warp per token), so that the
//     list of active experts needs no exchange.  Weights are cut into units of 32 rows over all of k; a unit is streamed in stages of 1024 k (one
//     TMA box of values, one of scales) by one warp through a ring that takes what shared memory is left.  fc1's units are dealt out evenly by the time they
//     take, and so are fc2's stages, whose sums may be cut anywhere.  fc2 reads all of fc1's outputs of an expert: a counter per expert in global memory says
//     when they are there, and the ring goes on filling with fc2's weights meanwhile (one token of four experts: all of them).
//     fc2's partial sums go to the workspace; a counter per 32 output columns says when they are complete, and a warp of whichever CTA adds up 32
//     outputs of a token in a fixed order (slots, then parts along k): the result does not depend on who comes last.
// Measured, 2880 x 2880, k = 4, 128 experts, router + layer: 1 token 3.7 + 23 us (54 MB), 4 tokens of 13 experts 4.2 + 48 (173 MB, 3.6 TB/s), 16 tokens of 26 experts
// 4.4 + 103 (345 MB, 3.3 TB/s), of 35 experts 125 (464 MB, 3.7 TB/s).  One token: selection 2.2, fc1's first sums 4 later, all of fc1 at 14, its rows staged 1.6 later, fc2 3, the meeting of the sums 2.5.  With more, a
// stage of 17.4 KB takes an SM 0.5 us (its bytes some 0.4 at the copy bandwidth): instructions, 60 % of issue slots and 50 % of the integer pipe, which the
// conversions of codes and scales are two thirds of; the loads of a warp's second tile ahead of the first one's arithmetic made it 7 % slower.
//
// Arithmetic: a code becomes fp16 exactly, tokens are fp16 scaled by their row's largest finite element, which is put in [2^13, 2^14):
// elements down to 2^-30 of it keep all of bf16's bits (27 fp16's), and a sum of more than 2^114 times it is infinite.  mma.sync m16n8k16 sums one scale group of 32 k in fp32, which
// is multiplied by the group's scale and added up in fp32.  The legacy tensor path is far more than 16 tokens need, and its fragments come straight
// from the packed words.  SwiGLU outputs stay fp32 in the workspace; as operand they are two fp16 terms of the row's scale, 2^-23 of a value off (2^-38 of
// the row's largest where it is that small).
#include "gemm_tc_common.cuh"
#include "topk_select.cuh"
#include <cuda_fp16.h>
#include <atomic>
#include <type_traits>

namespace {

constexpr int MT_MAX_TOKENS = 16;
constexpr int MT_MAX_K = 16;              // picks per token
constexpr int MT_MAX_EXPERTS = 256;
constexpr int MT_WARPS = 16;              // consumer warps: two teams of 4 shares of k times 2 slabs of 16 weight rows
constexpr int MT_CONSUMERS = MT_WARPS * 32;
constexpr int MT_EPILOGUE = 96;           // threads that take the sums on while the consumers are at the next unit
constexpr int MT_THREADS = MT_CONSUMERS + MT_EPILOGUE + 32;
constexpr int MT_UNIT = 32;               // weight rows of a unit
constexpr int MT_SHARES = 4;              // of k in a team
constexpr int MT_STAGE_KT = 8;            // 128-k tiles of a stage, two per share of k
constexpr int MT_STAGE_VALUES = MT_STAGE_KT * 4 * MT_UNIT * 16;
constexpr int MT_STAGE_BYTES = MT_STAGE_VALUES + MT_STAGE_KT * MT_UNIT * 4;
constexpr int MT_RED_LD = 36;             // pitch of a column of sums: the quads of an accumulator fragment go to distinct banks
constexpr int MT_MAX_STAGES = 12;
constexpr int MT_COUNTERS = 256;          // words of each of the three counter arrays
constexpr int MT_ROUTER_THREADS = 512;

// x / d by a product, right for x d < 2^40 and x < 2^24 d: a division by a number known at launch only costs some 20 instructions
struct Div { uint32_t d; uint64_t m; };
__device__ __forceinline__ int operator/(int x, const Div& v) { return (int)(((uint64_t)(uint32_t)x * v.m) >> 40); }

struct TokensParams {
  const void* x; int x_dtype; int64_t ld_x;
  int T, d, ff, E, k;
  const uint8_t* s1; const uint8_t* s2;
  const void* b1; int b1_dtype; int64_t ld_b1;
  const void* b2; int b2_dtype; int64_t ld_b2;
  float alpha, limit; int has_limit;
  void* y; int64_t ld_y; int y_dtype;
  // workspace
  float* logits; float* xmax;
  int32_t* done1; int32_t* done2; uint32_t* hmax;       // units of fc1 per expert, stages of fc2 per 32 columns, largest |h| per entry
  float* h; float* part;
  Div by_ctas, by_units1, by_units2, by_steps2;        // CTAs, units of an expert in fc1 and fc2, stages of a unit of fc2
  int stages, tok_bytes;                // of the ring; shared memory of the staged tokens
  int32_t* status;
};
struct TokensMaps { CUtensorMap v1, s1, v1t, s1t, v2, s2, v2t, s2t; };     // values and scales of whole and of last stages

// ---- router ----------------------------------------------------------------------------------------------------
template <typename TX> __device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const TX* e = reinterpret_cast<const TX*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<TX>(e[i]);
}

// Eight tokens by a row of the grid.  CTAs 0 .. E - 1 of a row: an expert's logits of the tokens.  The ones behind: the largest finite element of a
// token's row, which the second kernel scales by.  TP: tokens of a row of the grid, rounded up to a power of two.  A thread takes every 512th chunk of
// eight k of all of them, whose loads are on their way together: what bounds the kernel is how many trips to L2 follow one another (16 tokens of 2880,
// 128 experts: 4.4 us; 18.6 us with a trip per token, 8.4 with all 16 tokens by a thread; one token: 3.7 us).
template <typename TX, int TP>
__global__ void __launch_bounds__(MT_ROUTER_THREADS)
moe_tokens_router_kernel(const TX* x, int64_t ld_x, int T, int d, const __nv_bfloat16* wg, int64_t ld_wg, const void* bg, int bg_dtype, int E,
                         float* logits, float* xmax, int32_t* counters) {
  constexpr int WARPS = MT_ROUTER_THREADS / 32;
  __shared__ float s_sum[WARPS][TP];
  const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = blockIdx.y * 8;
  pdl_begin();
  x += first * ld_x;
  logits += first * E;
  xmax += first;
  T = min(T - first, 8);
  if (e >= E + T) return;
  if (e >= E) {
    float mx = 0.0f;
    for (int c = threadIdx.x; c < d / 8; c += MT_ROUTER_THREADS) {
      float v[8];
      unpack8<TX>(*reinterpret_cast<const uint4*>(x + (e - E) * ld_x + c * 8), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]);
        if (a < __int_as_float(0x7F800000)) mx = fmaxf(mx, a);
      }
    }
    const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(mx));
    if (lane == 0) s_sum[warp][0] = __uint_as_float(m);
    __syncthreads();
    if (threadIdx.x == 0) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v = fmaxf(v, s_sum[w][0]);
      xmax[e - E] = v;
    }
    return;
  }
  if (e == 0 && first == 0)
    for (int i = threadIdx.x; i < 3 * MT_COUNTERS; i += MT_ROUTER_THREADS) counters[i] = 0;
  float acc[TP];
#pragma unroll
  for (int t = 0; t < TP; ++t) acc[t] = 0.0f;
  for (int c = threadIdx.x; c < d / 8; c += MT_ROUTER_THREADS) {
    const uint4 row = *reinterpret_cast<const uint4*>(wg + e * ld_wg + c * 8);
    uint4 raw[TP];
#pragma unroll
    for (int t = 0; t < TP; ++t) raw[t] = *reinterpret_cast<const uint4*>(x + min(t, T - 1) * ld_x + c * 8);      // (sums from T on are left)
    float w[8];
    unpack8<__nv_bfloat16>(row, w);
#pragma unroll
    for (int t = 0; t < TP; ++t) {
      float v[8];
      unpack8<TX>(raw[t], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[t] = fmaf(w[i], v[i], acc[t]);
    }
  }
  // the warp's sums: each step halves the tokens that a lane goes on with, then the lanes that have the same token meet
#pragma unroll
  for (int n = TP / 2, o = 16; o >= 1; n >>= 1, o >>= 1) {
    if (n == 0) {
      acc[0] += __shfl_xor_sync(0xFFFFFFFFu, acc[0], o);
    } else {
      const bool upper = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < TP / 2; ++i)
        if (i < n) {
          const float keep = upper ? acc[i + n] : acc[i], give = upper ? acc[i] : acc[i + n];
          acc[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    }
  }
  if (lane % (32 / TP) == 0) s_sum[warp][lane / (32 / TP)] = acc[0];
  __syncthreads();
  if (threadIdx.x < T) {
    float v[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v[w] = s_sum[w][threadIdx.x];
#pragma unroll
    for (int n = WARPS / 2; n >= 1; n >>= 1)                  // (pairwise: four roundings)
#pragma unroll
      for (int w = 0; w < n; ++w) v[w] += v[w + n];
    if (bg) v[0] += load_bias(bg, bg_dtype, e);
    logits[threadIdx.x * E + e] = v[0];
  }
}

// ---- layer -----------------------------------------------------------------------------------------------------
// The eight e2m1 codes of a word (nibbles k0, k2, k4, k6 | k1, k3, k5, k7, lowest first) -> fp16 pairs (0, 2), (4, 6), (1, 3), (5, 7), exactly.  A resident
// stage, without waits, took 524 cycles of an SM this way, 760 with half of the pairs made by shifts and masks and 967 with all; with a byte brought down by a
// high product, off the integer pipe, a layer of 4 tokens took 71 us in place of 56.
__device__ __forceinline__ void e2m1_word(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// four matrices of 8 rows x 16 bytes at the lanes' addresses: a lane has word lane % 4 of row lane / 4 of each
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e8m0 bytes -> 2^(byte - 127): byte 0 is 0.0 as the dequantiser has it; byte 255, there NaN, gives infinity, which settle() takes up
__device__ __forceinline__ void e8m0_word(uint32_t w, float (&f)[4]) {
  f[0] = __uint_as_float((w << 23) & 0x7F800000u);
  f[1] = __uint_as_float((w << 15) & 0x7F800000u);
  f[2] = __uint_as_float((w << 7) & 0x7F800000u);
  f[3] = __uint_as_float((w >> 1) & 0x7F800000u);
}
// A sum over weight row `row` of expert e: a scale byte of 255 anywhere in the row makes it NaN.  Such a sum has become infinite (or NaN: a group of zeros),
// so only those look at the scales again.
__device__ __forceinline__ float settle(float v, const uint8_t* scales, int e, int NT, int KT, int row) {
  if (fabsf(v) == __int_as_float(0x7F800000)) {
    const uint8_t* at = scales + ((int64_t)(e * NT + (row >> 7)) * KT) * 512 + (row & 127) * 4;
    for (int kt = 0; kt < KT; ++kt) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(at + (int64_t)kt * 512);
      if (((w & 0x7F7F7F7Fu) + 0x01010101u) & w & 0x80808080u) return __int_as_float(0x7FC00000);
    }
  }
  return v;
}
// Exponent of the largest finite element of a row.  Its values as operands are scaled by 2^(13 - exponent): the largest in [2^13, 2^14).
__device__ __forceinline__ int row_exponent(float mx) { return max(-112, min(126, (int)(__float_as_uint(mx) >> 23) - 127)); }
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
// until the counter has got to `full`; bounded like mbar_wait
__device__ __forceinline__ bool wait_count(const int32_t* counter, int full, const Ctl& ctl, int code) {
  if (ld_acquire(counter) >= full) return true;
  const long long t0 = clock64();
  for (uint32_t i = 0;; ++i) {
    if (ld_acquire(counter) >= full) return true;
    if ((i & 7u) == 7u && *ctl.abort_flag) return false;
    if ((i & 255u) == 255u && clock64() - t0 > WAIT_LIMIT_CYCLES) {
      *ctl.abort_flag = 1;
      if (ctl.status) atomicExch(ctl.status, code);
      return false;
    }
  }
}
// named barriers: 1 consumers, 2 epilogue, 3 all but those that stage tokens
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
constexpr int MT_BOTH = MT_CONSUMERS + MT_EPILOGUE;

struct TokensShared {                   // beside ring, staged tokens and partial sums
  uint64_t full[MT_MAX_STAGES], empty[MT_MAX_STAGES];
  uint64_t sums[2], taken[2];           // a buffer of sums is complete, has been read
  int abort;
  int n_active, n_entries;
  uint8_t act[MT_MAX_EXPERTS];          // active experts in ascending order
  uint8_t from[MT_MAX_EXPERTS];         // an expert's first entry of fc2
  uint16_t entries[MT_MAX_EXPERTS];     // expert and (from bit 8 on) part of its tokens, see Entry; each has a token's pick, so there are at most 256
  uint16_t ahead1[MT_MAX_EXPERTS + 1], ahead2[MT_MAX_EXPERTS + 1];     // time of a step of fc1 in all active experts ahead, of fc2 in all entries, see step_time
  alignas(16) uint32_t tokens[MT_MAX_EXPERTS];     // its tokens, a bit each
  uint8_t slot[MT_MAX_EXPERTS][MT_MAX_TOKENS];     // which pick of its tokens it is
  uint8_t who[MT_MAX_EXPERTS][MT_MAX_TOKENS];      // its tokens one behind the other
  uint8_t sel[MT_MAX_TOKENS][MT_MAX_K];
  float gate[MT_MAX_TOKENS][MT_MAX_K];
  float undo1[MT_MAX_TOKENS];           // what the sums over staged rows are short of: of fc1's tokens, of fc2's last four entries
  float undo2[4][MT_MAX_TOKENS];
};

// A warp selects the k largest logits of token t, ties to the lower expert, and their softmax
__device__ __forceinline__ void select_token(const TokensParams& p, TokensShared& s, int t, int lane) {
  uint32_t key[MT_MAX_EXPERTS / 32];
#pragma unroll
  for (int i = 0; i < MT_MAX_EXPERTS / 32; ++i) {
    const int e = lane + 32 * i;
    key[i] = e < p.E ? sel_float_key(__ldcg(p.logits + t * p.E + e)) : 0u;
  }
  uint32_t mine = 0u;                   // lane j's: the j-th largest and its expert
  int expert = 0;
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = key[0];
    int at = lane;
#pragma unroll
    for (int i = 1; i < MT_MAX_EXPERTS / 32; ++i)
      if (32 * i < p.E && key[i] > best) { best = key[i]; at = lane + 32 * i; }
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
    const int e = __reduce_min_sync(0xFFFFFFFFu, best == top ? at : MT_MAX_EXPERTS);
#pragma unroll
    for (int i = 0; i < MT_MAX_EXPERTS / 32; ++i)
      if (32 * i < p.E && lane + 32 * i == e) key[i] = 0u;
    if (lane == j) { mine = top; expert = e; }
  }
  const float first = sel_key_float(__shfl_sync(0xFFFFFFFFu, mine, 0)), w = lane < p.k ? expf(sel_key_float(mine) - first) : 0.0f;
  float sum = w;
#pragma unroll
  for (int o = MT_MAX_K / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane < p.k) {
    s.sel[t][lane] = (uint8_t)expert;
    atomicOr(&s.tokens[expert], 1u << t);
    s.gate[t][lane] = __fdiv_rn(w, sum);
  }
}

// staged token column col, eight k from 8 * k8 on
__device__ __forceinline__ uint32_t tok_at(uint32_t toks, int nblk, int col, int k8) {
  return toks + (uint32_t)((((k8 >> 2) * nblk + (col >> 3)) * 8 + (col & 7)) * 64 + (k8 & 3) * 16);
}
// token t as a column of fc1, by a warp: chunks of 256 k, six of them on their way at a time
__device__ __forceinline__ void stage_x(const TokensParams& p, TokensShared& s, int nblk, uint32_t toks, int t) {
  const int lane = threadIdx.x & 31, end = ((p.d + 127) >> 7) * 16;
  const int ex = row_exponent(__ldcg(p.xmax + t));
  const float scale = pow2(13 - ex);
  for (int k0 = lane; k0 < end; k0 += 6 * 32) {
    uint4 raw[6];
#pragma unroll
    for (int u = 0; u < 6; ++u) {
      const int k8 = k0 + u * 32;
      raw[u] = make_uint4(0, 0, 0, 0);
      if (k8 * 8 < p.d) raw[u] = *reinterpret_cast<const uint4*>((const uint16_t*)p.x + t * p.ld_x + k8 * 8);
    }
#pragma unroll
    for (int u = 0; u < 6; ++u) {
      const int k8 = k0 + u * 32;
      if (k8 >= end) break;
      const uint16_t* e = reinterpret_cast<const uint16_t*>(&raw[u]);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = (p.x_dtype == MOE_F16 ? __half2float(__ushort_as_half(e[j])) : __uint_as_float((uint32_t)e[j] << 16)) * scale;
      sts128(tok_at(toks, nblk, t, k8), pack8(v));
    }
  }
  if (lane == 0) s.undo1[t] = pow2(ex - 13);
}
// fc2 has every hidden row in two columns, a term each.  An expert with more tokens than half of the columns is two entries of fc2: the weights of the second are
// read once more, mostly from L2 (with one term for the tokens of such experts a token's result hung on how many others had picked its expert, 2^-12
// of a hidden value in place of 2^-23).
struct Entry { int e, r0, n; };         // expert, first of its tokens, how many of them
template <int NBLK> __device__ __forceinline__ Entry entry_of(const TokensShared& s, int place) {
  const int v = s.entries[place], e = v & 255, r0 = (v >> 8) * 4 * NBLK;
  return {e, r0, min(__popc(s.tokens[e]) - r0, 4 * NBLK)};
}

// An entry's hidden rows as the columns of fc2, behind one another, their second terms behind the first: a warp takes 256 k of a row,
// two at a time
__device__ __forceinline__ void stage_h(const TokensParams& p, TokensShared& s, int nblk, uint32_t toks, const Entry& en, int KT2, int place, int warp) {
  const int lane = threadIdx.x & 31, n = en.n, e = en.e;
  const int chunks = (KT2 + 1) >> 1, total = n * chunks;
  for (int i0 = warp; i0 < total; i0 += 2 * MT_WARPS) {   // 256 k of a row by a warp, two at a time
    float4 raw[2][2];
    float mx[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = i0 + x * MT_WARPS, r = i / chunks, k8 = (i - r * chunks) * 32 + lane;
      raw[x][0] = raw[x][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      mx[x] = 0.0f;
      if (i < total) {
        const int t = s.who[e][en.r0 + r], entry = t * p.k + s.slot[e][t];
        mx[x] = __uint_as_float(__ldcg(p.hmax + entry));
        if (k8 * 8 < p.ff) {
          const float4* src = reinterpret_cast<const float4*>(p.h + (int64_t)entry * p.ff + k8 * 8);
          raw[x][0] = __ldcg(src);
          raw[x][1] = __ldcg(src + 1);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = i0 + x * MT_WARPS, r = i / chunks, k8 = (i - r * chunks) * 32 + lane;
      if (i >= total || k8 >= KT2 * 16) continue;
      const int ex = row_exponent(mx[x]);
      float v[8] = {raw[x][0].x, raw[x][0].y, raw[x][0].z, raw[x][0].w, raw[x][1].x, raw[x][1].y, raw[x][1].z, raw[x][1].w}, w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] *= pow2(13 - ex);
        const float left = v[j] - __half2float(__float2half_rn(v[j]));     // (infinities and NaN are the first term's)
        w[j] = isfinite(left) ? left : 0.0f;
      }
      sts128(tok_at(toks, nblk, r, k8), pack8(v));
      sts128(tok_at(toks, nblk, n + r, k8), pack8(w));
      if (k8 == 0) s.undo2[place][r] = pow2(ex - 13);
    }
  }
}

// What a stage of `columns` columns takes the tensor-core loop, relative to others: the second block of eight costs half as much as everything else.  (Dealt out
// evenly, 13 tokens of 64 experts, k = 8, took 71 us in place of 66: the last CTA came 8 us behind the mean.)
__device__ __forceinline__ uint32_t step_time(int columns, int nblk) { return nblk == 1 ? 1u : columns > 8 ? 3u : 2u; }
// Steps of a product, `per` an expert or entry, are dealt out to CTAs by that time.  The CTA of a step: where the time ahead of it falls.
template <int NBLK>
__device__ __forceinline__ int cta_of(const uint16_t* aheads, int step, int place, int per, int total, int G) {
  if (NBLK == 1) return step * G / total;
  const int ahead = aheads[place], each = aheads[place + 1] - ahead;
  return (ahead * per + (step - place * per) * each) * G / total;
}
// The first step of CTA c, by a warp: cta_of is c or more from there on
template <int NBLK>
__device__ __forceinline__ int first_step(const uint16_t* aheads, int places, int c, int per, int total, int G, const Div& by_ctas) {
  const int time = (total * c + G - 1) / by_ctas;
  if (NBLK == 1) return time;
  int place = -1;                       // the last one that begins at that time or before
#pragma unroll
  for (int i = 0; i < MT_MAX_EXPERTS / 32; ++i) {
    const int a = i * 32 + (threadIdx.x & 31);
    if (i * 32 < places) place += __popc(__ballot_sync(0xFFFFFFFFu, a < places && aheads[a] * per <= time));
  }
  const int ahead = aheads[place], each = aheads[place + 1] - ahead;
  return place * per + (time - ahead * per + each - 1) / each;
}

template <int NBLK>                     // blocks of eight token columns
__global__ void __launch_bounds__(MT_THREADS, 1) moe_tokens_kernel(const TokensParams p, const __grid_constant__ TokensMaps maps) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 127) & ~(uintptr_t)127);
  __shared__ TokensShared s;
  __shared__ __align__(16) float s_red[2][MT_SHARES][8 * NBLK * MT_RED_LD];      // [team][share of k][column][row]
  const uint32_t ring = smem_u32(smem), toks = ring + (uint32_t)(p.stages * MT_STAGE_BYTES);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;     // warp-uniform for the compiler
  auto FULL = [&](int i) { return smem_u32(&s.full[i]); };
  auto EMPTY = [&](int i) { return smem_u32(&s.empty[i]); };
  auto SUMS = [&](int i) { return smem_u32(&s.sums[i]); };
  auto TAKEN = [&](int i) { return smem_u32(&s.taken[i]); };
  const Ctl ctl{&s.abort, p.status};

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(FULL(i), 1);
      mbar_init(EMPTY(i), MT_WARPS / 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(SUMS(i), MT_WARPS / 2);
      mbar_init(TAKEN(i), MT_EPILOGUE / 32);
    }
    s.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < MT_MAX_EXPERTS) s.tokens[threadIdx.x] = 0;
  __syncthreads();
  // Half of the consumers stage the tokens while the others select; the weights are on their way before the tokens are there.
  if (warp >= MT_WARPS / 2 && warp < MT_WARPS) {
    for (int t = warp - MT_WARPS / 2; t < p.T; t += MT_WARPS / 2) stage_x(p, s, NBLK, toks, t);
  } else {
    constexpr int OTHERS = MT_THREADS - MT_CONSUMERS / 2;
    if (warp < MT_WARPS / 2)
      for (int t = warp; t < p.T; t += MT_WARPS / 2) select_token(p, s, t, lane);
    bar_sync(3, OTHERS);
    if (warp == MT_WARPS) {             // the lists of active experts and of fc2's entries, eight experts a lane; fc1's figures in low halves, fc2's in high ones
      constexpr int HALF = 4 * NBLK;    // tokens of an entry
      uint32_t takes[8], on = 0, time = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = __popc(s.tokens[lane * 8 + i]);
        takes[i] = n ? step_time(n, NBLK) | (step_time(2 * min(n, HALF), NBLK) + (n > HALF ? step_time(2 * (n - HALF), NBLK) : 0u)) << 16 : 0u;
        time += takes[i];
        on += n ? (n > HALF ? 0x20001u : 0x10001u) : 0u;
      }
      uint32_t at = on, ahead = time;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t q = __shfl_up_sync(0xFFFFFFFFu, at, o), w = __shfl_up_sync(0xFFFFFFFFu, ahead, o);
        if (lane >= o) { at += q; ahead += w; }
      }
      if (lane == 31) {
        s.n_active = (int)(at & 0xFFFFu);
        s.n_entries = (int)(at >> 16);
        s.ahead1[at & 0xFFFFu] = (uint16_t)ahead;
        s.ahead2[at >> 16] = (uint16_t)(ahead >> 16);
      }
      at -= on;
      ahead -= time;
      int a1 = (int)(at & 0xFFFFu), a2 = (int)(at >> 16);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (takes[i]) {
          const int e = lane * 8 + i;
          s.act[a1] = (uint8_t)e;
          s.ahead1[a1] = (uint16_t)ahead;
          ++a1;
          s.from[e] = (uint8_t)a2;
          s.entries[a2] = (uint16_t)e;
          s.ahead2[a2] = (uint16_t)(ahead >> 16);
          ++a2;
          if (__popc(s.tokens[e]) > HALF) {
            s.entries[a2] = (uint16_t)(e | 256);
            s.ahead2[a2] = (uint16_t)((ahead >> 16) + step_time(2 * HALF, NBLK));
            ++a2;
          }
          ahead += takes[i];
        }
    } else if (threadIdx.x < p.T * p.k) {
      const int t = threadIdx.x / p.k, j = threadIdx.x - t * p.k, e = s.sel[t][j];
      s.slot[e][t] = (uint8_t)j;
      s.who[e][__popc(s.tokens[e] & ((1u << t) - 1u))] = (uint8_t)t;
    }
    bar_sync(3, OTHERS);
  }
  if (warp < MT_WARPS) bar_sync(1, MT_CONSUMERS);

  const int A = s.n_active, A2 = s.n_entries, G = gridDim.x, c = blockIdx.x;
  const int KT1 = (p.d + 127) >> 7, KT2 = (p.ff + 127) >> 7, KS1 = (KT1 + MT_STAGE_KT - 1) / MT_STAGE_KT, KS2 = (KT2 + MT_STAGE_KT - 1) / MT_STAGE_KT;
  const int NB1 = 2 * p.ff / MT_UNIT, NB2 = p.d / MT_UNIT, NT1 = (2 * p.ff + 127) >> 7, NT2 = (p.d + 127) >> 7;
  const int U1 = A * NB1;
  const int time1 = s.ahead1[A] * NB1, time2 = s.ahead2[A2] * NB2 * KS2;      // (times the CTAs below 2^26: the widths' limits)
  const int u_begin = first_step<NBLK>(s.ahead1, A, c, NB1, time1, G, p.by_ctas), u_end = c + 1 == G ? U1 : first_step<NBLK>(s.ahead1, A, c + 1, NB1, time1, G, p.by_ctas);
  const int s_begin = first_step<NBLK>(s.ahead2, A2, c, NB2 * KS2, time2, G, p.by_ctas);
  const int s_end = c + 1 == G ? A2 * NB2 * KS2 : first_step<NBLK>(s.ahead2, A2, c + 1, NB2 * KS2, time2, G, p.by_ctas);
  const int first2 = s_begin / p.by_steps2, n1 = u_end - u_begin, n2 = s_end > s_begin ? (s_end - 1) / p.by_steps2 - first2 + 1 : 0;      // units here

  if (warp == MT_BOTH / 32) {
    // ================================= weights =================================================================
    // the warp goes through the loop as a whole and elects a lane at each instruction: a thread by itself took longer to issue a stage's copies
    // than they take from HBM
    // Units go to the two teams in turn, each of which has half of the ring for itself.
    const int half = p.stages / 2;
    int ri[2] = {0, 0};
    uint32_t rp[2] = {1, 1};
    bool ok = true;
    auto stage = [&](int team, const CUtensorMap* v, const CUtensorMap* sc, uint32_t bytes, int nb, int tile) {
      const int at = team * half + (team ? ri[1] : ri[0]);
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(EMPTY(at), team ? rp[1] : rp[0], ctl, 1001));
      if (!ok) return;
      const uint32_t dst = ring + (uint32_t)(at * MT_STAGE_BYTES);
      elect_expect_tx(FULL(at), bytes);
      elect_tile_2d(dst, v, (nb & 3) * 128, tile * 4, FULL(at));
      elect_tile_2d(dst + MT_STAGE_VALUES, sc, (nb & 3) * 32, tile, FULL(at));
      if (team) { if (++ri[1] == half) { ri[1] = 0; rp[1] ^= 1u; } }
      else { if (++ri[0] == half) { ri[0] = 0; rp[0] ^= 1u; } }
    };
    int m = 0;
    // units [from, from + units) of a product, their stages from js0 in the first to js1 in the last
    auto product = [&](auto expert, const CUtensorMap* v, const CUtensorMap* sc, const CUtensorMap* vt, const CUtensorMap* st, int NB, const Div& by, int NT, int KT, int KS, int from,
                       int units, int js0, int js1) {
      const uint32_t whole = MT_STAGE_KT * MT_UNIT * 68, tail = (uint32_t)((KT - (KS - 1) * MT_STAGE_KT) * MT_UNIT * 68);
      int place = from / by, nb = from - place * NB;
#pragma unroll 1
      for (int i = 0; i < units && ok; ++i, ++m) {
        const int tile = (expert(place) * NT + (nb >> 2)) * KT, end = i + 1 == units ? js1 : KS;
#pragma unroll 1
        for (int js = i == 0 ? js0 : 0; js < end && ok; ++js) {
          if (js < KS - 1) stage(m & 1, v, sc, whole, nb, tile + js * MT_STAGE_KT);
          else stage(m & 1, vt, st, tail, nb, tile + js * MT_STAGE_KT);
        }
        if (++nb == NB) { nb = 0; ++place; }
      }
    };
    product([&](int at) { return (int)s.act[at]; }, &maps.v1, &maps.s1, &maps.v1t, &maps.s1t, NB1, p.by_units1, NT1, KT1, KS1, u_begin, n1, 0, KS1);
    product([&](int at) { return s.entries[at] & 255; }, &maps.v2, &maps.s2, &maps.v2t, &maps.s2t, NB2, p.by_units2, NT2, KT2, KS2, first2, n2, s_begin - first2 * KS2, s_end - (first2 + n2 - 1) * KS2);
    if (!ok) __nanosleep(500000);                             // copies in flight land before the block's shared memory goes
    return;
  }

  if (warp >= MT_WARPS) {
    // ================================= epilogue ================================================================
    const int tid = threadIdx.x - MT_CONSUMERS;
    int a = u_begin / p.by_units1, nb = u_begin - a * NB1;    // of the unit
    const int i = tid & 15;
    // the bias of a unit is asked for while the one before is at work: its way from memory is longer than a unit's
    float bias[2] = {0.0f, 0.0f};
    auto ask = [&](int a, int nb) {
      if (p.b1 && a < A) {
        const int64_t at = s.act[a] * p.ld_b1 + 2 * (nb * 16 + i);
        bias[0] = load_bias(p.b1, p.b1_dtype, at);
        bias[1] = load_bias(p.b1, p.b1_dtype, at + 1);
      }
    };
    ask(a, nb);
    constexpr int STEP = MT_EPILOGUE / 16, ROUNDS = (8 * NBLK + STEP - 1) / STEP;
    float top[ROUNDS];                                        // largest output of each of the thread's tokens in this expert's units so far
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) top[q] = 0.0f;
#pragma unroll 1
    for (int m = 0; m < n1; ++m) {
      const int e = s.act[a], n = __popc(s.tokens[e]), o = nb * 16 + i, was = nb;
      const float bg = bias[0], bl = bias[1];
      if (++nb == NB1) { nb = 0; ++a; }
      ask(a, nb);
      mbar_wait_short(SUMS(m & 1), (m >> 1) & 1u, ctl, 1005);
      // sixteen outputs of a token by half a warp, MT_EPILOGUE / 16 tokens at a time
      const int r0 = tid >> 4, mine = (n - (tid >> 5 << 1) + STEP - 1) / STEP;       // rounds of this warp
      if (mine <= 0 && (tid & 31) == 0) mbar_arrive(TAKEN(m & 1));
#pragma unroll
      for (int q = 0; q < ROUNDS; ++q) {
        if (q >= mine) break;
        const int r = r0 + q * STEP;
        const bool live = r < n;
        const int t = s.who[e][live ? r : 0], entry = t * p.k + s.slot[e][t];
        float g = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < MT_SHARES; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(&s_red[m & 1][w][(live ? r : 0) * MT_RED_LD + 2 * i]);
          g += v.x;
          l += v.y;
        }
        if (q + 1 == mine) {                                  // the buffer may be filled again
          __syncwarp();
          if ((tid & 31) == 0) mbar_arrive(TAKEN(m & 1));
        }
        g = fmaf(settle(g, p.s1, e, NT1, KT1, 2 * o), s.undo1[t], bg);
        l = fmaf(settle(l, p.s1, e, NT1, KT1, 2 * o + 1), s.undo1[t], bl);
        if (p.has_limit) {
          g = min_nan(g, p.limit);
          l = max_nan(min_nan(l, p.limit), -p.limit);
        }
        const float sg = __fdividef(g, 1.0f + gemm_ex2(-p.alpha * g * 1.4426950408889634f)), v = fmaf(sg, l, sg);
        if (live) __stcg(p.h + (int64_t)entry * p.ff + o, v);
        top[q] = fmaxf(top[q], fabsf(v) < __int_as_float(0x7F800000) ? fabsf(v) : 0.0f);
      }
      if (m + 1 == n1 || nb == 0) {                           // the last of this expert's units here
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) {
          if (q >= mine) break;
#pragma unroll
          for (int x = 8; x >= 1; x >>= 1) top[q] = fmaxf(top[q], __shfl_xor_sync(0xFFFFFFFFu, top[q], x));
          const int r = r0 + q * STEP;
          if (r < n && i == 0) {
            const int t = s.who[e][r];
            atomicMax(p.hmax + t * p.k + s.slot[e][t], __float_as_uint(top[q]));
          }
          top[q] = 0.0f;
        }
        bar_sync(2, MT_EPILOGUE);
        if (tid == 0) {
          __threadfence();
          atomicAdd(p.done1 + e, min(was + 1, m + 1));
        }
      }
    }
    int have = -1, changes = -1;
#pragma unroll 1
    for (int m = n1; m < n1 + n2; ++m) {
      const int u = first2 + m - n1, place = u / p.by_units2, lane_row = tid & 31;
      const Entry en = entry_of<NBLK>(s, place);
      const int e = en.e, n = en.n;
      if (place != have) { have = place; ++changes; }
      mbar_wait_short(SUMS(m & 1), (m >> 1) & 1u, ctl, 1005);
      for (int r = tid >> 5; r < n; r += MT_EPILOGUE / 32) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < MT_SHARES; ++w) v += s_red[m & 1][w][r * MT_RED_LD + lane_row];
#pragma unroll
        for (int w = 0; w < MT_SHARES; ++w) v += s_red[m & 1][w][(n + r) * MT_RED_LD + lane_row];
        __stcg(p.part + ((int64_t)(u + c) * p.T + r) * MT_UNIT + lane_row, settle(v, p.s2, e, NT2, KT2, (u - place * NB2) * MT_UNIT + lane_row) * s.undo2[changes & 3][r]);
      }
      __syncwarp();
      if ((tid & 31) == 0) mbar_arrive(TAKEN(m & 1));
    }
    bar_sync(2, MT_EPILOGUE);
    for (int i = tid; i < n2; i += MT_EPILOGUE) {
      const int u = first2 + i;
      __threadfence();
      atomicAdd(p.done2 + (u - u / p.by_units2 * NB2), min(s_end, (u + 1) * KS2) - max(s_begin, u * KS2));
    }
    return;
  }

  // ================================= consumers =================================================================
  const int wk = warp & 3, slab = (warp >> 2) & 1, team = warp >> 3, half = p.stages / 2, qrow = lane >> 2, c4 = lane & 3, tid = threadIdx.x;
  // (where a wait runs out, this and the following ones return, the rest is gone through and its results are void)
  int ri = 0;                           // place in the team's half of the ring
  uint32_t rp = 0;
  float acc[NBLK][4];
  // This warp's tiles of a stage, 16 rows x 128 k each, times NB blocks of columns, k from `xt` on; `left`: k tiles from the stage on.  Every load of a
  // tile goes ahead of its arithmetic: what bounds the loop is the number of instructions and the way of one warp through a stage.
  const uint32_t my_ring = ring + (uint32_t)(team * half * MT_STAGE_BYTES);
  // (the eight rows of a matrix that the lane addresses: rows 0-7 and 8-15 of two groups of 32 k)
  const uint32_t my_w = my_ring + (uint32_t)(wk * 2048 + (lane >> 4) * 512 + (slab * 16 + (lane & 15)) * 16), my_s = my_ring + (uint32_t)(MT_STAGE_VALUES + wk * 128 + (slab * 16 + qrow) * 4);
  const uint32_t my_x = toks + (uint32_t)(wk * 4 * NBLK * 512 + c4 * 16);
  uint32_t col[NBLK];                   // where the lane's columns are
  auto multiply = [&](auto nb_tag, int left, uint32_t xt) {
    constexpr int NB = decltype(nb_tag)::value;
    const int at = team * half + ri;
    mbar_wait_short(FULL(at), rp, ctl, 1002);
    uint32_t wt = my_w + (uint32_t)(ri * MT_STAGE_BYTES), sc = my_s + (uint32_t)(ri * MT_STAGE_BYTES);
#pragma unroll
    for (int h = 0; h < MT_STAGE_KT / MT_SHARES; ++h) {
      if (wk + h * MT_SHARES < left) {
        const uint32_t sl = lds32(sc), sh = lds32(sc + 32);
        uint32_t wl[4], wh[4];
        uint4 xb[4][NB];
        ldmatrix_x4(wt, wl[0], wh[0], wl[1], wh[1]);
        ldmatrix_x4(wt + 1024, wl[2], wh[2], wl[3], wh[3]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
          for (int b = 0; b < NB; ++b) xb[g][b] = lds128(xt + col[b] + (uint32_t)(g * NBLK * 512));
        }
        float fl[4], fh[4];
        e8m0_word(sl, fl);
        e8m0_word(sh, fh);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t lo[4], hi[4];
          e2m1_word(wl[g], lo);
          e2m1_word(wh[g], hi);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float dd[4];
            mma_f16_zero(dd, lo[0], hi[0], lo[1], hi[1], xb[g][b].x, xb[g][b].y);
            mma_f16(dd, lo[2], hi[2], lo[3], hi[3], xb[g][b].z, xb[g][b].w);
            acc[b][0] = fmaf(fl[g], dd[0], acc[b][0]);
            acc[b][1] = fmaf(fl[g], dd[1], acc[b][1]);
            acc[b][2] = fmaf(fh[g], dd[2], acc[b][2]);
            acc[b][3] = fmaf(fh[g], dd[3], acc[b][3]);
          }
        }
      }
      wt += MT_SHARES * 2048;
      sc += MT_SHARES * 128;
      xt += MT_SHARES * 4 * NBLK * 512;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(EMPTY(at));
    if (++ri == half) { ri = 0; rp ^= 1u; }
  };

  // ---- all units, fc1's and fc2's ----
  int have = -1, changes = -1;          // entry whose rows of fc2 are staged
  int n_blocks = 1;                     // of the columns
  int place = u_begin / p.by_units1, rest = u_begin - place * NB1;   // the unit's active expert or entry, its place among that one's units
#pragma unroll 1
  for (int m = 0; m < n1 + n2; ++m, ++rest) {
    const bool one = m < n1;
    if (m == n1) { place = first2 / p.by_units2; rest = first2 - place * NB2; }
    if (rest == (one ? NB1 : NB2)) { rest = 0; ++place; }
    const int KT = one ? KT1 : KT2;
    const int js0 = m == n1 ? s_begin - first2 * KS2 : 0, js1 = one ? KS1 : m + 1 == n1 + n2 ? s_end - (first2 + n2 - 1) * KS2 : KS2;
    if (one) {
      const int e = s.act[place];
      n_blocks = __popc(s.tokens[e]) > 8 ? 2 : 1;             // fc1's columns are the expert's tokens among those of the batch
#pragma unroll
      for (int b = 0; b < NBLK; ++b) {
        const int t = s.who[e][b * 8 + qrow] & (MT_MAX_TOKENS - 1);      // (any column stands in for one without a token)
        col[b] = (uint32_t)((t >> 3) * 512 + (t & 7) * 64) & (uint32_t)(NBLK * 512 - 1);
      }
    } else if (place != have) {
      const Entry en = entry_of<NBLK>(s, place);
      if (tid == 0) wait_count(p.done1 + en.e, NB1, ctl, 1003);
      bar_sync(1, MT_CONSUMERS);                              // fc1's rows are there, and the staged ones have been read
      ++changes;
      stage_h(p, s, NBLK, toks, en, KT2, changes & 3, warp);
      bar_sync(1, MT_CONSUMERS);
      have = place;
      n_blocks = 2 * en.n > 8 ? 2 : 1;
#pragma unroll
      for (int b = 0; b < NBLK; ++b) col[b] = (uint32_t)(b * 512 + qrow * 64);
    }
    if ((m & 1) != team) continue;                            // the other team's
#pragma unroll
    for (int b = 0; b < NBLK; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[b][j] = 0.0f;
    uint32_t xt = my_x + (uint32_t)(js0 * MT_STAGE_KT * 4 * NBLK * 512);
    if (NBLK == 1 || n_blocks == 1) {
#pragma unroll 1
      for (int js = js0; js < js1; ++js, xt += MT_STAGE_KT * 4 * NBLK * 512)
        multiply(std::integral_constant<int, 1>(), KT - js * MT_STAGE_KT, xt);
    } else {
#pragma unroll 1
      for (int js = js0; js < js1; ++js, xt += MT_STAGE_KT * 4 * NBLK * 512)
        multiply(std::integral_constant<int, NBLK>(), KT - js * MT_STAGE_KT, xt);
    }
    // the warp's share of the unit's sums goes to the epilogue; a buffer per team
    if (m >= 2) mbar_wait_short(TAKEN(m & 1), ((m >> 1) & 1u) ^ 1u, ctl, 1006);
#pragma unroll
    for (int b = 0; b < NBLK; ++b)
      if (b < n_blocks) {
        float* at = &s_red[m & 1][wk][(b * 8 + c4 * 2) * MT_RED_LD + slab * 16 + qrow];
        at[0] = acc[b][0];
        at[MT_RED_LD] = acc[b][1];
        at[8] = acc[b][2];
        at[MT_RED_LD + 8] = acc[b][3];
      }
    __syncwarp();
    if (lane == 0) mbar_arrive(SUMS(m & 1));
  }

  // ---- the selected experts' sums meet: a warp takes 32 outputs of a token as soon as all of their stages are done ----
  for (int i = warp * G + c; i < NB2 * p.T; i += MT_WARPS * G) {
    const int t = i / p.by_units2, nb = i - t * NB2, o = nb * MT_UNIT + lane;
    float y = 0.0f;
    for (int j0 = 0; j0 < p.k; j0 += 4) {
      float v[4], b[4];
      int c0[4], c1[4];
      const float* part[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        b[x] = 0.0f;
        c0[x] = c1[x] = 0;
        part[x] = nullptr;
        if (j0 + x < p.k) {
          const int e = s.sel[t][j0 + x], all = __popc(s.tokens[e] & ((1u << t) - 1u)), second = all >= 4 * NBLK ? 1 : 0, r = all - second * 4 * NBLK;
          const int place = s.from[e] + second, u = place * NB2 + nb;
          // the CTAs whose ranges the unit's first and last stage are in
          c0[x] = cta_of<NBLK>(s.ahead2, u * KS2, place, NB2 * KS2, time2, G);
          c1[x] = cta_of<NBLK>(s.ahead2, u * KS2 + KS2 - 1, place, NB2 * KS2, time2, G);
          part[x] = p.part + ((int64_t)u * p.T + r) * MT_UNIT + lane;
          if (p.b2) b[x] = load_bias(p.b2, p.b2_dtype, e * p.ld_b2 + o);
        }
      }
      wait_count(p.done2 + nb, A2 * KS2, ctl, 1004);
      __syncwarp();
      // the first part and the last, most often all there are, side by side
      float last[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = j0 + x < p.k ? __ldcg(part[x] + (int64_t)c0[x] * p.T * MT_UNIT) : 0.0f;
        last[x] = c1[x] > c0[x] ? __ldcg(part[x] + (int64_t)c1[x] * p.T * MT_UNIT) : 0.0f;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (j0 + x >= p.k) break;
        if (c1[x] > c0[x] + 1) {
          const int e = s.sel[t][j0 + x], place = s.from[e] + (__popc(s.tokens[e] & ((1u << t) - 1u)) >= 4 * NBLK ? 1 : 0);
          for (int q = 1, was = c0[x]; q < KS2 - 1; ++q) {
            const int cc = cta_of<NBLK>(s.ahead2, (place * NB2 + nb) * KS2 + q, place, NB2 * KS2, time2, G);
            if (cc != was && cc != c1[x]) v[x] += __ldcg(part[x] + (int64_t)cc * p.T * MT_UNIT);
            was = cc;
          }
        }
        v[x] += last[x];
        y = fmaf(s.gate[t][j0 + x], v[x] + b[x], y);
      }
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
  const int64_t n = (int64_t)a.T * a.k, entries = n < 2 * a.E ? n : 2 * a.E;       // of fc2: two of an expert at most, each of a pick at least
  w.counters = take(3 * MT_COUNTERS * 4);
  w.logits = take((size_t)a.T * a.E * 4);
  w.xmax = take((size_t)a.T * 4);
  w.h = take((size_t)(n * a.ff) * 4);
  w.part = take((size_t)((entries * (a.d / MT_UNIT) + moe_sm_count()) * a.T) * MT_UNIT * 4);
  w.bytes = at;
  return w;
}

// the shared memory that is left for the ring, whole stages
constexpr int MT_SMEM = 232448;
template <int NBLK> constexpr int mt_static_smem() { return (int)(sizeof(TokensShared) + 2 * MT_SHARES * 8 * NBLK * MT_RED_LD * 4) + 64; }

// four stages at the widest that two blocks of columns take: with two, one a team, a layer of 4096 x 2880 and 16 tokens took 158 us in place of 105
static_assert(MT_SMEM - mt_static_smem<2>() - 128 - 4096 / 128 * 4 * 512 * 2 >= 4 * MT_STAGE_BYTES, "TokensShared has outgrown its room");

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
  MOE_CHECK_CUDA(launch_pdl(moe_tokens_router_kernel<TX, TP>, dim3((unsigned)(a.E + rows), (unsigned)cdiv64(a.T, 8)), dim3(MT_ROUTER_THREADS), (size_t)0, st, (const TX*)a.x, a.ld_x, \
                            a.T, a.d, (const __nv_bfloat16*)a.wg_t, a.ld_wg, a.bg, a.bg_dtype, a.E, logits, xmax, counters))
  const int rows = a.T < 8 ? a.T : 8;
  if (a.T <= 1) MT_ROUTER(1);
  else if (a.T <= 2) MT_ROUTER(2);
  else if (a.T <= 4) MT_ROUTER(4);
  else MT_ROUTER(8);
#undef MT_ROUTER
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <int NBLK> int mt_launch(TokensParams& p, const TokensMaps& maps, cudaStream_t st) {
  const int width = p.d > p.ff ? p.d : p.ff;
  p.tok_bytes = (int)cdiv64(width, 128) * 4 * 512 * NBLK;
  const int left = MT_SMEM - mt_static_smem<NBLK>() - 128 - p.tok_bytes;
  p.stages = (left / MT_STAGE_BYTES < MT_MAX_STAGES ? left / MT_STAGE_BYTES : MT_MAX_STAGES) & ~1;      // half for each team
  if (p.stages < 2) {
    moe_set_error("moe_layer_tokens: no shared memory left for weights (d = %d, ff = %d)", p.d, p.ff);
    return MOE_ERR_UNSUPPORTED;
  }
  const int smem = p.tok_bytes + p.stages * MT_STAGE_BYTES + 128;
  const auto div = [](int d) { return Div{(uint32_t)d, (1ull << 40) / (uint64_t)d + 1}; };
  p.by_ctas = div(moe_sm_count());
  p.by_units1 = div(2 * p.ff / MT_UNIT);
  p.by_units2 = div(p.d / MT_UNIT);
  p.by_steps2 = div((int)cdiv64(cdiv64(p.ff, 128), MT_STAGE_KT));
  // once per device (a microsecond of every call otherwise)
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  MOE_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev >= 64 || !(allowed.load(std::memory_order_acquire) & bit)) {
    MOE_CHECK_CUDA(cudaFuncSetAttribute(moe_tokens_kernel<NBLK>, cudaFuncAttributeMaxDynamicSharedMemorySize, MT_SMEM - mt_static_smem<NBLK>()));
    if (dev < 64) allowed.fetch_or(bit, std::memory_order_release);
  }
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
  p.s1 = (const uint8_t*)a.w1_scale; p.s2 = (const uint8_t*)a.w2_scale;
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
