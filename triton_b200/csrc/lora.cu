// A projection that all requests share, with each request's own low-rank adapter beside it:
//     y_t = x_t W + bias + s_a (x_t A_a) B_a,   a = indx[t]; no second part where indx[t] is no adapter.
//
// An adapter's ranks go in pieces of 16, so adapters of different ranks lie behind one another: A as rows of K, B as tiles in the order the tensor core
// takes them (lora_adapters layout in the header).  Two kernels:
//  1. lora_shrink_kernel: t = s_a x A_a for every token, fp32, into the workspace.  A piece of an adapter (16 rows of A) times 8 or 64 tokens is what a CTA
//     has, on mma.sync with operands straight from global memory: there are 16 ranks, too few for a tcgen05 operand of 128 rows, and at single
//     tokens reading A is all there is to do.
//  2. the product: W's tiles and x's through a ring by TMA, tcgen05.mma.kind::f16 into fp32 in tensor memory; then, into the same accumulator, one MMA per
//     piece and term: B's tile times the tokens' t, zero for the tokens of other adapters, so that a block of tokens may hold any mixture.  t enters in bf16
//     terms, two (17 bits of it) for bf16, three for fp16, whose B is two bf16 parts then: see "pieces as MMA operands".
// The second has two forms: lora_stream_kernel for few tokens, whose adapters' part runs on CUDA cores beside the product (one token's first part too), and
// lora_pair_kernel for many, as above.
// Measured, K = 2880, N = 5120, shrink + product: 1 token 9.3 us of one launch (29.7 MB at 3.2 TB/s; its start, the first loads and the meeting of the shares of
// k are half), 64 tokens with an adapter each of 1 to 64 ranks 7 + 20 (55 MB), 300 tokens 6.4 + 23, 8192 tokens 18 + 213: 231 one call at a time
// (1.05 PFLOP/s; the product's kernel by itself 1.13), 258 in a long run, whose clock the power limit takes to 1.6 GHz (0.94).  What bounds the last: a CTA takes in 48 KB for 1024 cycles of MMA, and an SM some 32 B a cycle.
#include "gemm_pair_common.cuh"
#include <cuda_fp16.h>
#include <atomic>
#include <type_traits>

namespace {

constexpr int LR_PIECE = 16;                   // ranks of a piece
constexpr int LR_TILE_N = 128;                 // outputs of a weight tile
constexpr int LR_PIECE_BYTES = LR_TILE_N * LR_PIECE * 2;

struct LoraParams {
  const void* x; int64_t ld_x; int T, K, N, NP;        // NP: outputs rounded up to 128, rows of a piece of B
  const void* bias; int bias_dtype;
  const void* a; int64_t ld_a;
  const uint8_t* b;
  const int32_t* first; const float* scale; int n_adapters, max_pieces;
  const int32_t* ranks;                                // of every adapter, or NULL: whole pieces
  const int32_t* indx;
  float* t; int64_t ld_t; int t_parts; int64_t t_part_stride;     // shares of k whose sums make up t
  void* y; int64_t ld_y;
  int32_t* list; int list_tb;                          // of every block of list_tb tokens [LR_LIST]: how many adapters, how many pieces, the adapters
  int32_t* status;
};
constexpr int LR_MAX_PARTS = 4;
constexpr int LR_MAX_TB = 512, LR_LIST = LR_MAX_TB + 4;

// ---- shrink ----------------------------------------------------------------------------------------------------
template <typename T16> __device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T16) == 2 && std::is_same<T16, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int SH_WARPS = 8;

// Adapter of each of `rows` tokens from row0 on (-1: none, and for the rows past them) and the list of those that occur, in the order of their first
// token.  All threads of the block call; `idx` and `list`, ROWS each, and `table`, 4 ROWS, are in shared memory; behind a barrier, with one at the end.
// An adapter's first token is found through a hash table of 2 ROWS places, half of which stay free (every token with every one before it: 4 us of 512).
template <int ROWS>
__device__ __forceinline__ void adapters_of(const LoraParams& p, int64_t row0, int rows, int* idx, int* list, int* table, int* count) {
  constexpr int SLOTS = 2 * ROWS, MINE = (ROWS + SH_WARPS * 32 - 1) / (SH_WARPS * 32);
  int *key = table, *least = table + SLOTS;
  for (int i = threadIdx.x; i < SLOTS; i += SH_WARPS * 32) { key[i] = -1; least[i] = ROWS; }
  for (int r = threadIdx.x; r < ROWS; r += SH_WARPS * 32) {
    const int a = r < rows && p.indx ? p.indx[row0 + r] : -1;
    idx[r] = a >= 0 && a < p.n_adapters ? a : -1;
  }
  __syncthreads();
  int at[MINE];
#pragma unroll
  for (int m = 0; m < MINE; ++m) {
    const int r = threadIdx.x + m * SH_WARPS * 32, a = r < ROWS ? idx[r] : -1;
    at[m] = -1;
    if (a >= 0 && (r == 0 || idx[r - 1] != a)) {              // (most often runs)
      uint32_t h = (uint32_t)a * 2654435761u % SLOTS;
      for (;;) {
        const int was = atomicCAS(key + h, -1, a);
        if (was == -1 || was == a) break;
        h = (h + 1) % SLOTS;
      }
      atomicMin(least + h, r);
      at[m] = (int)h;
    }
  }
  __syncthreads();
  uint32_t fresh[MINE];                                       // of the warp's 32 tokens
#pragma unroll
  for (int m = 0; m < MINE; ++m) {
    const int r = threadIdx.x + m * SH_WARPS * 32;
    fresh[m] = __ballot_sync(0xFFFFFFFFu, at[m] >= 0 && least[at[m]] == r);
    if ((threadIdx.x & 31) == 0 && r < ROWS) key[r >> 5] = __popc(fresh[m]);      // (the keys have been read)
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MINE; ++m) {
    const int r = threadIdx.x + m * SH_WARPS * 32, lane = threadIdx.x & 31;
    int n = 0;
    if (r < ROWS)
      for (int i = 0; i < r >> 5; ++i) n += key[i];
    if ((fresh[m] >> lane) & 1u) list[n + __popc(fresh[m] & ((1u << lane) - 1u))] = idx[r];
    if (r == ROWS - 32) *count = n + __popc(fresh[m]);
  }
  __syncthreads();
}

// grid: (blocks of 8 NB tokens, pieces of an adapter, [the lists,] places in the list of the block's adapters x shares of k).  A block of threads has one
// adapter of its tokens (eights), or every `places`-th (sixty-fours), and splits k over its warps: what it takes is one or two trips to memory, and a warp
// with an adapter to itself took four times as many.  The blocks that take longest, the lists', come first, and those of later places, most of which find
// no adapter, last.
template <typename T16, int NB>
__global__ void __launch_bounds__(SH_WARPS * 32, NB == 1 ? 3 : 2) lora_shrink_kernel(const LoraParams p) {
  __shared__ int s_idx[8 * NB], s_list[8 * NB], s_table[NB == 1 ? 1 : 32 * NB], s_count;
  constexpr int SUM_WORDS = SH_WARPS * NB * 128, LIST_WORDS = 6 * LR_MAX_TB;
  __shared__ __align__(16) float s_words[SUM_WORDS > LIST_WORDS ? SUM_WORDS : LIST_WORDS];
  float (&s_sum)[SH_WARPS][NB][32][4] = *reinterpret_cast<float (*)[SH_WARPS][NB][32][4]>(s_words);
  pdl_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qrow = lane >> 2, c4 = lane & 3, lists = p.list_tb > 0 ? 1 : 0;
  if ((int)blockIdx.z < lists) {
    // the adapters of the product's blocks of tokens, for its kernel
    if (blockIdx.y == 0 && (int64_t)blockIdx.x * p.list_tb < p.T) {
      int *idx = reinterpret_cast<int*>(s_words), *list = idx + LR_MAX_TB;
      const int64_t from = (int64_t)blockIdx.x * p.list_tb;
      adapters_of<LR_MAX_TB>(p, from, (int)min((int64_t)p.list_tb, (int64_t)p.T - from), idx, list, list + LR_MAX_TB, &s_count);
      int32_t* out = p.list + (int64_t)blockIdx.x * LR_LIST;
      const int n = s_count;
      int total = 0;
      for (int i = threadIdx.x; i < n; i += SH_WARPS * 32) {
        const int a = list[i];
        out[2 + i] = a;
        total += p.first[a + 1] - p.first[a];
      }
      total = __reduce_add_sync(0xFFFFFFFFu, total);
      __syncthreads();
      if (threadIdx.x == 0) s_count = 0;
      __syncthreads();
      if (lane == 0) atomicAdd(&s_count, total);
      __syncthreads();
      if (threadIdx.x == 0) { out[0] = n; out[1] = s_count; }
    }
    return;
  }
  const int64_t row0 = (int64_t)blockIdx.x * (8 * NB);
  const int rows = (int)min((int64_t)(8 * NB), (int64_t)p.T - row0);
  const int z = blockIdx.z - lists, place = z / p.t_parts, part = z - place * p.t_parts, places = ((int)gridDim.z - lists) / p.t_parts;
  int count, only = -1;
  if constexpr (NB == 1) {                                    // every warp for itself: most blocks of threads find that there is nothing for them
    int a = lane < rows ? p.indx[row0 + lane] : -1;
    a = a >= 0 && a < p.n_adapters ? a : -1;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, a);
    uint32_t fresh = __ballot_sync(0xFFFFFFFFu, a >= 0 && __ffs(same) - 1 == lane);
    count = __popc(fresh);
    if (place >= count) return;
    for (int i = 0; i < place; ++i) fresh &= fresh - 1;
    only = __shfl_sync(0xFFFFFFFFu, a, __ffs(fresh) - 1);
    if (warp == 0 && lane < 8) s_idx[lane] = a;
  } else {
    adapters_of<8 * NB>(p, row0, rows, s_idx, s_list, s_table, &s_count);
    count = s_count;
  }
  const int K8 = (p.K + 7) & ~7, blocks = (K8 + 31) >> 5, b0 = blocks * part / p.t_parts, b1 = blocks * (part + 1) / p.t_parts;
  for (int l = place; l < count; l += places) {
    const int a = NB == 1 ? only : s_list[l], f = p.first[a];
    const float scale = p.scale[a];                           // (asked for here: behind the sums its trip to memory would be one more)
    const int ranks = p.ranks ? p.ranks[a] : LR_PIECE * p.max_pieces;
    if ((int)blockIdx.y >= p.first[a + 1] - f) continue;      // (uniform)
    const T16* ra = (const T16*)p.a + (int64_t)(f + blockIdx.y) * LR_PIECE * p.ld_a;
    float acc[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
    constexpr int UNROLL = NB == 1 ? 4 : 2;
    for (int b = b0 + warp; b < b1; b += UNROLL * SH_WARPS) {
      uint4 lo[UNROLL], hi[UNROLL], xv[UNROLL][NB];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int k = (b + u * SH_WARPS) * 32 + c4 * 8;       // a lane's eight consecutive k are its places in two MMAs
        const bool in = b + u * SH_WARPS < b1 && k < K8;
        lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
        if (in) {
          lo[u] = *reinterpret_cast<const uint4*>(ra + qrow * p.ld_a + k);
          hi[u] = *reinterpret_cast<const uint4*>(ra + (qrow + 8) * p.ld_a + k);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          xv[u][n] = make_uint4(0, 0, 0, 0);
          if (in && n * 8 + qrow < rows) xv[u][n] = *reinterpret_cast<const uint4*>((const T16*)p.x + (row0 + n * 8 + qrow) * p.ld_x + k);
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          mma_16816<T16>(acc[n], lo[u].x, hi[u].x, lo[u].y, hi[u].y, xv[u][n].x, xv[u][n].y);
          mma_16816<T16>(acc[n], lo[u].z, hi[u].z, lo[u].w, hi[u].w, xv[u][n].z, xv[u][n].w);
        }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) *reinterpret_cast<float4*>(s_sum[warp][n][lane]) = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    __syncthreads();
    for (int i = threadIdx.x; i < NB * 128; i += SH_WARPS * 32) {
      const int n = i >> 7, token = i >> 4, rank = i & 15;    // accumulator: rank rows, token columns
      const int ln = (rank & 7) * 4 + ((token & 7) >> 1), j = (rank >> 3) * 2 + (token & 1);
      if (s_idx[token] != a) continue;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < SH_WARPS; ++w) v += s_sum[w][n][ln][j];
      // A rank that the adapter does not have adds nothing: its row of zeros times an infinity would be NaN, and NaN times B's zeros too
      p.t[part * p.t_part_stride + (row0 + token) * p.ld_t + blockIdx.y * LR_PIECE + rank] = (int)blockIdx.y * LR_PIECE + rank < ranks ? v * scale : 0.0f;
    }
    __syncthreads();
  }
}

// ---- pieces as MMA operands --------------------------------------------------------------------------------------
// Operands of 16 k without swizzle: eight rows of 16 bytes are 128 bytes in a row, the two halves of k follow one another, then the next eight rows.
constexpr uint32_t PIECE_DESC_LO = (128u >> 4) << 16;                   // leading byte offset: between the halves of k
// (An address of a CTA in a cluster has its rank from bit 24 on, which in a descriptor would be part of the leading byte offset.)
__device__ __forceinline__ uint32_t piece_desc(uint32_t at) { return PIECE_DESC_LO | ((at & 0x3FFFFu) >> 4); }
constexpr uint32_t PIECE_DESC_HI = (256u >> 4) | (1u << 14);            // stride byte offset: between groups of eight rows; sm_100, no swizzle
__device__ __forceinline__ uint32_t lr_idesc(bool f16, int m, int n) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// A piece as operands.  bf16: B's tile, and t in two terms (17 bits of it, 2^-17 of a value: the result keeps 8).  fp16: its range ends at 65504 and its steps
// at 2^-24, t's do not, and an MMA's operands have one type.  So both go in as bf16, which has fp32's range: t in three terms, all of its 24 bits; a value of
// B, which has 11, in two tiles.  B's second tile times t's third term is left out, 2^-23 of a product.
template <typename T16> constexpr bool LR_F16 = std::is_same<T16, __half>::value;
constexpr int lr_tiles(bool f16) { return f16 ? 2 : 1; }
constexpr int lr_terms(bool f16) { return f16 ? 3 : 2; }
constexpr int lr_piece_bytes(bool f16, int tb) { return lr_tiles(f16) * LR_PIECE_BYTES + lr_terms(f16) * tb * 16; }     // of one CTA: half of the block's tokens

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat16 h[2] = {__float2bfloat16_rn(a), __float2bfloat16_rn(b)};
  return *reinterpret_cast<const uint32_t*>(h);
}
// what bf16 has of a value, rounded (two terms) or cut off (three: the rest of a sum of cut-off terms is exact); all of one that is not finite
template <bool CUT> __device__ __forceinline__ float bf16_term(float v) {
  return CUT && isfinite(v) ? __uint_as_float(__float_as_uint(v) & 0xFFFF0000u) : __bfloat162float(__float2bfloat16_rn(v));
}
// Eight fp16 values -> their two bf16 parts.  Both have the value's sign and, but for a zero, neither is zero, so that an infinite t times the two is infinite with that
// sign: where the leading eight bits are all there is, a step of them goes to the second part.
__device__ __forceinline__ void split_f16(const uint4& v, uint4& hi, uint4& lo) {
  const __half* e = reinterpret_cast<const __half*>(&v);
  uint32_t h[8], l[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = __half2float(e[j]);
    const uint32_t u = __float_as_uint(f);
    h[j] = (u & 0x7FFFFFFFu) == 0u ? u : (u & 0xFFFF0000u) - ((u & 0xFFFFu) == 0u ? 0x10000u : 0u);
    l[j] = __float_as_uint(f - __uint_as_float(h[j]));
  }
  hi = make_uint4(h[0] >> 16 | h[1], h[2] >> 16 | h[3], h[4] >> 16 | h[5], h[6] >> 16 | h[7]);
  lo = make_uint4(l[0] >> 16 | l[1], l[2] >> 16 | l[3], l[4] >> 16 | l[5], l[6] >> 16 | l[7]);
}
// Sixteen ranks of a token (`live`: it has this adapter) as row `at` of the operand: the first terms at dst, what each leaves `step` bytes on
template <typename T16>
__device__ __forceinline__ void write_piece_row(const LoraParams& p, bool live, int64_t token, int rank0, uint32_t dst, uint32_t step, int at) {
  constexpr int TERMS = lr_terms(LR_F16<T16>);
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.0f;
  if (live) {
    const float4* src = reinterpret_cast<const float4*>(p.t + token * p.ld_t + rank0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 q = src[i];
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
    for (int s = 1; s < p.t_parts; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 q = *(reinterpret_cast<const float4*>(p.t + s * p.t_part_stride + token * p.ld_t + rank0) + i);
        v[4 * i] += q.x; v[4 * i + 1] += q.y; v[4 * i + 2] += q.z; v[4 * i + 3] += q.w;
      }
  }
  const uint32_t to = dst + (uint32_t)((at >> 3) * 256 + (at & 7) * 16);
#pragma unroll
  for (int term = 0; term < TERMS; ++term) {
    float h[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      h[i] = bf16_term<TERMS == 3>(v[i]);
      const float d = v[i] - h[i];
      v[i] = isfinite(d) ? d : 0.0f;                          // infinities and NaN are the first term's
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sts128(to + (uint32_t)term * step + (uint32_t)i * 128u,
             make_uint4(pack_bf16(h[8 * i], h[8 * i + 1]), pack_bf16(h[8 * i + 2], h[8 * i + 3]), pack_bf16(h[8 * i + 4], h[8 * i + 5]), pack_bf16(h[8 * i + 6], h[8 * i + 7])));
  }
}

// whether the word at this place is zero in the first n CTAs of the cluster (a lane asks one of them: one after the other they took 2 us)
__device__ __forceinline__ bool cluster_fine(uint32_t at, int n) {
  uint32_t v = 0;
  const int lane = threadIdx.x & 31;
  if (lane < n)
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\tld.shared::cluster.u32 %0, [ra];\n\t}" : "=r"(v) : "r"(at), "r"(lane) : "memory");
  return __all_sync(0xFFFFFFFFu, v == 0);
}
// The shares of k of a cluster's CTAs meet, in their order: sums [token][128 outputs] at `at` in the shared memory of the CTAs step * r + base, r < S <=
// MOST.  Tokens t0 .. t1 of the block for outputs n0 on; four outputs a thread, U of those and all shares on their way at a time (one share after the other
// the sums of 300 tokens took 6 us, this way 3.8).
// (a thread's items there are a multiple of 32 apart, so its outputs are the same four: their biases are asked for before the CTAs wait for one another)
__device__ __forceinline__ void sums_bias(const LoraParams& p, int n0, float (&bias)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + (threadIdx.x & 31) * 4 + j;
    bias[j] = p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, n) : 0.0f;
  }
}
template <typename T16, int MOST, int U>
__device__ __forceinline__ void cluster_sums(const LoraParams& p, uint32_t at, int S, uint32_t step, uint32_t base, int64_t row0, int t0, int t1, int n0, const float (&bias)[4]) {
  const bool vec = p.N % 4 == 0 && p.ld_y % 4 == 0 && ((uintptr_t)p.y & 7u) == 0;
  uint32_t from[MOST];
#pragma unroll
  for (int r = 0; r < MOST; ++r)
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from[r]) : "r"(at), "r"(step * (uint32_t)min(r, S - 1) + base));
  for (int i0 = threadIdx.x; i0 < (t1 - t0) * 32; i0 += U * blockDim.x) {
    float q[U][MOST][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * (int)blockDim.x, (t1 - t0) * 32 - 1);
      const uint32_t off = (uint32_t)((t0 + (i >> 5)) * LR_TILE_N + (i & 31) * 4) * 4u;
#pragma unroll
      for (int r = 0; r < MOST; ++r)
        if (r < S)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(q[u][r][0]), "=f"(q[u][r][1]), "=f"(q[u][r][2]), "=f"(q[u][r][3]) : "r"(from[r] + off) : "memory");
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * (int)blockDim.x, n = n0 + (i & 31) * 4;
      if (i >= (t1 - t0) * 32 || n >= p.N) continue;
      T16* y = (T16*)p.y + (row0 + t0 + (i >> 5)) * p.ld_y + n;
      T16 o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v = q[u][0][j];
#pragma unroll
        for (int r = 1; r < MOST; ++r)
          if (r < S) v += q[u][r][j];
        o[j] = from_f32<T16>(v + bias[j]);
      }
      if (vec) {
        *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(o);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) y[j] = o[j];
      }
    }
  }
}

// ---- few tokens ------------------------------------------------------------------------------------------------
constexpr int LS_THREADS = 320;                // warp 0 producer, 1 MMA, 2-9 adapters and then epilogue
constexpr int LS_MAX_STAGES = 8, LS_MAX_TB = 64, LS_MAX_SPLITS = 6;

struct StreamPlan { int tb, splits, stages, smem, direct; };   // tokens of a block, cluster, ring of k steps, bytes, x A made here

__device__ __forceinline__ void adapter_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Single tokens have an adapter each, and an MMA for one of them in 64 columns would be 63 parts zeros that somebody writes: here the second product is
// made on CUDA cores beside the first.  A thread has an output; 16 ranks of it are 32 bytes of B.
template <typename T16>
__global__ void __launch_bounds__(LS_THREADS, 2)
lora_stream_kernel(const LoraParams p, const StreamPlan pl, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  __shared__ __align__(8) uint64_t bars[2 * LS_MAX_STAGES + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ __align__(16) int s_idx[LS_MAX_TB];
  __shared__ int s_first[LS_MAX_TB], s_from[LS_MAX_TB], s_count;
  __shared__ unsigned long long s_mask[LS_MAX_TB];             // the tokens of an adapter
  __shared__ float s_t[LR_PIECE];
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int TB = pl.tb;
  const uint32_t X_BYTES = (uint32_t)TB * 128u, stage_bytes = SUBTILE_BYTES + X_BYTES;
  float* part = reinterpret_cast<float*>(smem);                // [token][output], over the ring once the product is done
  float* extra = reinterpret_cast<float*>(smem + pl.stages * stage_bytes);      // the same of the adapters
  auto FULL = [&](int s) { return smem_u32(&bars[s]); };
  auto EMPTY = [&](int s) { return smem_u32(&bars[LS_MAX_STAGES + s]); };
  const uint32_t ACC = smem_u32(&bars[2 * LS_MAX_STAGES]);
  const Ctl ctl{&s_abort, p.status};
  const uint32_t tmem_cols = TB <= 32 ? 32u : 64u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < LS_MAX_STAGES; ++s) { mbar_init(FULL(s), 1); mbar_init(EMPTY(s), 1); }
    mbar_init(ACC, 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&x_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w_map) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, s_tmem, 0);
  pdl_begin();

  const int n0 = blockIdx.x * LR_TILE_N, rank = blockIdx.z, S = pl.splits;
  const int64_t row0 = (int64_t)blockIdx.y * TB;
  const int rows = (int)min((int64_t)TB, (int64_t)p.T - row0);
  const int KT = (p.K + BLOCK_K - 1) / BLOCK_K, kt0 = KT * rank / S, kt1 = KT * (rank + 1) / S;

  if (warp == 0) {
    // ================================= producer ================================================================
    int it = 0;
    bool ok = true;
    for (int kt = kt0; kt < kt1 && ok; ++kt, ++it) {
      const int s = it % pl.stages;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(EMPTY(s), ((it / pl.stages) & 1u) ^ 1u, ctl, 1101));
      if (!ok) break;
      const uint32_t st = sbase + (uint32_t)s * stage_bytes;
      elect_expect_tx(FULL(s), stage_bytes);
      elect_tile_2d(st, &w_map, kt * BLOCK_K, n0, FULL(s));
      elect_tile_2d(st + SUBTILE_BYTES, &x_map, kt * BLOCK_K, (int)row0, FULL(s));
    }
    if (!ok && lane == 0)                                     // copies in flight land before the block's shared memory goes
      for (int j = it > pl.stages ? it - pl.stages : 0; j < it; ++j)
        for (uint32_t w = 0; w < (1u << 16) && !mbar_test(FULL(j % pl.stages), (j / pl.stages) & 1u); ++w) __nanosleep(64);
    __syncwarp();
  } else if (warp == 1) {
    // ================================= MMA =====================================================================
    int it = 0;
    bool ok = true;
    const uint32_t idesc = lr_idesc(std::is_same<T16, __half>::value, 128, TB);
    for (int kt = kt0; kt < kt1; ++kt, ++it) {
      const int s = it % pl.stages;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(FULL(s), (it / pl.stages) & 1u, ctl, 1102));
      if (!ok) break;
      tc_fence_after();
      const uint32_t st = (sbase + (uint32_t)s * stage_bytes) & 0x3FFFFu;
      const uint32_t a_lo = DESC_LO | (st >> 4), b_lo = DESC_LO | ((st + SUBTILE_BYTES) >> 4);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) elect_mma_bf16(tmem, a_lo + kk * 2, b_lo + kk * 2, idesc, (it | kk) ? 1u : 0u);
      elect_commit(EMPTY(s));
    }
    elect_commit(ACC);
    if (!ok)
      for (uint32_t w = 0; w < (1u << 16) && !mbar_test(ACC, 0); ++w) __nanosleep(64);
    __syncwarp();
  } else {
    // ================================= adapters ================================================================
    // two teams of four warps, one for the even tokens and one for the odd
    const int tid = (threadIdx.x - 64) & 127, team = (warp - 2) >> 2;         // output n0 + tid
    const unsigned long long mine_of = 0x5555555555555555ull << team;
    for (int t = team; t < TB; t += 2) extra[t * LR_TILE_N + tid] = 0.0f;
    if (team == 0 && tid < TB) {
      const int a = tid < rows && p.indx ? p.indx[row0 + tid] : -1;
      s_idx[tid] = a >= 0 && a < p.n_adapters ? a : -1;
    }
    adapter_bar();
    // an adapter counts at its first token: its tokens and its pieces, the pieces numbered through
    if (warp == 6) {                                          // a lane has tokens lane and lane + 32, side by side
      uint32_t mask[2][2] = {{0u, 0u}, {0u, 0u}};
      const int a[2] = {lane < TB ? s_idx[lane] : -1, lane + 32 < TB ? s_idx[lane + 32] : -1};
#pragma unroll
      for (int i = 0; i < LS_MAX_TB; i += 4) {
        if (i >= TB) break;                                   // (a multiple of 16)
        const int4 v = *reinterpret_cast<const int4*>(s_idx + i);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          mask[h][i >> 5] |= (uint32_t)((v.x == a[h] ? 1 : 0) | (v.y == a[h] ? 2 : 0) | (v.z == a[h] ? 4 : 0) | (v.w == a[h] ? 8 : 0)) << (i & 31);
      }
      int f[2], np[2];
      bool fresh[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        fresh[h] = a[h] >= 0 && (h == 0 ? (mask[0][0] & ((1u << lane) - 1u)) == 0 : mask[1][0] == 0 && (mask[1][1] & ((1u << lane) - 1u)) == 0);
        f[h] = fresh[h] ? p.first[a[h]] : 0;
        np[h] = fresh[h] ? p.first[a[h] + 1] : 0;
      }
      int run = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        np[h] -= f[h];
        int sum = np[h];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int q = __shfl_up_sync(0xFFFFFFFFu, sum, o);
          if (lane >= o) sum += q;
        }
        const int t = lane + 32 * h;
        if (t < TB) {
          s_mask[t] = a[h] >= 0 ? (unsigned long long)mask[h][1] << 32 | mask[h][0] : 0ull;
          s_first[t] = f[h];
          s_from[t] = run + sum - np[h];                      // (of tokens that are not the first of their adapter: no pieces)
        }
        run += __shfl_sync(0xFFFFFFFFu, sum, 31);
      }
      if (lane == 0) s_count = run;
    }
    adapter_bar();
    // Every S-th piece is this CTA's, with each of its adapter's tokens.  Few pieces go to all CTAs, and a piece's tokens by twos: 64 tokens of one
    // adapter took 27.6 us with its one piece in one CTA, 17.4 this way.  (With up to 4 S pieces
    // dealt out so, 16 tokens of an adapter each took 17.4 in place of 13.8: a look at each piece in every CTA.)
    const uint8_t* b = p.b + (int64_t)(n0 >> 3) * 256;
    const bool spread = s_count <= S, all = spread || pl.direct;
    const int from = all ? 0 : rank, by = all ? 1 : S, n_mine = s_count > from ? (s_count - from + by - 1) / by : 0;
    unsigned long long twos = 0;                              // tokens 0, 1, 2 S, 2 S + 1, 4 S, ..
    for (int t = 0; t < TB; t += 2 * S) twos |= 3ull << t;
    // -> the list place of this CTA's j-th piece, and which of that adapter's pieces it is
    auto find = [&](int j, int& l, int& i) {
      const int g = from + by * j;
      int lo = 0, hi = TB;                                    // the last place that starts at or before g is the one with pieces
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_from[mid] <= g) lo = mid; else hi = mid;
      }
      l = lo;
      i = g - s_from[lo];
    };
    for (int j = tid + 128 * team; j < n_mine; j += 256) {
      int l, i;
      find(j, l, i);
      l2_hint(b + (int64_t)(s_first[l] + i) * p.NP * 32, LR_PIECE_BYTES);
    }
    b += (tid >> 3) * 256 + (tid & 7) * 16;
    int j = -1, my_l = 0, my_i = 0, l = 0, i = 0, t = 0;      // a lane knows one piece of every 32
    unsigned long long mask = 0;
    auto advance = [&]() {                                    // to the next token of a piece; false behind the last
      while (mask == 0) {
        if (++j >= n_mine) return false;
        if ((j & 31) == 0 && j + lane < n_mine) find(j + lane, my_l, my_i);
        l = __shfl_sync(0xFFFFFFFFu, my_l, j & 31);
        i = __shfl_sync(0xFFFFFFFFu, my_i, j & 31);
        mask = s_mask[l] & mine_of;
        if (spread && !pl.direct) mask &= twos << (2 * ((rank + S - j % S) % S));
      }
      t = __ffsll((long long)mask) - 1;
      mask &= mask - 1;
      return true;
    };
    if (pl.direct) {
      // x A over this CTA's share of k, two ranks a warp: as it is linear, B takes the share like the whole, and the shares of y meet as they do anyway
      if (s_count > 0) {
        const int k1 = min(kt1 * BLOCK_K, (p.K + 7) & ~7), r = (warp - 2) * 2;
        const T16 *a = (const T16*)p.a + ((int64_t)s_first[0] * LR_PIECE + r) * p.ld_a, *x = (const T16*)p.x;
        const float scale = p.scale[s_idx[0]];
        const int ranks = p.ranks ? p.ranks[s_idx[0]] : LR_PIECE;
        float v[2] = {0.0f, 0.0f};
#pragma unroll 2
        for (int k = kt0 * BLOCK_K + lane * 8; k < k1; k += 256) {
          const uint4 xv = *reinterpret_cast<const uint4*>(x + k), a0 = *reinterpret_cast<const uint4*>(a + k), a1 = *reinterpret_cast<const uint4*>(a + p.ld_a + k);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float f = to_f32<T16>(reinterpret_cast<const T16*>(&xv)[j]);
            v[0] = fmaf(f, to_f32<T16>(reinterpret_cast<const T16*>(&a0)[j]), v[0]);
            v[1] = fmaf(f, to_f32<T16>(reinterpret_cast<const T16*>(&a1)[j]), v[1]);
          }
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
          v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
          v[1] += __shfl_xor_sync(0xFFFFFFFFu, v[1], o);
        }
        if (lane < 2) s_t[r + lane] = r + lane < ranks ? (lane ? v[1] : v[0]) * scale : 0.0f;      // (as in the shrink kernel)
      }
      adapter_bar();
    }
    const float* ranks = (pl.direct ? s_t : p.t + row0 * p.ld_t) + (lane & 15);      // a lane holds one of the sixteen ranks of a token
    const int parts = pl.direct ? 1 : p.t_parts;
    bool more = advance();
    // four pairs on their way: as one is taken on, the next takes its place
    constexpr int U = 4;
    uint4 w[U][2];
    float r[U][4];
    int at[U], rest[U];
    auto ask = [&](int u) {
      at[u] = -1;
      if (!more) return;
      const uint4* src = reinterpret_cast<const uint4*>(b + (int64_t)(s_first[l] + i) * p.NP * 32);
      w[u][0] = src[0];
      w[u][1] = src[8];
      at[u] = t;
      rest[u] = t * (int)p.ld_t + i * LR_PIECE;
#pragma unroll
      for (int q = 0; q < LR_MAX_PARTS; ++q) r[u][q] = q < parts ? ranks[q * p.t_part_stride + rest[u]] : 0.0f;
      more = advance();
    };
#pragma unroll
    for (int u = 0; u < U; ++u) ask(u);
    while (at[0] >= 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (at[u] < 0) break;
        const float mine = (r[u][0] + r[u][1]) + (r[u][2] + r[u][3]);
        const T16* e = reinterpret_cast<const T16*>(&w[u][0]);
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) v = fmaf(__shfl_sync(0xFFFFFFFFu, mine, j), to_f32<T16>(e[j]), v);
        extra[at[u] * LR_TILE_N + tid] += v;
        ask(u);
      }
    }
    // ================================= accumulator and adapters' share to shared memory ==================================
    adapter_bar();
    if (__all_sync(0xFFFFFFFFu, mbar_wait(ACC, 0, ctl, 1103))) {
      tc_fence_after();
      const int qd = warp & 3;                                // the lanes of tensor memory that a warp reaches
      for (int c0 = 16 * team; c0 < TB; c0 += 32) {
        uint32_t v[16];
        tmem_ld16(tmem + (uint32_t)c0 + ((uint32_t)(qd * 32) << 16), v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int o = (c0 + j) * LR_TILE_N + qd * 32 + lane;
          part[o] = __uint_as_float(v[j]) + extra[o];
        }
      }
    }
    tc_fence_before();
  }
  float bias[4];
  sums_bias(p, n0, bias);
  __syncthreads();
  if (S > 1) cluster_sync_all();
  const bool ok = cluster_fine(smem_u32(&s_abort), S);
  if (ok) cluster_sums<T16, LS_MAX_SPLITS, 2>(p, sbase, S, 1u, 0u, row0, rows * rank / S, rows * (rank + 1) / S, n0, bias);
  if (S > 1) cluster_sync_all();                              // no CTA leaves while its sums are read
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
  }
}

// ---- many tokens -----------------------------------------------------------------------------------------------
// A cluster of two CTAs computes 256 outputs x up to 512 tokens with tcgen05.mma.cta_group::2: weight rows are the MMA's 256 rows (128 in each CTA),
// tokens its columns, in one or two MMAs of up to 256.  What bounds it is the way from L2 into an SM, some 43 B/ns (no operand is shared between
// clusters): a k step of 64 brings (128 + tb / 2) rows of 128 bytes into each SM, so the tile is as large as tensor memory, one accumulator
// at a time, and the ring is filled again while it is drained.  With few tiles k is cut over up to four pairs of a larger cluster, whose sums meet through distributed
// shared memory as in the kernel above.
constexpr int LP_THREADS = 320, LP_MAX_STAGES = 4, LP_MAX_PIECES = 4, LP_MAX_SPLITS = 4;
struct PairPlan { int tb, mmas, splits, stages, pieces, tiles_n, blocks, clusters, smem; };

__device__ __forceinline__ void elect_mma_pair_f16(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(hi)
      : "memory");
}
// arrive on the barrier at this offset in both CTAs of this pair once every MMA issued so far has completed
__device__ __forceinline__ void elect_commit_both(uint32_t bar, uint32_t mask) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
      "h"((uint16_t)mask)
      : "memory");
}
// a tile into this CTA's shared memory whose bytes count on the barrier of the pair's even CTA
__device__ __forceinline__ void elect_tile_pair(uint32_t dst, const CUtensorMap* tmap, int col, int row, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\t"
      "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
      "l"(tmap), "r"(col), "r"(row), "r"(bar & 0xFEFFFFFFu)
      : "memory");
}

template <typename T16>
__global__ void __launch_bounds__(LP_THREADS, 1)
lora_pair_kernel(const LoraParams p, const PairPlan pl, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  __shared__ __align__(8) uint64_t bars[2 * LP_MAX_STAGES + 3 * LP_MAX_PIECES + 3];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank(), half_id = crank & 1u, even = crank & ~1u, both = 3u << even;
  const int S = pl.splits, split = (int)(crank >> 1), TB = pl.tb, n_mma = TB / pl.mmas, half = n_mma / 2;
  constexpr bool F16 = LR_F16<T16>;
  constexpr uint32_t B_BYTES = lr_tiles(F16) * LR_PIECE_BYTES;
  const uint32_t X_BYTES = (uint32_t)(TB / 2) * 128u, stage_bytes = SUBTILE_BYTES + X_BYTES, T_BYTES = (uint32_t)(TB / 2) * 32u,
                 piece_bytes = (uint32_t)lr_piece_bytes(F16, TB);
  const uint32_t piece0 = sbase + (uint32_t)pl.stages * stage_bytes;
  auto FULL = [&](int s) { return smem_u32(&bars[s]); };                                   // of the even CTA: both CTAs' tiles
  auto EMPTY = [&](int s) { return smem_u32(&bars[LP_MAX_STAGES + s]); };
  auto PTILE = [&](int s) { return smem_u32(&bars[2 * LP_MAX_STAGES + s]); };              // B's tile of a piece in this CTA
  auto PFULL = [&](int s) { return smem_u32(&bars[2 * LP_MAX_STAGES + LP_MAX_PIECES + s]); };      // of the even CTA: the piece in both
  auto PEMPTY = [&](int s) { return smem_u32(&bars[2 * LP_MAX_STAGES + 2 * LP_MAX_PIECES + s]); };
  const uint32_t ACC = smem_u32(&bars[2 * LP_MAX_STAGES + 3 * LP_MAX_PIECES]), ACC_FREE = ACC + 8u, DRAIN = ACC + 16u;
  const Ctl ctl{&s_abort, p.status};
  const uint32_t tmem_cols = TB <= 64 ? 64u : TB <= 128 ? 128u : TB <= 256 ? 256u : 512u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < LP_MAX_STAGES; ++s) { mbar_init(FULL(s), 1); mbar_init(EMPTY(s), 1); }
    for (int s = 0; s < LP_MAX_PIECES; ++s) { mbar_init(PTILE(s), 1); mbar_init(PFULL(s), 8); mbar_init(PEMPTY(s), 1); }
    mbar_init(ACC, 1);
    mbar_init(ACC_FREE, 8);
    mbar_init(DRAIN, 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&x_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w_map) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                         // every CTA's barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, s_tmem, 0);
  pdl_begin();

  const int KT = (p.K + BLOCK_K - 1) / BLOCK_K, kt0 = KT * split / S, kt1 = KT * (split + 1) / S;
  const int tiles = pl.tiles_n * pl.blocks, me = blockIdx.x / (2 * S);
  // consecutive tiles have the same tokens; one tile per cluster where k is cut
  const int tile0 = (int)((int64_t)tiles * me / pl.clusters), tile1 = (int)((int64_t)tiles * (me + 1) / pl.clusters);
  // The loops that issue copies and MMAs look at nothing that differs between lanes, as far as the compiler can tell: an operand that it takes from a vector
  // register, or a loop that it takes for divergent, costs them more than the instruction (with the pieces' list in them, 194 us of 154).
  if (warp == 0) {
    // ================================= producer ================================================================
    int it = 0;
    bool ok = true;
    for (int tile = tile0; tile < tile1 && ok; ++tile) {
      const int block = tile / pl.tiles_n, n0 = (tile - block * pl.tiles_n) * 256 + (int)half_id * LR_TILE_N;
      for (int kt = kt0; kt < kt1; ++kt, ++it) {
        const int s = it % pl.stages;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(EMPTY(s), ((it / pl.stages) & 1u) ^ 1u, ctl, 1111));
        if (!ok) break;
        const uint32_t st = sbase + (uint32_t)s * stage_bytes;
        if (half_id == 0) elect_expect_tx(FULL(s), 2 * stage_bytes);
        elect_tile_pair(st, &w_map, kt * BLOCK_K, n0, FULL(s));
        for (int j = 0; j < pl.mmas; ++j)
          elect_tile_pair(st + SUBTILE_BYTES + (uint32_t)(j * half) * 128u, &x_map, kt * BLOCK_K, block * TB + j * n_mma + (int)half_id * half, FULL(s));
      }
    }
    if (!ok) __nanosleep(500000);                             // copies in flight land before the block's shared memory goes
    __syncwarp();
  } else if (warp == 1) {
    if (half_id == 0) {
      // ================================= MMA ===================================================================
      int it = 0, m = 0;
      bool ok = true;
      const uint32_t idesc = lr_idesc(F16, 256, n_mma), idesc_piece = lr_idesc(false, 256, n_mma);
      for (int tile = tile0, tc = 0; tile < tile1 && ok; ++tile, ++tc) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(ACC_FREE, (tc & 1u) ^ 1u, ctl, 1113));
        if (!ok) break;
        tc_fence_after();
        // this split's pieces of the block: every S-th
        const int total = p.list ? __shfl_sync(0xFFFFFFFFu, p.list[(int64_t)(tile / pl.tiles_n) * LR_LIST + 1], 0) : 0;
        const int end = m + (total > split ? (total - split + S - 1) / S : 0);
        for (int kt = kt0; kt < kt1; ++kt, ++it) {
          const int s = it % pl.stages;
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(FULL(s), (it / pl.stages) & 1u, ctl, 1114));
          if (!ok) break;
          tc_fence_after();
          const uint32_t st = (sbase + (uint32_t)s * stage_bytes) & 0x3FFFFu, a_lo = DESC_LO | (st >> 4), b_lo = DESC_LO | ((st + SUBTILE_BYTES) >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            for (int j = 0; j < pl.mmas; ++j)
              elect_mma_pair_f16(tmem + (uint32_t)(j * n_mma), a_lo + kk * 2, b_lo + (uint32_t)(j * half * 8) + kk * 2, DESC_HI, idesc, kt > kt0 || kk > 0 ? 1u : 0u);
          elect_commit_both(EMPTY(s), both);
        }
        for (; m < end && ok; ++m) {
          const int s = m % pl.pieces;
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(PFULL(s), (m / pl.pieces) & 1u, ctl, 1115));
          if (!ok) break;
          tc_fence_after();
          const uint32_t st = piece0 + (uint32_t)s * piece_bytes, a_lo = piece_desc(st), b_lo = piece_desc(st + B_BYTES);
          for (int j = 0; j < pl.mmas; ++j)
#pragma unroll
            for (int tile_of_b = 0; tile_of_b < lr_tiles(F16); ++tile_of_b)
#pragma unroll
              for (int term = 0; term < lr_terms(F16) - tile_of_b; ++term)
                elect_mma_pair_f16(tmem + (uint32_t)(j * n_mma), a_lo + (uint32_t)tile_of_b * (LR_PIECE_BYTES >> 4),
                                   b_lo + (uint32_t)term * (T_BYTES >> 4) + (uint32_t)(j * half * 2), PIECE_DESC_HI, idesc_piece, 1u);
          elect_commit_both(PEMPTY(s), both);
        }
        if (ok) elect_commit_both(ACC, both);
      }
      elect_commit_pair_local(DRAIN);                         // every MMA has retired before tensor memory is freed
      for (uint32_t w = 0; w < (1u << 16) && !mbar_test(DRAIN, 0); ++w) __nanosleep(64);
    }
    __syncwarp();
  } else if (warp < 6) {
    // ================================= epilogue ================================================================
    const int qd = warp & 3;
    for (int tile = tile0, tc = 0; tile < tile1; ++tile, ++tc) {
      const int block = tile / pl.tiles_n, n = (tile - block * pl.tiles_n) * 256 + (int)half_id * LR_TILE_N + qd * 32 + lane;
      const int64_t row0 = (int64_t)block * TB;
      const int cols = (int)min((int64_t)TB, (int64_t)p.T - row0);
      const float bias = S == 1 && p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, n) : 0.0f;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(ACC, tc & 1u, ctl, 1116))) break;
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem);
      for (int c0 = 0; c0 < cols; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tmem + (uint32_t)c0 + ((uint32_t)(qd * 32) << 16), v);
        tmem_ld_wait();
        if (S > 1) {
#pragma unroll
          for (int j = 0; j < 32; ++j) part[(c0 + j) * LR_TILE_N + qd * 32 + lane] = __uint_as_float(v[j]);
        } else if (n < p.N) {
          T16* y = (T16*)p.y + (row0 + c0) * p.ld_y + n;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c0 + j < cols) y[j * p.ld_y] = from_f32<T16>(__uint_as_float(v[j]) + bias);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(ACC_FREE, even);
    }
  } else {
    // ================================= pieces ==================================================================
    int m = 0;
    bool ok = true;
    for (int tile = tile0; tile < tile1 && ok && p.list; ++tile) {
      const int block = tile / pl.tiles_n, n0 = (tile - block * pl.tiles_n) * 256 + (int)half_id * LR_TILE_N;
      const int32_t* list = p.list + (int64_t)block * LR_LIST;
      const int n = list[0];
      int g = 0, my_a = 0, my_first = 0, my_np = 0;           // the block's adapters 32 at a time, one a lane
      for (int l = 0; l < n && ok; ++l) {
        if ((l & 31) == 0 && l + lane < n) {
          my_a = list[2 + l + lane];
          my_first = p.first[my_a];
          my_np = p.first[my_a + 1] - my_first;
        }
        const int a = __shfl_sync(0xFFFFFFFFu, my_a, l & 31), first = __shfl_sync(0xFFFFFFFFu, my_first, l & 31), np = __shfl_sync(0xFFFFFFFFu, my_np, l & 31);
        for (int i = 0; i < np && ok; ++i, ++g) {
          if (g % S != split) continue;
          const int s = m % pl.pieces;
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(PEMPTY(s), ((m / pl.pieces) & 1u) ^ 1u, ctl, 1112));
          if (!ok) break;
          const uint32_t dst = piece0 + (uint32_t)s * piece_bytes;
          if (warp == 6 && lane == 0) {
            mbar_expect_tx(PTILE(s), LR_PIECE_BYTES);
            // (rows of B are padded to 128: the odd CTA of the last tile may have none)
            bulk_g2s(dst, p.b + ((int64_t)(first + i) * p.NP + (n0 < p.NP ? n0 : 0)) * 32, LR_PIECE_BYTES, PTILE(s));
          }
          for (int r = (warp - 6) * 32 + lane; r < TB / 2; r += 128) {
            const int j = r >= half ? 1 : 0;
            const int64_t token = (int64_t)block * TB + j * n_mma + (int)half_id * half + (r - j * half);
            write_piece_row<T16>(p, token < p.T && p.indx[token] == a, token, i * LR_PIECE, dst + B_BYTES, T_BYTES, r);
          }
          if (F16 || warp == 6) ok = __all_sync(0xFFFFFFFFu, mbar_wait(PTILE(s), (m / pl.pieces) & 1u, ctl, 1117));
          if (!ok) break;
          if (F16)                                            // B's tile becomes its two bf16 parts, the first in its place
            for (uint32_t at = dst + (uint32_t)((warp - 6) * 32 + lane) * 16u; at < dst + LR_PIECE_BYTES; at += 128 * 16u) {
              uint4 hi, lo;
              split_f16(lds128(at), hi, lo);
              sts128(at, hi);
              sts128(at + LR_PIECE_BYTES, lo);
            }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(PFULL(s), even);
          ++m;
        }
      }
    }
    if (!ok) __nanosleep(500000);
  }
  tc_fence_before();
  const int sums_n0 = tile0 % pl.tiles_n * 256 + (int)half_id * LR_TILE_N;
  float bias[4];
  if (S > 1) sums_bias(p, sums_n0, bias);
  __syncthreads();
  cluster_sync_all();
  if (S > 1) {
    // ---- the splits' sums meet, in their order: each CTA takes a share of the tokens of its half of the outputs ----
    const bool ok = cluster_fine(smem_u32(&s_abort), 2 * S);
    if (ok && tile0 < tile1) {
      const int64_t row0 = (int64_t)(tile0 / pl.tiles_n) * TB;
      const int rows = (int)min((int64_t)TB, (int64_t)p.T - row0);
      cluster_sums<T16, LP_MAX_SPLITS, 4>(p, sbase, S, 2u, half_id, row0, rows * split / S, rows * (split + 1) / S, sums_n0, bias);
    }
    cluster_sync_all();                                       // no CTA leaves while its sums are read
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
  }
}

// ---- host ------------------------------------------------------------------------------------------------------
// rows of K 16-bit values as boxes of 64 x box_rows in the 128-byte swizzle; zeros outside
int lr_map(const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows, bool f16, CUtensorMap* map) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  static std::mutex mu;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!encode) {
      void* fn = nullptr;
      cudaDriverEntryPointQueryResult qr;
      MOE_CHECK_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &qr));
      if (qr != cudaDriverEntryPointSuccess || !fn) {
        moe_set_error("moe_lora_matmul: the driver does not provide cuTensorMapEncodeTiled");
        return MOE_ERR_UNSUPPORTED;
      }
      encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }
  }
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    moe_set_error("moe_lora_matmul: cuTensorMapEncodeTiled failed with code %d (rows %lld, K %lld, pitch %lld)", (int)r, (long long)rows, (long long)K, (long long)ld);
    return MOE_ERR_CUDA;
  }
  return MOE_OK;
}

struct ShrinkPlan { int nb, places, parts; };
ShrinkPlan lr_shrink_plan(int64_t T, int K, int max_pieces, int n_adapters) {
  ShrinkPlan s;
  // Eights read an adapter's rows more often, sixty-fours have fewer blocks for the adapters of single tokens.  K = 2880, N = 5120, 32 adapters of one piece, eights
  // against sixty-fours, us of the whole operator: tokens in turns 512 65 : 98, 1024 95 : 136, 2048 179 : 259, 3000 205 : 345, 4096 290 : 440; in runs 512 33 : 34, 1024
  // 44.6 : 46.1, 2048 73.7 : 75.3, 3000 93.7 : 96.3, 4096 115 : 109.  1200 tokens in runs, adapters of up to four pieces: 28.5 : 26.7.
  s.nb = T <= 1024 || T * max_pieces <= 3500 ? 1 : 8;
  const int most = s.nb == 1 ? 8 : 4;                         // (a place without an adapter costs a block of threads all the same)
  s.places = n_adapters < most ? n_adapters : most;
  // shares of k while the blocks that have something to do, a quarter of them say, are hardly more than the SMs
  const int64_t blocks = cdiv64(T, 8 * s.nb) * max_pieces * (s.nb == 1 && s.places > 2 ? s.places / 2 : 1);
  int parts = 1;
  while (parts < LR_MAX_PARTS && blocks * parts <= moe_sm_count() * 3 / 2 && K / (32 * SH_WARPS) >= 2 * parts) parts *= 2;
  s.parts = parts;
  // no more than some two and a half rounds of blocks (two per SM) for the sake of places, most of which find no adapter
  while (s.nb > 1 && s.places > 1 && blocks * parts * s.places > 5 * moe_sm_count()) s.places = (s.places + 1) / 2;
  return s;
}

// A token's x A within the product's kernel: saves a launch, and costs every CTA its share of A's rows, some 1 us a token and piece.  K = 2880, N = 5120: one
// token and piece 10.2 us in place of 11.5, two 12.0 and 11.8, four 14.3 and 12.5, eight 19.0 and 12.5.
bool lr_direct(int64_t T, int max_pieces) { return T * max_pieces <= 1; }

StreamPlan lr_stream_plan(int64_t T, int K, int N, int max_pieces) {
  StreamPlan pl;
  pl.direct = max_pieces > 0 && lr_direct(T, max_pieces);
  pl.tb = T >= LS_MAX_TB ? LS_MAX_TB : (int)cdiv64(T, 16) * 16;
  const int64_t tiles = cdiv64(N, LR_TILE_N) * cdiv64(T, pl.tb), KT = cdiv64(K, BLOCK_K);
  const int stage = SUBTILE_BYTES + pl.tb * 128, sums = pl.tb * LR_TILE_N * 4;
  // Two CTAs per SM.  k is cut as long as the clusters fit side by side, which they do not up to the last place: 40 tiles took 21.5 us in clusters of four
  // to six CTAs and 29.7 in clusters of seven (280 CTAs of 296), where some wait for a second round.
  int64_t s = moe_sm_count() * 5 / 3 / tiles;
  if (s > KT / 4) s = KT / 4;
  pl.splits = (int)(s < 1 ? 1 : s > LS_MAX_SPLITS ? LS_MAX_SPLITS : s);
  const int st = (104 * 1024 - sums) / stage;
  pl.stages = st > LS_MAX_STAGES ? LS_MAX_STAGES : st;
  pl.smem = pl.stages * stage + sums + 1024;                  // (the product's sums take the ring's place: two stages are enough for them)
  return pl;
}

// Clusters of 2 s CTAs of the pair kernel that run side by side (asked once per device)
int64_t lr_pair_clusters(int s) {
  static std::mutex mu;
  static int cached[64][5] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  std::lock_guard<std::mutex> lk(mu);
  if (cached[dev][s] == 0) {
    const int smem = 225 * 1024;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * s * 256));
    cfg.blockDim = dim3(LP_THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)(2 * s); at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(lora_pair_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, lora_pair_kernel<__nv_bfloat16>, &cfg) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = moe_sm_count() / (2 * s) > 0 ? moe_sm_count() / (2 * s) : 1;
    }
    cached[dev][s] = n;
  }
  return cached[dev][s];
}

// Form of the product for many tokens.  Tokens are cut into blocks and k over up to four pairs; a round of tiles costs what comes into an SM, in rows of
// 128 bytes, and draining the accumulator about as much as 2.6 rows a token.
PairPlan lr_pair_plan(int64_t T, int K, int N, bool f16) {
  PairPlan best = {};
  const int64_t KT = cdiv64(K, BLOCK_K), tiles_n = cdiv64(N, 256);
  int64_t side[LP_MAX_SPLITS + 1];                            // clusters of so many pairs that run side by side
  for (int s = 1; s <= LP_MAX_SPLITS; ++s) side[s] = lr_pair_clusters(s);
  double least = 0.0;
  const int64_t fewest = cdiv64(T, LR_MAX_TB);
  for (int64_t nb = fewest; nb <= fewest + 8; ++nb) {
    int64_t tb = cdiv64(cdiv64(T, nb), 32) * 32;
    if (tb < 64) tb = 64;
    const int64_t blocks = cdiv64(T, tb), tiles = tiles_n * blocks;
    int64_t s = tb > 416 ? 1 : KT / 4 < LP_MAX_SPLITS ? KT / 4 : LP_MAX_SPLITS;       // (a split's sums are tb x 128 fp32 in shared memory)
    while (s > 1 && tiles > side[s]) --s;
    if (s < 1) s = 1;
    const double rounds = (double)cdiv64(tiles, side[s]);
    const double cost = rounds * ((double)cdiv64(KT, s) * (128 + tb / 2) + 2.6 * tb);
    if (best.tb == 0 || cost < least) {
      least = cost;
      best.tb = (int)tb; best.blocks = (int)blocks; best.splits = (int)s; best.tiles_n = (int)tiles_n;
      best.clusters = (int)(s > 1 || tiles < side[1] ? tiles : side[1]);
    }
  }
  best.mmas = best.tb > 256 ? 2 : 1;
  // Two pieces of fp16, larger ones, at the least, so that they take no stage away that bf16 has
  const int stage = SUBTILE_BYTES + best.tb * 64, piece = lr_piece_bytes(f16, best.tb), room = 224 * 1024;
  best.stages = (room - (f16 ? 2 : LP_MAX_PIECES) * piece) / stage;
  if (best.stages > LP_MAX_STAGES) best.stages = LP_MAX_STAGES;
  best.pieces = (room - best.stages * stage) / piece;
  if (best.pieces > LP_MAX_PIECES) best.pieces = LP_MAX_PIECES;
  int bytes = best.stages * stage + best.pieces * piece;
  if (best.splits > 1 && bytes < best.tb * LR_TILE_N * 4) bytes = best.tb * LR_TILE_N * 4;
  best.smem = bytes + 1024;
  return best;
}
// Up to 128 tokens, decode's batches, weight rows by themselves fill the SMs (two CTAs each), and a token with an adapter of its own costs some fma; beyond,
// a pair reads the tokens half as often, and a run of tokens of one adapter costs an MMA.  K = 2880, N = 5120, stream against pair, us: 32 adapters in
// turns, 32 tokens 16.9 : 29.7, 64 21.0 : 30.2, 96 22.5 : 31.2, 128 25.1 : 33.3, 256 42.5 : 35.3; one adapter per 64 tokens, 32 tokens 14.3 : 15.4, 64 17.5 :
// 16.4, 96 18.9 : 17.4, 128 21.0 : 18.4, 256 35.3 : 22.5.
bool lr_many(int64_t T) { return T > 128; }

size_t lr_t_bytes(const MoeLoraArgs& a, ShrinkPlan s) { return ((size_t)s.parts * (size_t)a.T * (size_t)a.max_pieces * LR_PIECE * 4 + 255) / 256 * 256; }
size_t lr_list_bytes(const MoeLoraArgs& a) { return lr_many(a.T) ? (size_t)lr_pair_plan(a.T, a.K, a.N, a.dtype == MOE_F16).blocks * LR_LIST * 4 : 0; }

int lr_check(const MoeLoraArgs* a) {
  MOE_CHECK_ARG(a, "moe_lora_matmul: NULL argument");
  MOE_CHECK_ARG(a->T >= 0 && a->K > 0 && a->N > 0 && a->n_adapters >= 0 && a->max_pieces >= 0, "moe_lora_matmul: sizes must be positive");
  MOE_CHECK_ARG(a->dtype == MOE_BF16 || a->dtype == MOE_F16, "moe_lora_matmul: x, W and the adapters are bf16 or fp16");
  if (a->T >= (1ll << 31) - 512 || a->K > (1 << 30) || a->N > (1 << 30) || a->max_pieces > 64) {
    moe_set_error("moe_lora_matmul: takes fewer than 2^31 tokens and ranks up to 1024 (got T = %lld, K = %d, N = %d, %d pieces of 16 ranks)", (long long)a->T, a->K,
                  a->N, a->max_pieces);
    return MOE_ERR_UNSUPPORTED;
  }
  return MOE_OK;
}

// allows a kernel its dynamic shared memory, once per device (a microsecond of every call otherwise)
int lr_allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  MOE_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return MOE_OK;
  MOE_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
  return MOE_OK;
}
template <typename K> int lr_allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& done) { return lr_allow_smem((const void*)kernel, bytes, done); }

template <typename T16> int lr_shrink(const LoraParams& p, const ShrinkPlan& sp, cudaStream_t st) {
  const dim3 grid((unsigned)cdiv64(p.T, 8 * sp.nb), (unsigned)p.max_pieces, (unsigned)(sp.places * sp.parts + (p.list_tb > 0 ? 1 : 0)));
  if (sp.nb == 1) MOE_CHECK_CUDA(launch_pdl(lora_shrink_kernel<T16, 1>, grid, dim3(SH_WARPS * 32), (size_t)0, st, p));
  else MOE_CHECK_CUDA(launch_pdl(lora_shrink_kernel<T16, 8>, grid, dim3(SH_WARPS * 32), (size_t)0, st, p));
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <typename T16> int lr_stream(const LoraParams& p, const MoeLoraArgs& a, cudaStream_t st) {
  const bool f16 = std::is_same<T16, __half>::value;
  const StreamPlan pl = lr_stream_plan(p.T, p.K, p.N, p.max_pieces);
  CUtensorMap w_map, x_map;
  if (int rc = lr_map(a.w_t, a.N, a.K, a.ld_w, LR_TILE_N, f16, &w_map)) return rc;
  if (int rc = lr_map(a.x, a.T, a.K, a.ld_x, pl.tb, f16, &x_map)) return rc;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = lr_allow_smem(lora_stream_kernel<T16>, 112 * 1024, allowed)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cdiv64(p.N, LR_TILE_N), (unsigned)cdiv64(p.T, pl.tb), (unsigned)pl.splits);
  cfg.blockDim = dim3(LS_THREADS);
  cfg.dynamicSmemBytes = (size_t)pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 1; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = (unsigned)pl.splits;
  cfg.attrs = at;
  cfg.numAttrs = pl.splits > 1 ? 2 : 1;
  MOE_CHECK_CUDA(cudaLaunchKernelEx(&cfg, lora_stream_kernel<T16>, p, pl, w_map, x_map));
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <typename T16> int lr_pair(const LoraParams& p, const MoeLoraArgs& a, const PairPlan& pl, cudaStream_t st) {
  const bool f16 = std::is_same<T16, __half>::value;
  CUtensorMap w_map, x_map;
  if (int rc = lr_map(a.w_t, a.N, a.K, a.ld_w, LR_TILE_N, f16, &w_map)) return rc;
  if (int rc = lr_map(a.x, a.T, a.K, a.ld_x, pl.tb / pl.mmas / 2, f16, &x_map)) return rc;
  static std::atomic<uint64_t> allowed{0};
  if (int rc = lr_allow_smem(lora_pair_kernel<T16>, 225 * 1024, allowed)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pl.clusters * 2 * pl.splits));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.dynamicSmemBytes = (size_t)pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)(2 * pl.splits); at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  MOE_CHECK_CUDA(cudaLaunchKernelEx(&cfg, lora_pair_kernel<T16>, p, pl, w_map, x_map));
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

}  // namespace

extern "C" __attribute__((visibility("default"))) size_t moe_lora_matmul_workspace_bytes(const MoeLoraArgs* a) {
  if (lr_check(a) != MOE_OK || a->n_adapters == 0 || lr_direct(a->T, a->max_pieces)) return 0;
  return lr_t_bytes(*a, lr_shrink_plan(a->T, a->K, a->max_pieces, a->n_adapters)) + lr_list_bytes(*a);
}

extern "C" __attribute__((visibility("default"))) int moe_lora_matmul(const MoeLoraArgs* args, void* stream) {
  if (int rc = lr_check(args)) return rc;
  const MoeLoraArgs& a = *args;
  if (a.T == 0) return MOE_OK;
  MOE_CHECK_ARG(a.x && a.w_t && a.y, "moe_lora_matmul: NULL argument");
  MOE_CHECK_ARG(a.ld_x >= a.K && a.ld_w >= a.K, "moe_lora_matmul: rows of x and W^T are K values apart at least");
  MOE_CHECK_ARG(a.ld_x % 8 == 0 && a.ld_w % 8 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.w_t % 16 == 0,
                "moe_lora_matmul: rows of x and W^T must be 16-byte aligned");
  const bool adapters = a.n_adapters > 0 && a.max_pieces > 0, direct = adapters && lr_direct(a.T, a.max_pieces);
  ShrinkPlan sp = {1, 1, 1};
  if (adapters) {
    MOE_CHECK_ARG(a.a && a.b && a.first && a.scale && a.indx, "moe_lora_matmul: NULL argument of the adapters");
    MOE_CHECK_ARG(a.ld_a % 8 == 0 && a.ld_a >= (a.K + 7) / 8 * 8 && (uintptr_t)a.a % 16 == 0 && (uintptr_t)a.b % 16 == 0,
                  "moe_lora_matmul: adapters must be 16-byte aligned, their rows padded to 8 values");
    MOE_CHECK_ARG(a.ld_x >= (a.K + 7) / 8 * 8, "moe_lora_matmul: rows of x must be padded to 8 values");
    sp = lr_shrink_plan(a.T, a.K, a.max_pieces, a.n_adapters);
    const size_t need = direct ? 0 : lr_t_bytes(a, sp) + lr_list_bytes(a);
    MOE_CHECK_ARG(need == 0 || (a.workspace && (uintptr_t)a.workspace % 256 == 0 && a.workspace_bytes >= need),
                  "moe_lora_matmul: needs a 256-byte aligned workspace of %zu bytes", need);
  }
  cudaStream_t st = (cudaStream_t)stream;
  LoraParams p = {};
  p.x = a.x; p.ld_x = a.ld_x; p.T = (int)a.T; p.K = a.K; p.N = a.N; p.NP = (int)cdiv64(a.N, LR_TILE_N) * LR_TILE_N;
  p.bias = a.bias; p.bias_dtype = a.bias_dtype;
  if (adapters) {
    p.a = a.a; p.ld_a = a.ld_a; p.b = (const uint8_t*)a.b; p.first = a.first; p.scale = a.scale; p.n_adapters = a.n_adapters; p.max_pieces = a.max_pieces;
    p.ranks = a.ranks; p.indx = a.indx;
    p.t = (float*)a.workspace; p.ld_t = (int64_t)a.max_pieces * LR_PIECE; p.t_parts = sp.parts; p.t_part_stride = a.T * p.ld_t;
  }
  p.y = a.y; p.ld_y = a.ld_y; p.status = a.status;
  const bool many = lr_many(a.T);
  const PairPlan pl = many ? lr_pair_plan(a.T, a.K, a.N, a.dtype == MOE_F16) : PairPlan{};
  if (adapters && many) {
    p.list = (int32_t*)((uint8_t*)a.workspace + lr_t_bytes(a, sp));
    p.list_tb = pl.tb;
  }
  if (adapters && !direct)
    if (int rc = a.dtype == MOE_F16 ? lr_shrink<__half>(p, sp, st) : lr_shrink<__nv_bfloat16>(p, sp, st)) return rc;
  if (many) return a.dtype == MOE_F16 ? lr_pair<__half>(p, a, pl, st) : lr_pair<__nv_bfloat16>(p, a, pl, st);
  return a.dtype == MOE_F16 ? lr_stream<__half>(p, a, st) : lr_stream<__nv_bfloat16>(p, a, st);
}
