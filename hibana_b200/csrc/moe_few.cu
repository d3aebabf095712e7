// A mixture-of-experts layer for up to 16 tokens.
//
//   logits = r R^T                       r the router's input rows (the layer's, or the wider ones of a latent layer)
//   score  = softmax(logits) or sigmoid(logits);  ids = the top-k of score (+ selection bias), ties to the lower index
//   w_j    = scale * score_j (/ sum of the chosen scores)
//   mid_j  = silu(W1g x) * (W1u x)  or  relu(W1 x)^2          W1, W2 of expert ids_j
//   out    = sum_j w_j W2 mid_j (+ shared)                    rounded once
//
// Three launches:
//   route : router logits; the rows of x as an operand of the tensor cores;
//   fc1   : top-k and plan, the chosen experts' first product, the activation;
//   fc2   : the second product, the weighted sum, the shared expert's rows.
//
// At these sizes the layer is the stream of its experts' weights: every chosen expert is read once, whatever it does to one or to
// eight rows. So the weights take the 128-row side of tcgen05.mma as they lie in memory, and never pass through registers: decoding
// FP4 there costs 0.1 instructions a weight, which bounds one token as much as sixteen (measured: 1.7 TB/s of weights).
//
// Activations are not quantised to FP4. With FP4 weights the tensor cores want FP4 activations, so a number becomes five of them: a block (32
// elements, 16 for NVFP4) is scaled by a power of two to 14-bit integers, X = sum_p d_p 8^p with digits d_p of -4 .. 4, which
// e2m1 holds exactly. The digits of a row are five columns of the product (five rows of operand B, with the block's scale), and
// the epilogue adds them up: 8^p D_p. What is lost is half a unit of X, 2^-14 to 2^-15 of the largest number of its block. An NVFP4
// scale spans 2^-9 .. 2^8; blocks further below the largest of their row share the lowest one. Rows of mid have one scale each, so that
// half a unit is 2^-14 to 2^-15 of the row's largest number. With bf16 weights x is one column, and mid two (two bf16 numbers, 16 bits).
//
// Warp roles (fc1, fc2): one issues the weights' TMA copies into a ring of stages; one or two (each for every other unit, with its own
// accumulator and its own half of the stages) issue MMAs; two groups of four read the accumulators back; in fc2 four convert the rows of
// mid that a K tile needs, straight into the stage's B tile. fc1 walks (expert, 128
// rows) over all CTAs with all tokens' columns resident; in fc2 the CTAs of a cluster share an output block of 128 rows, each with its
// part of the experts, and add up through distributed shared memory in order.
//
// Measured (us a call among others, weights from memory; in brackets route / fc1 / fc2 on their own, and the time of the bytes at the copy
// rate): 512 experts, 2560-640 SwiGLU, MXFP4, top 10: 1 token 23 (4.1 / 14 / 14; 4.4), 16 tokens 77 (4.4 / 51 / 35; 56); 512
// experts, 1024-2688 squared ReLU, NVFP4, top 22, router over 4096: 4 tokens 60 (5.7 / 35 / 35; 40); 64 experts, 2048-768 SwiGLU, bf16,
// top 8: 7 tokens 68 (3.6 / 50 / 31; 56). The products stream 5 to 6.6 TB/s while they stream. Bound by what happens before the first
// weights can be named and between kernels: logits 4, top-k 2.5 and plan 1, first tiles 2 each, from fc1's last tile to fc2's first 5,
// the cluster's sums 3. fc2 runs on the clusters that fit (80 to 120 of 148 SMs: 120 with clusters of six on 20 output blocks). Fetching the
// first of W2 into L2 from fc1's last tiles on made 16 tokens 2 us slower (one token, whose fc1 leaves CTAs and memory idle, was not tried).
#include <algorithm>
#include <cstddef>

#include "gemm.cuh"
#include "hb_api.h"
#include "hb_common.cuh"
#include "rownorm.cuh"

namespace hb {
namespace {

constexpr int MAX_TOKENS = 16;
constexpr int MAX_TOPK = 32;
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_PAIRS = MAX_TOKENS * MAX_TOPK;
constexpr int WARPS = 16;
constexpr int THREADS = WARPS * 32;
constexpr int COLS = 8;                  // tokens of an entry of the plan
constexpr int MAX_STAGES = 10;
constexpr int MAX_CLUSTER = 16;          // of fc2 (more than eight CTAs need a kernel attribute)
constexpr int MAX_SMEM = 227 * 1024;
constexpr int A_BYTES = 128 * 128;       // 128 weight rows x 128 bytes of K
constexpr int CANDIDATES = 64;           // of a token's top-k
constexpr int CAND_BYTES = (2 * CANDIDATES + MAX_TOPK) * 4;

template <int KIND>
struct Traits {
  static constexpr bool kFp4 = KIND != kGemmBf16;
  static constexpr int TILE_K = kFp4 ? 256 : 64;            // K elements of a 128-byte row
  static constexpr int MMA_K = kFp4 ? 64 : 16;
  static constexpr int BLOCK = KIND == kGemmMxfp4 ? 32 : 16;
  static constexpr int ATOMS = sf_atoms(KIND);
  static constexpr int SF_BYTES = ATOMS * 512;
  static constexpr int XP = kFp4 ? 5 : 1;                   // columns of a row of x, of a row of mid
  static constexpr int MP = kFp4 ? 5 : 2;
  static constexpr int B2_ROWS = (COLS * MP + 15) / 16 * 16;
  static constexpr int STAGE1 = A_BYTES + SF_BYTES;
  static constexpr int STAGE2 = A_BYTES + SF_BYTES + B2_ROWS * 128;
};

struct FewParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* route_x;
  const __nv_bfloat16* router;
  const float* sel_bias;
  const __nv_bfloat16* shared;
  __nv_bfloat16* out;
  long long ldx, ld_route, ld_router, ld_shared, ldo;
  int tokens, experts, topk, hidden, inter, h_out, route_k;
  int sigmoid, renorm, swiglu;
  float scale;
  const uint8_t *sf1, *sf2;
  const float *gs1, *gs2;
  int ka1, ka2;
  // workspace
  float* logits;                         // [tokens][experts]
  float* x_factor;                       // [tokens] NVFP4: what the blocks' scales of a row are relative to
  uint8_t* x_img;                        // [K tiles][n][128] swizzled B tiles, then [K tiles][SF_BYTES] scales
  struct EntryRecord* entries;           // [pairs] the plan, for fc2
  float* mid;                            // [pairs][inter]
  uint8_t* mid_exp;                      // [pairs][exp_ld] biased exponent of the largest number of 32 rows of fc1 (FP4)
  int exp_ld, n, stages;
  int* status;
};

// The routing as every CTA holds it: entries, an expert and up to eight of its tokens, in the order in which the tokens' lists first
// name them.
struct Plan {
  int entries;
  int ids[MAX_PAIRS];
  float weights[MAX_PAIRS];
  uint32_t chosen[MAX_TOKENS][MAX_EXPERTS / 32];      // bit e: the token chose expert e
  int starts[THREADS / 32];
  unsigned short entry_of[MAX_EXPERTS * 2];             // entry of an expert's tokens 0 .. 7, 8 .. 15
  unsigned short expert[MAX_PAIRS], count[MAX_PAIRS];   // of entries
  alignas(16) unsigned short pair[MAX_PAIRS * COLS];    // [entry][column]: token * topk + j
  int row_exp[MAX_PAIRS];                               // fc2, FP4: exponent of the row's largest number
};
static_assert(alignof(Plan) == 16, "entries are stored as 16-byte pieces");
struct alignas(16) EntryRecord {
  int expert, count, entries, unused;
  unsigned short pair[COLS];
  float weight[COLS];
};
static_assert(sizeof(EntryRecord) == 64 && offsetof(EntryRecord, pair) == 16 && offsetof(EntryRecord, weight) == 32, "read in 16-byte pieces");

// ---------------------------------------------------------------- rows of activations as operand B
// Byte of K element `k` (of the K tile) in row n of a B tile: 128-byte rows, 16-byte chunks permuted by the row (SWIZZLE_128B).
__device__ __forceinline__ int b_offset(int n, int byte) { return n * 128 + (((byte >> 4) ^ (n & 7)) << 4) + (byte & 15); }
__device__ __forceinline__ int sf_offset(int n, int g) { return (g >> 2) * 512 + (n & 31) * 16 + (n >> 5) * 4 + (g & 3); }

// 2^e as the scale byte of the format; `e` 128: NaN.
template <int KIND>
__device__ __forceinline__ uint32_t scale_byte(int e) {
  if constexpr (KIND == kGemmMxfp4) return e == 128 ? 255u : static_cast<uint32_t>(e + 127);
  else return e == 128 ? 0x7Fu : e >= -6 ? static_cast<uint32_t>(e + 7) << 3 : 1u << (e + 9);
}

// Eight consecutive numbers times f (magnitudes of 2^14 at most; more only in rows that come out as NaN) -> five words of eight e2m1
// digits. Eighty instructions: with a shift and a table look-up a digit they were 290, and the converters of fc2 were what it waited for.
__device__ __forceinline__ void digits8(const float (&v)[8], float f, uint32_t (&w)[5]) {
  // X + 4 + 4 * 8 + .. + 4 * 8^4 is sixteen bits, three a digit (four the top one), rounded by the addition: an fp32 number of this
  // size counts in ones
  uint32_t y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    constexpr float kOnes = 12582912.f + (4 + 32 + 256 + 2048 + 16384);
    y[j] = __byte_perm(__float_as_uint(fmaf(v[2 * j], f, kOnes)), __float_as_uint(fmaf(v[2 * j + 1], f, kOnes)), 0x5410);
  }
#pragma unroll
  for (int p = 0; p < 5; ++p) {
    uint32_t sel = 0;                        // digits as indexes: of the even numbers in the lower half, of the odd ones in the upper
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = 4 * j >= 3 * p ? y[j] << (4 * j - 3 * p) : y[j] >> (3 * p - 4 * j);
      sel |= at & ((p == 4 ? 0x000F000Fu : 0x00070007u) << (4 * j));
    }
    // codes of the digits -4 .. 3, a byte each; 4, which only the top digit takes, is the code of -4 without its sign
    uint32_t even = __byte_perm(0x0A0C0D0Eu, 0x05040200u, sel & 0x7777u), odd = __byte_perm(0x0A0C0D0Eu, 0x05040200u, (sel >> 16) & 0x7777u);
    if (p == 4) {
      even ^= __byte_perm(0u, 8u, (sel >> 1) & 0x4444u);
      odd ^= __byte_perm(0u, 8u, (sel >> 17) & 0x4444u);
    }
    w[p] = even | odd << 4;
  }
}
// A block whose largest magnitude (bits) is `top`: the factor of its numbers, 2^(140 - e) with e the biased exponent of `top`, and the
// block's scale byte. `row_e`: that exponent of the whole row (NVFP4), which x_factor undoes.
template <int KIND>
__device__ __forceinline__ float block_factor(uint32_t top, int row_e, uint32_t& scale) {
  int e = static_cast<int>(top >> 23);
  if constexpr (KIND == kGemmMxfp4) {
    const bool bad = e == 255;
    e = max(e, 13);
    scale = scale_byte<KIND>(bad ? 128 : e - 140);
  } else {
    const bool bad = row_e == 255;
    row_e = max(row_e, 13);
    e = max(min(max(e, row_e - 17), row_e), 13);
    scale = scale_byte<KIND>(bad ? 128 : e - row_e + 8);      // 2^-9 .. 2^8
  }
  return __int_as_float((267 - e) << 23);
}
__device__ __forceinline__ float pow2(int e) {              // -149 < e < 128
  return e >= -126 ? __int_as_float((e + 127) << 23) : __int_as_float(0x00400000 >> (-127 - e));
}
__device__ __forceinline__ float x_factor(int row_e) { return pow2(max(min(row_e, 254), 13) - 148); }
// Rows of mid have one scale, that of their largest number (exponent e; 255: the row holds an infinity or a NaN, and all that is made
// of it is NaN).
__device__ __forceinline__ float mid_factor(int e) { return __int_as_float((267 - max(e, 13)) << 23); }
__device__ __forceinline__ float mid_back(int e) { return e == 255 ? __int_as_float(0x7FC00000) : pow2(max(e, 13) - 140); }

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// Largest magnitude (bits) of the lanes of a block: eight elements a lane.
template <int KIND>
__device__ __forceinline__ uint32_t block_top(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[j]));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  if constexpr (KIND == kGemmMxfp4) top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  return top;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------- route
// CTAs up to experts / 16: the logits of sixteen experts, K split over the warps. A lane holds eight consecutive K of two router rows
// and of a token, so K is permuted alike on both sides of the products. The others: one row of x each.
constexpr int ROUTE_WARPS = 16;
template <int KIND>
__global__ void __launch_bounds__(ROUTE_WARPS * 32) moe_few_route_kernel(const __grid_constant__ FewParams p) {
  using T = Traits<KIND>;
  __shared__ float part[ROUTE_WARPS][256];
  __shared__ uint32_t s_top[ROUTE_WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int e_tiles = (p.experts + 15) / 16;
  grid_dep_wait();
  grid_dep_launch();
  if (static_cast<int>(blockIdx.x) < e_tiles) {
    const int e0 = blockIdx.x * 16, blocks = (p.route_k + 31) / 32;
    const __nv_bfloat16* ra = p.router + static_cast<long long>(min(e0 + g, p.experts - 1)) * p.ld_router;
    const __nv_bfloat16* rb = p.router + static_cast<long long>(min(e0 + g + 8, p.experts - 1)) * p.ld_router;
    const __nv_bfloat16* xa = p.route_x + min(g, p.tokens - 1) * p.ld_route;
    const __nv_bfloat16* xb = p.route_x + min(g + 8, p.tokens - 1) * p.ld_route;
    const bool two = p.tokens > 8;
    float acc[2][4] = {};
    // Loads of 512 columns in flight. us at widths of 1024, 2560, 4096, 7168 (512 experts, one token): two 3.2, 5.3, 6.5, 9.9, four 3.3, 4.9,
    // 5.7, 8.5, five 3.3, 4.0, 5.7, 8.0, eight 5.8, 6.6, 7.9, 11.6.
    constexpr int U = 5;
    for (int b0 = warp; b0 < blocks; b0 += ROUTE_WARPS * U) {
      uint4 wa[U], wb[U], va[U], vb[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int k = (b0 + i * ROUTE_WARPS) * 32 + t * 8;
        wa[i] = wb[i] = va[i] = vb[i] = make_uint4(0, 0, 0, 0);
        if (k < p.route_k) {
          wa[i] = ld_step(reinterpret_cast<const uint4*>(ra + k));
          wb[i] = ld_step(reinterpret_cast<const uint4*>(rb + k));
          va[i] = ld_step(reinterpret_cast<const uint4*>(xa + k));
          if (two) vb[i] = ld_step(reinterpret_cast<const uint4*>(xb + k));
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        mma_16816(acc[0], wa[i].x, wb[i].x, wa[i].y, wb[i].y, va[i].x, va[i].y);
        mma_16816(acc[0], wa[i].z, wb[i].z, wa[i].w, wb[i].w, va[i].z, va[i].w);
        if (two) {
          mma_16816(acc[1], wa[i].x, wb[i].x, wa[i].y, wb[i].y, vb[i].x, vb[i].y);
          mma_16816(acc[1], wa[i].z, wb[i].z, wa[i].w, wb[i].w, vb[i].z, vb[i].w);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      part[warp][(n * 8 + 2 * t) * 16 + g] = acc[n][0];
      part[warp][(n * 8 + 2 * t + 1) * 16 + g] = acc[n][1];
      part[warp][(n * 8 + 2 * t) * 16 + g + 8] = acc[n][2];
      part[warp][(n * 8 + 2 * t + 1) * 16 + g + 8] = acc[n][3];
    }
    __syncthreads();
    const int tok = tid >> 4, e = e0 + (tid & 15);
    if (tid < 256 && tok < p.tokens && e < p.experts) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < ROUTE_WARPS; ++w) s += part[w][tid];
      p.logits[tok * p.experts + e] = s;
    }
    return;
  }
  const int tok = blockIdx.x - e_tiles, k_tiles = (p.hidden + T::TILE_K - 1) / T::TILE_K, pieces = k_tiles * T::TILE_K / 8;
  const __nv_bfloat16* row = p.x + tok * p.ldx;
  int row_e = 0;
  if constexpr (KIND == kGemmNvfp4) {
    uint32_t top = 0;
    for (int c = tid; c * 8 < p.hidden; c += ROUTE_WARPS * 32) {
      const uint4 v = ld_step(reinterpret_cast<const uint4*>(row + c * 8));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, max((w[i] << 16) & 0x7FFF0000u, w[i] & 0x7FFF0000u));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ROUTE_WARPS; ++w) top = max(top, s_top[w]);
    row_e = static_cast<int>(top >> 23);
    if (tid == 0) p.x_factor[tok] = x_factor(row_e);
  }
  // (pieces is a multiple of 32 for FP4: whole warps take the shuffles)
  for (int c = tid; c < pieces; c += ROUTE_WARPS * 32) {
    const uint4 raw = c * 8 < p.hidden ? ld_step(reinterpret_cast<const uint4*>(row + c * 8)) : make_uint4(0, 0, 0, 0);
    if constexpr (!T::kFp4) {
      *reinterpret_cast<uint4*>(p.x_img + static_cast<size_t>(c >> 3) * p.n * 128 + b_offset(tok, (c & 7) * 16)) = raw;
    } else {
      const int kt = c >> 5, byte = (c & 31) * 4;
      float v[8];
      unpack8(raw, v);
      uint32_t w[5];
      uint32_t sf;
      const float f = block_factor<KIND>(block_top<KIND>(v), row_e, sf);
      digits8(v, f, w);
      uint8_t* img = p.x_img + static_cast<size_t>(kt) * p.n * 128;
      uint8_t* sfs = p.x_img + static_cast<size_t>(k_tiles) * p.n * 128 + static_cast<size_t>(kt) * T::SF_BYTES;
      const bool first = (c & (T::BLOCK / 8 - 1)) == 0;
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int n = tok * 5 + i;
        *reinterpret_cast<uint32_t*>(img + b_offset(n, byte)) = w[i];
        if (first) sfs[sf_offset(n, (c & 31) / (T::BLOCK / 8))] = static_cast<uint8_t>(sf);
      }
    }
  }
}

// ---------------------------------------------------------------- plan
// Entries of the routing in plan.ids and plan.chosen, by a whole CTA. Bit masks and ballots: nothing depends on timing.
__device__ __forceinline__ void make_plan(Plan& plan, int tokens, int topk) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pairs = tokens * topk;
  static_assert(THREADS == MAX_TOKENS * MAX_EXPERTS / 32 && THREADS >= MAX_PAIRS, "one mask word, one pair a thread");
  __syncthreads();
  const int my_token = tid / topk, e = tid < pairs ? plan.ids[tid] : 0;
  int slot = 1, all = 0;                       // tokens before this one that chose the expert, and all that did
  if (tid < pairs) {
    slot = 0;
    for (int t = 0; t < tokens; ++t) {
      const int in = (plan.chosen[t][e >> 5] >> (e & 31)) & 1;
      all += in;
      slot += t < my_token ? in : 0;
    }
  }
  const bool start = slot % COLS == 0;
  const uint32_t starts = __ballot_sync(0xffffffffu, start);
  if (lane == 0) plan.starts[warp] = __popc(starts);
  __syncthreads();
  int before = lane < THREADS / 32 ? plan.starts[lane] : 0;
  const int total = __reduce_add_sync(0xffffffffu, before);
  const int entry = __reduce_add_sync(0xffffffffu, lane < warp ? before : 0) + __popc(starts & ((1u << lane) - 1u));
  if (tid == 0) plan.entries = total;
  if (start) {
    plan.expert[entry] = static_cast<unsigned short>(e);
    plan.count[entry] = static_cast<unsigned short>(min(COLS, all - slot));
    plan.pair[entry * COLS] = static_cast<unsigned short>(tid);
    plan.entry_of[e * 2 + slot / COLS] = static_cast<unsigned short>(entry);
  }
  __syncthreads();
  if (tid < pairs && !start) plan.pair[plan.entry_of[e * 2 + slot / COLS] * COLS + slot % COLS] = static_cast<unsigned short>(tid);
  __syncthreads();
}

// Orders floats as unsigned numbers, NaN in front of all; never 0. (NaN is asked for by itself: the compiler may make `b | 0x80000000` a
// floating-point -|v|, which turns a NaN into one without the sign bit, between the positive and the negative numbers.)
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return v != v ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Top-k of one token by one warp, PER experts a lane. Lane j < topk returns id and weight, in descending order of score
// (+ bias), ties by the lower id, as `route` orders them; softmax scores are ordered by their logits, and only the chosen ones'
// (renorm) are computed. No lane whose best key is below the topk-th largest of the 32 lanes' best keys can hold a chosen
// expert; that threshold is moved up until 32 candidates or fewer are left, which rank themselves. Where equal scores keep them
// above CANDIDATES, they are found one by one.
template <int PER>
__device__ __forceinline__ void warp_topk(const FewParams& p, const float* logit, uint32_t* cand_key, uint32_t* cand_id, int& id,
                                          float& weight) {
  const int lane = threadIdx.x & 31, E = p.experts, K = p.topk;
  float s[PER];
  uint32_t key[PER], best = 0;
  const bool biased = p.sigmoid && p.sel_bias != nullptr;
#pragma unroll
  for (int i = 0; i < PER; ++i) s[i] = i * 32 + lane < E ? ld_step(logit + i * 32 + lane) : -INFINITY;
  if (p.sigmoid) {
    float b[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) b[i] = biased && i * 32 + lane < E ? ld_step(p.sel_bias + i * 32 + lane) : 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = __fdividef(1.f, 1.f + __expf(-s[i]));
      key[i] = order_key(s[i] + b[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = order_key(s[i]);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = i * 32 + lane < E ? key[i] : 0u;
    best = max(best, key[i]);
  }
  int rank = 0;
#pragma unroll 8
  for (int i = 0; i < 32; ++i) {
    const uint32_t other = __shfl_sync(0xffffffffu, best, i);
    rank += other > best || (other == best && i < lane);
  }
  uint32_t thr = max(__shfl_sync(0xffffffffu, best, __ffs(__ballot_sync(0xffffffffu, rank == K - 1)) - 1), 1u);
  uint32_t high = __reduce_max_sync(0xffffffffu, best);
  auto count = [&](uint32_t at_least) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) c += key[i] >= at_least;
    return c;
  };
  int mine = count(thr), n = __reduce_add_sync(0xffffffffu, mine);
  while (n > 32 && high - thr > 1) {        // at least K keys are >= thr all the time, fewer than K are >= high (or one value is left)
    const uint32_t mid = thr + (high - thr) / 2;
    const int c = count(mid), all = __reduce_add_sync(0xffffffffu, c);
    if (all >= K) {
      thr = mid;
      mine = c;
      n = all;
    } else {
      high = mid;
    }
  }
  int at = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += up;
  }
  at -= mine;
  id = 0;
  if (n <= CANDIDATES) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] >= thr) {
        cand_key[at] = key[i];
        cand_id[at++] = i * 32 + lane;
      }
    __syncwarp();
    for (int c = lane; c < n; c += 32) {
      const uint32_t k = cand_key[c], e = cand_id[c];
      int place = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const uint32_t ok = cand_key[i], oe = cand_id[i];
        place += ok > k || (ok == k && oe < e);
      }
      if (place < K) cand_id[CANDIDATES + place] = e;
    }
    __syncwarp();
    if (lane < K) id = static_cast<int>(cand_id[CANDIDATES + lane]);
  } else {
    for (int j = 0; j < K; ++j) {
      uint32_t top_mine = 0;
      int e = lane;
#pragma unroll
      for (int i = PER - 1; i >= 0; --i)
        if (key[i] >= top_mine && key[i] != 0) {
          top_mine = key[i];
          e = i * 32 + lane;
        }
      const uint32_t top = __reduce_max_sync(0xffffffffu, top_mine);
      const int win = static_cast<int>(__reduce_min_sync(0xffffffffu, top_mine == top ? static_cast<uint32_t>(e) : 0x7FFFFFFFu));
      if (lane == j) id = win;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i * 32 + lane == win) key[i] = 0;
    }
  }
  // the chosen ones' scores (softmax: logits so far): lane id % 32 has the one of expert `id` in s[id / 32]
  weight = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float v = __shfl_sync(0xffffffffu, s[i], id & 31);
    if ((id >> 5) == i) weight = v;
  }
  if (lane >= K) weight = p.sigmoid ? 0.f : -INFINITY;
  if (!p.sigmoid) {
    const float mx = __shfl_sync(0xffffffffu, weight, 0);
    weight = __expf(weight - mx);
    if (!p.renorm) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += __expf(s[i] - mx);
      weight /= warp_sum(sum);
    }
  }
  if (p.renorm) {
    const float sum = warp_sum(weight);
    weight = weight / (sum < 1e-20f ? 1e-20f : sum);          // (fmaxf would put the bound in a NaN's place)
  }
  weight *= p.scale;
}

// ---------------------------------------------------------------- the experts' products
// Tile load of what is read once: first to leave L2, which holds instructions, activations and the router otherwise.
__device__ __forceinline__ void tma_load_2d_once(uint32_t smem_dst, const CUtensorMap* m, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n\t.reg .b64 pol;\n\t"
      "createpolicy.fractional.L2::evict_first.b64 pol, 1.0;\n\t"
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], pol;\n\t}" ::"r"(
          smem_dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__host__ __device__ constexpr int align_to(int v, int a) { return (v + a - 1) / a * a; }
constexpr int BAR_BYTES = (3 * MAX_STAGES + 8) * 8;
// Shared memory, from a 1024-byte boundary on: fc1: B tiles of x | stages | scales of x | candidates of the top-k | plan | barriers;
// fc2: stages | sums [2][tokens][128] | scales of one | plan | barriers
__host__ __device__ inline int k_tiles_of(int k, int tile) { return (k + tile - 1) / tile; }
template <int KIND>
__host__ __device__ inline int fc1_fixed_bytes(int tokens, int n, int hidden) {
  using T = Traits<KIND>;
  return 1024 + k_tiles_of(hidden, T::TILE_K) * (n * 128 + T::SF_BYTES) + tokens * CAND_BYTES + align_to(sizeof(Plan), 16) + BAR_BYTES;
}
template <int KIND>
__host__ __device__ constexpr int fc2_fixed_bytes(int tokens) {
  return 1024 + 2 * tokens * 512 + 512 + align_to(sizeof(Plan), 16) + BAR_BYTES;
}
constexpr int ACC_COLS = 96;              // two accumulators, then scales of A (a tile's of each) and of B (all tiles' where they fit)
constexpr int SFA_COL = 192, SFB_COL = 224;
constexpr int TMEM_COLS = 512;

template <int KIND, bool SECOND>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_experts_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ FewParams p) {
  using T = Traits<KIND>;
  constexpr int STAGE = SECOND ? T::STAGE2 : T::STAGE1;
  constexpr int P = SECOND ? T::MP : T::XP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int K = SECOND ? p.inter : p.hidden, k_tiles = k_tiles_of(K, T::TILE_K);
  const int x_bytes = SECOND ? 0 : k_tiles * p.n * 128, xsf_bytes = SECOND ? 0 : k_tiles * T::SF_BYTES;
  uint8_t* ring = sm + x_bytes;
  uint8_t* after = ring + p.stages * STAGE;
  float* sums = reinterpret_cast<float*>(after);                                // fc2: [2][tokens][128]
  uint8_t* xsf = SECOND ? after + 2 * p.tokens * 512 : after;                   // scales of operand B
  uint8_t* plan_at = after + (SECOND ? 2 * p.tokens * 512 + 512 : xsf_bytes + p.tokens * CAND_BYTES);
  Plan& plan = *reinterpret_cast<Plan*>(plan_at);
  uint64_t* full = reinterpret_cast<uint64_t*>(plan_at + align_to(sizeof(Plan), 16));
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* b_full = empty + MAX_STAGES;      // fc2: the stage's B tile has been written
  uint64_t* accum = b_full + MAX_STAGES;      // [2] accumulator complete
  uint64_t* acc_free = accum + 2;             // [2] and read back (four warps)
  uint64_t* x_full = acc_free + 2;
  uint64_t* sfb_full = x_full + 1;            // scales of B that stay are in tensor memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sfb_full + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t cluster_n = 1, cluster_rank = 0;
  if constexpr (SECOND) {
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cluster_n));
    cluster_rank = cluster_ctarank();
  }

  if (tid == 0) {
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&b_full[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accum[i], 1);
      mbar_init(&acc_free[i], 4);
    }
    mbar_init(x_full, 1);
    mbar_init(sfb_full, 1);
    *abort = 0;
    fence_mbar_init();
    prefetch_tmap(&tw);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if constexpr (SECOND) {
    for (int i = tid; i < 2 * p.tokens * 128; i += THREADS) sums[i] = 0.f;
    if (tid < 128) reinterpret_cast<uint32_t*>(xsf)[tid] = KIND == kGemmMxfp4 ? 0x7F7F7F7Fu : 0x38383838u;
    fence_proxy_async_smem();
  } else {
    (&plan.chosen[0][0])[tid] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_dep_wait();
  grid_dep_launch();

  const int pairs = p.tokens * p.topk;
  if constexpr (SECOND) {
    if (tid < pairs) {                        // (records past the last entry hold anything: nobody asks for them)
      const EntryRecord* rec = p.entries + tid;
      const uint4 head = ld_step(reinterpret_cast<const uint4*>(rec)), cols = ld_step(reinterpret_cast<const uint4*>(rec->pair));
      const uint4 w0 = ld_step(reinterpret_cast<const uint4*>(rec->weight)), w1 = ld_step(reinterpret_cast<const uint4*>(rec->weight + 4));
      const int entries = ld_step(&p.entries->entries);
      if (tid == 0) plan.entries = entries;
      plan.expert[tid] = static_cast<unsigned short>(head.x);
      plan.count[tid] = static_cast<unsigned short>(head.y);
      *reinterpret_cast<uint4*>(plan.pair + tid * COLS) = cols;
      const uint32_t c[4] = {cols.x, cols.y, cols.z, cols.w}, w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int j = 0; j < COLS; ++j)
        if (tid < entries && j < static_cast<int>(head.y)) plan.weights[(c[j >> 1] >> (16 * (j & 1))) & 0xFFFFu] = __uint_as_float(w[j]);
    }
    __syncthreads();
  } else {
    if (warp == 15 && lane == 0) {            // (the last warp to get a token)
      mbar_expect_tx(x_full, x_bytes + xsf_bytes);
      bulk_load(sm, p.x_img, x_bytes, x_full);      // (a copy takes this lane 0.3 us: tile by tile they held up the plan)
      if (xsf_bytes > 0) bulk_load(xsf, p.x_img + x_bytes, xsf_bytes, x_full);
    }
    __syncwarp();
    if (warp < p.tokens) {
      uint32_t* cand = reinterpret_cast<uint32_t*>(xsf + xsf_bytes + warp * CAND_BYTES);
      const float* logit = p.logits + warp * p.experts;
      int id;
      float w;
      if (p.experts <= 128) warp_topk<4>(p, logit, cand, cand + CANDIDATES, id, w);
      else if (p.experts <= 512) warp_topk<16>(p, logit, cand, cand + CANDIDATES, id, w);
      else warp_topk<32>(p, logit, cand, cand + CANDIDATES, id, w);
      if (lane < p.topk) {
        const int at = warp * p.topk + lane;
        plan.ids[at] = id;
        plan.weights[at] = w;
        atomicOr(&plan.chosen[warp][id >> 5], 1u << (id & 31));
      }
    }
    make_plan(plan, p.tokens, p.topk);
    if (blockIdx.x == 0 && tid < plan.entries) {
      EntryRecord rec;
      rec.expert = plan.expert[tid];
      rec.count = plan.count[tid];
      rec.entries = plan.entries;
      rec.unused = 0;
#pragma unroll
      for (int j = 0; j < COLS; ++j) {
        const bool in = j < rec.count;
        rec.pair[j] = in ? plan.pair[tid * COLS + j] : 0;
        rec.weight[j] = in ? plan.weights[rec.pair[j]] : 0.f;
      }
      p.entries[tid] = rec;
    }
  }

  // Units: fc1: (entry, 128 weight rows), round the CTAs; fc2: the entries of this CTA of the cluster, on its 128 output rows.
  const int rows_per_expert = SECOND ? p.h_out : p.swiglu ? 2 * p.inter : p.inter;
  const int tiles = SECOND ? 1 : (rows_per_expert + 127) / 128;
  // (shuffled, so that the compiler knows that the warps' loops are uniform: the operands of tcgen05 and TMA instructions then live
  // in uniform registers. Bounds straight from shared memory cost 0.45 us per K tile, more than its bytes take.)
  const int units = __shfl_sync(0xffffffffu, plan.entries, 0) * tiles;
  const int u0 = SECOND ? __shfl_sync(0xffffffffu, static_cast<int>(cluster_rank), 0) : static_cast<int>(blockIdx.x);
  const int stride = SECOND ? __shfl_sync(0xffffffffu, static_cast<int>(cluster_n), 0) : static_cast<int>(gridDim.x);
  const int out_block = SECOND ? static_cast<int>(blockIdx.x) / stride : 0;

  if constexpr (SECOND && T::kFp4) {          // the largest exponent of every row this CTA reads
    const int words = (p.swiglu ? 2 * p.inter : p.inter) / 128;      // of four exponents
    for (int u = u0 + warp * stride; u < units; u += WARPS * stride)
      for (int c = 0; c < plan.count[u]; ++c) {
        const int pr = plan.pair[u * COLS + c];
        uint32_t m = 0;
        for (int i = lane; i < words; i += 32)
          m = __vmaxu4(m, ld_step(reinterpret_cast<const uint32_t*>(p.mid_exp + static_cast<size_t>(pr) * p.exp_ld) + i));
        m = __vmaxu4(m, m >> 16);
        m = __reduce_max_sync(0xffffffffu, max(m & 255u, (m >> 8) & 255u));
        if (lane == 0) plan.row_exp[pr] = static_cast<int>(m);
      }
    __syncthreads();
  }

  // Streams: warps that issue MMAs, each with its share of the stages. A K tile's waits, copies of scales, MMAs and commits take one warp
  // 460 cycles, 0.24 us; the 16 KB of one on each of 120 SMs are 0.3 at memory's rate, on fewer SMs less. fc2 with one warp and with two,
  // 8 and 16 tokens: 256 bf16 experts, top 22, 1024-2688 169 / 149 and 238 / 213 us, 512 MXFP4 ones 63 / 57 and 100 / 85; 256 of bf16,
  // top 10, 2560-640 56 / 54 and 83 / 82. fc1 has all SMs, and a unit without a second has half the stages, so two streams lose where
  // every CTA has work to the end (16 tokens over 64 bf16 experts 67 / 70, 512 MXFP4 ones 51 / 55) or the last units stand alone (one
  // token 21 / 25). They win where the last round is the second of a pair and sparse: the CTAs with one unit more then have it beside
  // their last but one (8 tokens over 64 bf16 experts 54 / 51, one over 256, top 22, 33 / 29).
  const int rounds = (units + stride - 1) / stride;
  const bool two = SECOND || (p.stages >= 6 && rounds % 2 == 0 && 2 * (rounds * stride - units) >= stride);
  const int streams = two ? 2 : 1, S = two ? p.stages & ~1 : p.stages;
  // With two streams units go in pairs, K tile by K tile: the first's stages are the even ones, the second's the odd ones.
  const uint32_t ring_addr = __shfl_sync(0xffffffffu, smem_u32(ring), 0), xsf_addr = __shfl_sync(0xffffffffu, smem_u32(xsf), 0);
  int issued = 0, alone = 0x7FFFFFFF;         // warp 0: tiles asked for so far; from `alone` on every other place is left out
  if (warp == 0) {
    // ---- weights: the whole warp walks the loop (waits included), one elected lane issues
    int i = 0, s = 0;                         // place in the ring's order
    uint32_t phase = 1;                       // (the first round finds every stage free)
    bool ok = true;
    for (int u = u0; u < units && ok; u += streams * stride) {
      const int of_pair = two && u + stride < units ? 2 : 1;
      if (two && of_pair == 1) alone = i;
      int rows[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int v = h < of_pair ? u + h * stride : u, entry = v / tiles;
        rows[h] = __shfl_sync(0xffffffffu, static_cast<int>(plan.expert[entry]) * rows_per_expert +
                                               (SECOND ? out_block : v - entry * tiles) * 128, 0);
      }
      for (int kt = 0; kt < k_tiles && ok; ++kt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h >= of_pair || !ok) break;
          const int at = s + h, row0 = rows[h];
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[at], phase, abort, p.status, kTimeoutEmpty));
          if (!ok) break;
          if (elect_one()) {
            const uint32_t st = ring_addr + at * STAGE, bar = smem_u32(&full[at]);
            mbar_expect_tx(&full[at], A_BYTES + T::SF_BYTES);
            tma_load_2d_once(st, &tw, bar, kt * (T::kFp4 ? 128 : 64), row0);
            if constexpr (T::kFp4)
              bulk_load(st + A_BYTES, (SECOND ? p.sf2 : p.sf1) + (static_cast<size_t>(row0 >> 7) * (SECOND ? p.ka2 : p.ka1) + kt * T::ATOMS) * 512,
                        T::SF_BYTES, bar);
          }
          __syncwarp();
          ++i;
        }
        if (!ok) break;
        i += streams - of_pair;
        s += streams;
        if (s == S) {
          s = 0;
          phase ^= 1;
        }
      }
    }
    issued = i;
    __syncwarp();
  } else if (warp == 1 || (two && warp == 3)) {
    // ---- products
    const int set = warp >> 1;
    int s = set, it = 0;                      // (of this warp's units)
    uint32_t phase = 0;
    bool ok = true, ready = false;
    if constexpr (!SECOND) ok = __all_sync(0xffffffffu, mbar_wait(x_full, 0, abort, p.status, kTimeoutFull));
    // Scales of B that stay: fc2's are one; fc1's are every tile's, for as many columns as there are (a wider NVFP4 row copies them
    // tile by tile). Each copy is 0.02 us of this warp's time per tile, which is what bounds a CTA that has its bytes.
    const bool resident = SECOND || SFB_COL + k_tiles * T::ATOMS * 4 <= TMEM_COLS;
    if constexpr (T::kFp4) {
      tc_fence_after();
      // (not by a CTA without a unit: nobody there waits for these copies, and it would leave while they run)
      if (resident && set == 0 && u0 < units && ok && elect_one()) {
        for (int at = 0; at < (SECOND ? 1 : k_tiles * T::ATOMS); ++at)
          tmem_cp_32x128b_x4(tmem + SFB_COL + at * 4, make_desc_sf(xsf_addr + at * 512));
        tc_commit(sfb_full);
      }
      __syncwarp();
      if (resident && set == 1 && u0 + stride < units && ok) ok = __all_sync(0xffffffffu, mbar_wait(sfb_full, 0, abort, p.status, kTimeoutAccum));
    }
    const uint32_t sfa = tmem + SFA_COL + set * 16;
    for (int u = u0 + set * stride; u < units && ok; u += streams * stride, ++it) {
      const int buf = two ? set : it & 1, turn = two ? it : it >> 1;      // accumulator, and its use
      const uint32_t acc = tmem + buf * ACC_COLS;
      const int n = __shfl_sync(0xffffffffu, SECOND ? (plan.count[u] * P + 15) / 16 * 16 : p.n, 0);
      if (turn >= 1) ok = __all_sync(0xffffffffu, mbar_wait(&acc_free[buf], (turn - 1) & 1, abort, p.status, kTimeoutAccum));
      if (!ok) break;
      tc_fence_after();
      for (int kt = 0; kt < k_tiles; ++kt) {
        if (!ready) {
          ok = __all_sync(0xffffffffu, mbar_wait(&full[s], phase, abort, p.status, kTimeoutFull));
          if (SECOND && ok) ok = __all_sync(0xffffffffu, mbar_wait(&b_full[s], phase, abort, p.status, kTimeoutFull));
        }
        if (!ok) break;
        tc_fence_after();
        const int s_at = s;
        s += streams;
        if (s >= S) {
          s = set;
          phase ^= 1;
        }
        // Of the next tile, answered while this one is issued: a wait that finds its barrier complete takes 0.1 us all the same. In fc2
        // odd lanes ask for B: one test of both.
        const bool peek = mbar_test_wait((SECOND && (lane & 1) ? b_full : full) + s, phase);
        const uint32_t st = ring_addr + s_at * STAGE;
        const uint32_t b_at = SECOND ? st + A_BYTES + T::SF_BYTES : ring_addr - x_bytes + kt * p.n * 128;
        const uint32_t sfb = tmem + SFB_COL + (SECOND ? 0 : resident ? kt * T::ATOMS * 4 : set * 16);
        const uint64_t adesc = make_desc_sw128(st), bdesc = make_desc_sw128(b_at);
        const int mmas = min(4, (K - kt * T::TILE_K + T::MMA_K - 1) / T::MMA_K);
        if (elect_one()) {
          if constexpr (T::kFp4) {
#pragma unroll
            for (int at = 0; at < T::ATOMS; ++at) tmem_cp_32x128b_x4(sfa + at * 4, make_desc_sf(st + A_BYTES + at * 512));
            if (!SECOND && !resident) {
#pragma unroll
              for (int at = 0; at < T::ATOMS; ++at) tmem_cp_32x128b_x4(sfb + at * 4, make_desc_sf(xsf_addr + kt * T::SF_BYTES + at * 512));
            }
          }
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) {
            if (kb >= mmas) break;
            const uint32_t more = kt > 0 || kb > 0 ? 1u : 0u;
            if constexpr (KIND == kGemmMxfp4)
              mma_mxf4(acc, adesc + kb * 2, bdesc + kb * 2, make_idesc_mxf4(128, 0, kb & 1) | static_cast<uint32_t>(n >> 3) << 17, more,
                       sfa + (kb >> 1) * 4, SECOND ? sfb : sfb + (kb >> 1) * 4);
            else if constexpr (KIND == kGemmNvfp4)
              mma_nvf4(acc, adesc + kb * 2, bdesc + kb * 2, make_idesc_nvf4(128, 0) | static_cast<uint32_t>(n >> 3) << 17, more,
                       sfa + kb * 4, SECOND ? sfb : sfb + kb * 4);
            else
              mma_f16(acc, adesc + kb * 2, bdesc + kb * 2, make_idesc_bf16(128, 0) | static_cast<uint32_t>(n >> 3) << 17, more);
          }
          tc_commit(&empty[s_at]);
          if (kt == k_tiles - 1) tc_commit(&accum[buf]);
        }
        ready = __all_sync(0xffffffffu, peek);
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // ---- accumulators: group `set` takes every other unit; thread = row
    const int set = (warp - 4) >> 2, q = warp & 3, row_in = q * 32 + lane;
    const uint32_t acc = tmem + set * ACC_COLS + (static_cast<uint32_t>(q * 32) << 16);
    int it = set;
    for (int u = u0 + set * stride; u < units; u += 2 * stride, it += 2) {
      if (!__all_sync(0xffffffffu, mbar_wait(&accum[set], (it >> 1) & 1, abort, p.status, kTimeoutAccum))) break;
      tc_fence_after();
      const int entry = u / tiles, tile = u - entry * tiles, n = plan.count[entry], expert = plan.expert[entry];
      const float* gp = SECOND ? p.gs2 : p.gs1;
      const float gs = KIND == kGemmNvfp4 ? ld_step(gp + expert) : 1.f;
      const int row = tile * 128 + row_in;
#pragma unroll 1
      for (int c = 0; c < n; ++c) {
        const int pr = plan.pair[entry * COLS + c], tok = pr / p.topk;
        uint32_t r[8];
        tmem_ld_32x8(acc + (SECOND ? c : tok) * P, r);
        tmem_ld_wait();
        if (c == n - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_free[set]);
        }
        float v = __uint_as_float(r[P - 1]);
#pragma unroll
        for (int i = P - 2; i >= 0; --i) v = fmaf(v, T::kFp4 ? 8.f : 1.f, __uint_as_float(r[i]));
        if constexpr (SECOND) {
          const float f = T::kFp4 ? mid_back(plan.row_exp[pr]) * gs : gs;
          sums[(set * p.tokens + tok) * 128 + row_in] += v * f * plan.weights[pr];
        } else {
          v *= KIND == kGemmNvfp4 ? ld_step(p.x_factor + tok) * gs : gs;
          if (p.swiglu) {
            const float up = __shfl_xor_sync(0xffffffffu, v, 1);      // rows come in pairs: gate, up
            v = v / (1.f + __expf(-v)) * up;
          } else {
            v = v <= 0.f ? 0.f : v * v;                               // (a NaN stays one)
          }
          const bool mine = row < rows_per_expert && (!p.swiglu || (lane & 1) == 0);
          if (mine) p.mid[static_cast<size_t>(pr) * p.inter + (p.swiglu ? row >> 1 : row)] = v;
          if constexpr (T::kFp4) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, mine ? magnitude(v) : 0u);
            if (lane == 0) p.mid_exp[static_cast<size_t>(pr) * p.exp_ld + tile * 4 + q] = static_cast<uint8_t>(m >> 23);
          }
        }
      }
    }
  } else if (SECOND && warp >= 12) {
    // ---- rows of mid: two warps write the B tiles of the even stages in turn, two those of the odd ones. (A warp sees two of a stage's
    // uses apart by its parity only, so the tiles it takes are never more than a ring apart among those of one MMA warp.)
    const int set = warp & 1;
    int s = set, turns = (warp >> 1) & 1;     // the stage of the tile at hand; tiles until this warp's next one
    uint32_t phase = 1;
    bool ok = true;
    for (int u = u0 + set * stride; u < units && ok; u += 2 * stride) {
      const int n = plan.count[u];
      for (int kt = 0; kt < k_tiles; ++kt) {
        const int mine = s;
        const uint32_t turn = phase;
        s += 2;
        if (s >= S) {
          s = set;
          phase ^= 1;
        }
        if (turns-- != 0) continue;
        turns = 1;
        // (of FP4 a warp takes a row at a time, of bf16 four; the first numbers are under way before the stage is free)
        constexpr int LANES = T::TILE_K / 8, STEP = 32 / LANES;
        const int k = kt * T::TILE_K + (lane % LANES) * 8;
        float v[8], next[8];
        auto fetch = [&](int c, float (&to)[8]) {
#pragma unroll
          for (int e = 0; e < 8; ++e) to[e] = 0.f;
          if (c < n && k < p.inter) {
            const float4* at = reinterpret_cast<const float4*>(p.mid + static_cast<size_t>(plan.pair[u * COLS + c]) * p.inter + k);
            const float4 lo = ld_step(at), hi = ld_step(at + 1);
            to[0] = lo.x; to[1] = lo.y; to[2] = lo.z; to[3] = lo.w; to[4] = hi.x; to[5] = hi.y; to[6] = hi.z; to[7] = hi.w;
          }
        };
        fetch(lane / LANES, next);
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[mine], turn, abort, p.status, kTimeoutEmpty));
        if (!ok) break;
        uint8_t* b = ring + mine * STAGE + A_BYTES + T::SF_BYTES;
#pragma unroll 1
        for (int c = lane / LANES; c < n; c += STEP) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = next[e];
          fetch(c + STEP, next);
          if constexpr (T::kFp4) {
            uint32_t w[5];
            digits8(v, mid_factor(plan.row_exp[plan.pair[u * COLS + c]]), w);
#pragma unroll
            for (int d = 0; d < 5; ++d) *reinterpret_cast<uint32_t*>(b + b_offset(c * 5 + d, lane * 4)) = w[d];
          } else {
            float h[8];
            const uint4 top = pack8(v);
            unpack8(top, h);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = fabsf(h[e]) == INFINITY ? 0.f : v[e] - h[e];
            *reinterpret_cast<uint4*>(b + b_offset(2 * c, (lane & 7) * 16)) = top;
            *reinterpret_cast<uint4*>(b + b_offset(2 * c + 1, (lane & 7) * 16)) = pack8(h);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_full[mine]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort) {                               // (one answer for the whole CTA: behind the barrier nobody raises it any more)
    // bounded wait for the copies still in flight, whichever warp gave up: none may land after the CTA has gone
    if (tid == 0) {
      volatile int ignore = 0;
      if constexpr (!SECOND) mbar_wait(x_full, 0, &ignore, nullptr, kTimeoutDrain);
      for (int j = max(issued - S, 0); j < issued; ++j)
        if (j < alone || (j & 1) == 0) mbar_wait(&full[j % S], (j / S) & 1, &ignore, nullptr, kTimeoutDrain);
    }
    __syncthreads();
  }
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
  if constexpr (SECOND) {
    const int n_out = p.tokens * 128;
    for (int i = tid; i < n_out; i += THREADS) sums[i] += sums[n_out + i];
    if (cluster_n > 1) cluster_sync_all();
    else __syncthreads();
    for (int i = tid + static_cast<int>(cluster_rank) * THREADS; i < n_out; i += THREADS * static_cast<int>(cluster_n)) {
      float s = 0.f;
      if (cluster_n > 1) {                  // all loads under way before the first sum
        const uint32_t at = smem_u32(sums + i);
        float part[MAX_CLUSTER];
#pragma unroll
        for (uint32_t r = 0; r < MAX_CLUSTER; ++r) part[r] = r < cluster_n ? ld_dsmem_f32(map_to_cta(at, r)) : 0.f;
#pragma unroll
        for (uint32_t r = 0; r < MAX_CLUSTER; ++r) s += part[r];
      } else {
        s = sums[i];
      }
      const int tok = i >> 7, row = out_block * 128 + (i & 127);
      if (row < p.h_out) {
        if (p.shared != nullptr) s += __bfloat162float(p.shared[tok * p.ld_shared + row]);
        p.out[tok * p.ldo + row] = __float2bfloat16(s);
      }
    }
    if (cluster_n > 1) cluster_sync_all();     // nobody leaves while a peer may still read its sums
  }
}

// Clusters of `size` CTAs of the second kernel that the chip holds at once (0: none).
template <int KIND>
int resident(int size) {
  static DeviceCounts<MAX_CLUSTER + 1> known;
  return known.get(device_index(), size, [size] {
    int n = 0;
    cudaLaunchConfig_t q = {};
    q.gridDim = dim3(size);
    q.blockDim = dim3(THREADS);
    q.dynamicSmemBytes = MAX_SMEM;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    q.attrs = at;
    q.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, moe_few_experts_kernel<KIND, true>, &q) != cudaSuccess) {
      (void)cudaGetLastError();
      n = -1;
    }
    return n;
  });
}

template <int KIND>
int fc1_stages(int tokens, int n, int hidden) {
  return std::min(MAX_STAGES, (MAX_SMEM - fc1_fixed_bytes<KIND>(tokens, n, hidden)) / Traits<KIND>::STAGE1);
}
int columns(int tokens, int per) { return (tokens * per + 15) / 16 * 16; }

// Most tokens of a call: at least two stages of weights beside the rows of x.
template <int KIND>
int most_tokens(int hidden) {
  for (int t = MAX_TOKENS; t > 0; --t)
    if (fc1_stages<KIND>(t, columns(t, Traits<KIND>::XP), hidden) >= 2) return t;
  return 0;
}

struct WsLayout {
  long long logits, factor, img, entries, mid, exp, bytes;
  int exp_ld;
};
template <int KIND>
WsLayout ws_layout(int tokens, int experts, int topk, int hidden, int inter) {
  using T = Traits<KIND>;
  const auto up = [](long long v) { return (v + 127) / 128 * 128; };
  const long long pairs = static_cast<long long>(tokens) * topk;
  WsLayout w;
  w.exp_ld = align_to((2 * inter + 127) / 128 * 4, 16);
  w.img = 0;
  w.mid = up(static_cast<long long>(k_tiles_of(hidden, T::TILE_K)) * (columns(tokens, T::XP) * 128 + T::SF_BYTES));
  w.logits = w.mid + up(pairs * inter * 4);
  w.factor = w.logits + up(4ll * tokens * experts);
  w.entries = w.factor + up(4ll * tokens);
  w.exp = w.entries + up(sizeof(EntryRecord) * pairs);
  w.bytes = w.exp + up(pairs * w.exp_ld);
  return w;
}

template <int KIND>
cudaError_t launch_few(FewParams& p, const void* w1, const void* w2, uint8_t* ws, cudaStream_t st) {
  using T = Traits<KIND>;
  auto k1 = moe_few_experts_kernel<KIND, false>;
  auto k2 = moe_few_experts_kernel<KIND, true>;
  static bool ready[kMaxDevices] = {};
  if (bool& done = ready[device_index()]; !done) {
    cudaError_t e = cudaFuncSetAttribute(k1, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k2, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k2, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    done = true;
  }
  const WsLayout w = ws_layout<KIND>(p.tokens, p.experts, p.topk, p.hidden, p.inter);
  p.x_img = ws + w.img;
  p.mid = reinterpret_cast<float*>(ws + w.mid);
  p.logits = reinterpret_cast<float*>(ws + w.logits);
  p.x_factor = reinterpret_cast<float*>(ws + w.factor);
  p.entries = reinterpret_cast<EntryRecord*>(ws + w.entries);
  p.mid_exp = ws + w.exp;
  p.exp_ld = w.exp_ld;
  p.n = columns(p.tokens, T::XP);
  const int n1 = p.swiglu ? 2 * p.inter : p.inter;
  const auto map = [&](const void* base, int rows, int k, CUtensorMap* out) {
    const TmapKey key{base, static_cast<uint64_t>(p.experts) * rows, static_cast<uint64_t>(T::kFp4 ? k / 2 : k),
                      static_cast<uint64_t>(T::kFp4 ? k / 2 : k * 2), 128u, T::kFp4 ? 128u : 64u, T::kFp4 ? 1 : 0};
    return get_tmap_2d(key, out);
  };
  CUtensorMap t1, t2;
  if (!map(w1, n1, p.hidden, &t1) || !map(w2, p.h_out, p.inter, &t2)) return cudaErrorInvalidValue;
  cudaError_t e = launch_dep(moe_few_route_kernel<KIND>, dim3((p.experts + 15) / 16 + p.tokens), dim3(ROUTE_WARPS * 32), 0, st, p);
  if (e != cudaSuccess) return e;
  p.stages = fc1_stages<KIND>(p.tokens, p.n, p.hidden);
  e = launch_dep(k1, dim3(kNumSms), dim3(THREADS), MAX_SMEM, st, t1, p);
  if (e != cudaSuccess) return e;
  static_assert((MAX_SMEM - fc2_fixed_bytes<KIND>(MAX_TOKENS)) / T::STAGE2 >= 4, "what the converters' waits rest on");
  p.stages = std::min(MAX_STAGES, (MAX_SMEM - fc2_fixed_bytes<KIND>(p.tokens)) / T::STAGE2) & ~1;
  // CTAs of a cluster share an output block's experts: the number that leaves each the least to do
  const int blocks = (p.h_out + 127) / 128;
  int cluster = 1;
  double best = 1e30;
  for (int c = 1; c <= MAX_CLUSTER; ++c) {
    const int room = resident<KIND>(c);
    if (room < 1) continue;
    const double cost = static_cast<double>((blocks + room - 1) / room) / c;
    if (cost < best) {
      best = cost;
      cluster = c;
    }
  }
  return launch_dep_cluster(k2, dim3(blocks * cluster), dim3(THREADS), cluster, MAX_SMEM, st, t2, p);
}

}  // namespace
}  // namespace hb

extern "C" {

#define HB_FEW_KIND(CALL)                                        \
  (kind == hb::kGemmMxfp4 ? CALL(hb::kGemmMxfp4) : kind == hb::kGemmNvfp4 ? CALL(hb::kGemmNvfp4) : CALL(hb::kGemmBf16))

// Most tokens that one call takes at this width (0: none).
int hb_moe_few_tokens(int kind, int hidden) {
#define HB_CALL(K) hb::most_tokens<K>(hidden)
  return HB_FEW_KIND(HB_CALL);
#undef HB_CALL
}
// Workspace bytes of a call (-1: too large).
int hb_moe_few_ws(int kind, int tokens, int experts, int topk, int hidden, int inter) {
#define HB_CALL(K) hb::ws_layout<K>(tokens, experts, topk, hidden, inter).bytes
  const long long n = HB_FEW_KIND(HB_CALL);
#undef HB_CALL
  return n > 0x7FFFFFFF ? -1 : static_cast<int>(n);
}

int hb_moe_few(int kind, const void* x, long long ldx, const void* route_x, long long ld_route, const void* router,
               long long ld_router, int route_k, const void* sel_bias, int tokens, int experts, int topk, int sigmoid, int renorm,
               float scale, int hidden, int inter, int h_out, int swiglu, const void* w1, const void* sf1, const void* gs1, int ka1,
               const void* w2, const void* sf2, const void* gs2, int ka2, const void* shared, long long ld_shared, void* out,
               long long ldo, void* ws, void* status, void* stream) {
  using namespace hb;
  const bool fp4 = is_fp4(kind);
  if (!fp4 && kind != kGemmBf16) return 1;
  if (tokens < 1 || experts < 1 || experts > MAX_EXPERTS || topk < 1 || topk > MAX_TOPK || topk > experts) return 1;
  const int n1 = swiglu ? 2 * inter : inter, rows = fp4 ? 128 : 8, k_of = fp4 ? 32 : 8;
  if (hidden < 1 || inter < 1 || n1 % rows || h_out < 1 || h_out % rows || hidden % k_of || inter % k_of) return 1;
  if (tokens > hb_moe_few_tokens(kind, hidden)) return 1;
  if (router == nullptr || route_x == nullptr || route_k < 8 || route_k % 8) return 1;
  const int tile = fp4 ? 256 : 64;
  if (fp4 && (ka1 < (hidden + tile - 1) / tile * sf_atoms(kind) || ka2 < (inter + tile - 1) / tile * sf_atoms(kind))) return 1;
  if (static_cast<long long>(experts) * n1 > 0x7FFFFFFFll || static_cast<long long>(experts) * h_out > 0x7FFFFFFFll) return 1;
  FewParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(x); p.route_x = static_cast<const __nv_bfloat16*>(route_x);
  p.router = static_cast<const __nv_bfloat16*>(router);
  p.sel_bias = static_cast<const float*>(sel_bias); p.shared = static_cast<const __nv_bfloat16*>(shared);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldx = ldx; p.ld_route = ld_route; p.ld_router = ld_router; p.ld_shared = ld_shared; p.ldo = ldo;
  p.tokens = tokens; p.experts = experts; p.topk = topk; p.hidden = hidden; p.inter = inter; p.h_out = h_out; p.route_k = route_k;
  p.sigmoid = sigmoid; p.renorm = renorm; p.swiglu = swiglu; p.scale = scale;
  p.sf1 = static_cast<const uint8_t*>(sf1); p.sf2 = static_cast<const uint8_t*>(sf2);
  p.gs1 = static_cast<const float*>(gs1); p.gs2 = static_cast<const float*>(gs2);
  p.ka1 = ka1; p.ka2 = ka2;
  p.status = static_cast<int*>(status);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define HB_CALL(K) launch_few<K>(p, w1, w2, static_cast<uint8_t*>(ws), st)
  const cudaError_t e = HB_FEW_KIND(HB_CALL);
#undef HB_CALL
  return e == cudaSuccess ? 0 : 2;
}
#undef HB_FEW_KIND

}  // extern "C"
