// A whole mixture-of-experts layer for up to 16 tokens in two kernels.
//
//   logits = r R^T                       r the router's input rows (the layer's, or the wider ones of a latent layer)
//   score  = softmax(logits) or sigmoid(logits);  ids = the top-k of score (+ selection bias), ties to the lower index
//   w_j    = scale * score_j (/ sum of the chosen scores)
//   mid_j  = silu(W1g x) * (W1u x)  or  relu(W1 x)^2          W1, W2 of expert ids_j
//   out    = sum_j w_j W2 mid_j (+ shared)                    experts in ascending order, rounded once
//
//   fc1 : router, top-k and plan, then the first product and the activation;
//   fc2 : the second product, the weighted sum and the shared expert's rows.
//
// At these sizes the layer is the stream of its experts' weights: every chosen expert is read once, whatever it does to one
// or to eight rows. So weights go from HBM to shared memory by 16-byte asynchronous copies, each warp through a ring of its own
// (no block-wide meeting in the main loop), are decoded in registers and multiplied by mma.sync with sixteen weight rows on
// the M side and an expert's tokens on the N side. The activations are NOT quantised: weights become fp16 (exact), activations
// are scaled by a power of two per row into fp16's range, which keeps all 8 bits of a bf16 number down to 2^-29 of its row's
// largest, and the sums are fp32. bf16 weights meet bf16 rows in fc1; mid keeps 11 bits against FP4 weights and 8 against bf16.
//
// Every CTA of fc1 needs the routing, and there is no grid-wide barrier: each cluster computes all of it, the experts' logits
// split over its CTAs, the tokens' top-k likewise, exchanged through distributed shared memory.
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
constexpr int COLS = 8;                  // tokens of an entry: the N side of mma.m16n8k16
constexpr int MAX_SMEM = 227 * 1024;

struct FewParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* route_x;          // null: x
  const __nv_bfloat16* router;
  const float* sel_bias;
  const __nv_bfloat16* shared;
  __nv_bfloat16* out;
  long long ldx, ld_route, ld_router, ld_shared, ldo;
  int tokens, experts, topk, hidden, inter, h_out, route_k;
  int sigmoid, renorm, swiglu;
  float scale;
  const uint8_t *w1, *w2, *sf1, *sf2;
  const float *gs1, *gs2;
  int ka1, ka2;
  int* ids;                              // workspace: what fc1 leaves for fc2
  float* weights;
  float* mid;                            // [pairs][inter]
  int row_tiles, batch;                  // fc2: row tiles of a CTA, pairs whose rows fit its shared memory at once
};

// The routing as every CTA holds it: entries (an expert and up to eight of its tokens) in ascending order of experts.
struct Plan {
  int entries;
  int ids[MAX_PAIRS];
  float weights[MAX_PAIRS];
  uint32_t chosen[MAX_TOKENS][MAX_EXPERTS / 32];     // bit e: the token chose expert e
  uint32_t any[MAX_EXPERTS / 32], two[MAX_EXPERTS / 32];   // some token, more than eight tokens did
  int before[MAX_EXPERTS / 32];                       // entries of the experts below 32 w
  unsigned short expert[MAX_PAIRS], count[MAX_PAIRS];     // of entries
  unsigned short pair[MAX_PAIRS * COLS];              // [entry][column]: token * topk + j
};

template <int FMT>
struct Traits {
  static constexpr bool kFp4 = FMT != kGemmBf16;
  static constexpr int STEP_K = kFp4 ? 128 : 32;            // K elements of 64 bytes of a row
  static constexpr int SC_BYTES = FMT == kGemmMxfp4 ? 64 : FMT == kGemmNvfp4 ? 128 : 0;
  static constexpr int STAGE = 16 * 64 + SC_BYTES;
  static constexpr int PARTS = kFp4 ? 1 : 2;                // 16-bit numbers that stand for one of mid
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Two ue8m0 bytes (low half of v) -> two floats.
__device__ __forceinline__ float2 ue8m0x2(uint32_t v) {
  uint32_t r;
  const uint16_t in = static_cast<uint16_t>(v);
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"(in));
  return make_float2(bf16_lo(r), bf16_hi(r));
}
// One e4m3 byte -> fp16 in both halves.
__device__ __forceinline__ uint32_t e4m3_h2(uint32_t byte) {
  uint32_t h2;
  const uint16_t in = static_cast<uint16_t>((byte & 255u) * 0x0101u);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(in));
  return h2;
}
// Eight e2m1 codes -> fp16 numbers of 2^-14 of their values: h[q] holds codes q (low half) and q + 4. Sign and the three other bits
// of a code land on bits 15 and 11 .. 9 (0.5 is then a subnormal number). cvt.rn.f16x2.e2m1x2 does this too, at a quarter of the rate
// of these shifts and masks: with it the conversions alone took twice the time the weights take from HBM.
__device__ __forceinline__ void decode8(uint32_t w, uint32_t (&h)[4]) {
  h[0] = ((w << 9) & 0x0E000E00u) | ((w << 12) & 0x80008000u);
  h[1] = ((w << 5) & 0x0E000E00u) | ((w << 8) & 0x80008000u);
  h[2] = ((w << 1) & 0x0E000E00u) | ((w << 4) & 0x80008000u);
  h[3] = ((w >> 3) & 0x0E000E00u) | (w & 0x80008000u);
}
// Eight consecutive activations in the order of those pairs: 0 4 1 5 2 6 3 7.
__device__ __forceinline__ uint4 pack_pairs(const float (&e)[8], float f) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(e[i] * f, e[i + 4] * f);
  return *reinterpret_cast<const uint4*>(h);
}

// A row of largest magnitude m (its bits) goes to fp16 times 2^(141 - E), E the biased exponent of m: m lands in [2^14, 2^15). With
// the weights' 2^-14 a product comes out times 2^(127 - E). Rows of all but nothing keep E = 15, where both factors are still
// normal numbers; an infinity or a NaN stays one.
__device__ __forceinline__ int range_exp(uint32_t bits) { return min(max(static_cast<int>(bits >> 23), 15), 254); }
__device__ __forceinline__ float range_in(int e) { return __int_as_float((268 - e) << 23); }
__device__ __forceinline__ float range_out(int e) { return __int_as_float(e << 23); }

// The rows of tile `tile` of an expert's matrix. FP4: four rows each of the four 32-row quarters of a 128-row scale block, whose
// scales are 64 consecutive bytes of an atom; otherwise sixteen consecutive rows.
template <int FMT>
__device__ __forceinline__ int tile_row(int tile, int m) {
  if constexpr (Traits<FMT>::kFp4) return (tile >> 3) * 128 + (tile & 7) * 4 + (m & 3) + 32 * (m >> 2);
  return tile * 16 + m;
}

// One warp's ring of D stages of 64 bytes of K of 16 rows, and the pieces that this lane copies. Lane l brings chunk l % 4 of rows
// l / 4 and l / 4 + 8; chunks are permuted within a pair of rows so that the reads of eight rows hit all banks.
template <int FMT, int D>
struct Feed {
  using T = Traits<FMT>;
  uint32_t ring, dst;
  const uint8_t* a;
  int to_b;                        // from row m to row m + 8
  const uint8_t* s;
  int left;                        // bytes of the row from this lane's chunk on

  __device__ __forceinline__ void init(uint32_t ring_addr, int row_bytes, int lane) {
    ring = ring_addr;
    const int m = lane >> 2, c = lane & 3;
    dst = m * 64 + ((c ^ ((m >> 1) & 3)) << 4);
    left = row_bytes - c * 16;
    to_b = (T::kFp4 ? 64 : 8) * row_bytes;
  }
  __device__ __forceinline__ void set(const uint8_t* w, const uint8_t* sf, long long row0, int tile, int row_bytes, int ka, int lane) {
    const int m = lane >> 2, c = lane & 3;
    a = w + (row0 + tile_row<FMT>(tile, m)) * row_bytes + c * 16;
    if constexpr (T::kFp4) {
      s = sf + ((row0 >> 7) + (tile >> 3)) * static_cast<long long>(ka) * 512 + (tile & 7) * 64 + (lane & 3) * 16;
      if constexpr (FMT == kGemmNvfp4) s += ((lane >> 2) & 1) * 512;
    }
  }
  __device__ __forceinline__ void issue(int slot, int step, int lane) {
    const uint32_t st = ring + slot * T::STAGE;
    const bool in = step * 64 < left;
    const uint8_t* p = in ? a + step * 64 : a;
    cp_async16(st + dst, p, in);
    cp_async16(st + dst + 512, p + to_b, in);
    if constexpr (T::kFp4)
      if (lane < T::SC_BYTES / 16) cp_async16(st + 1024 + lane * 16, s + step * (T::SC_BYTES * 8), true);
  }
};

// One step: acc += W[16 rows][STEP_K] * b, where b(block, part) gives the lane's eight 16-bit activations at 32 * block + 8 *
// (lane % 4) of its column lane / 4. A lane holds those same K positions of its two weight rows, so K is permuted alike on both sides.
template <int FMT, int PARTS, typename B>
__device__ __forceinline__ void step_mma(float (&acc)[4], uint32_t st, int lane, B&& b) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (FMT == kGemmBf16) {
    const uint32_t at = st + g * 64 + ((t ^ ((g >> 1) & 3)) << 4);
    const uint4 u = lds128(at), v = lds128(at + 512);
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const uint4 x = b(0, i);
      mma_16816<true>(acc, u.x, v.x, u.y, v.y, x.x, x.y);
      mma_16816<true>(acc, u.z, v.z, u.w, v.w, x.z, x.w);
    }
  } else {
    // ldmatrix: lane (g, t) receives word t of the 16 bytes (one MXFP4 block) that row g has in each chunk
    const int m = lane & 15, hi = lane >> 4;
    const uint32_t sw = (m >> 1) & 3;
    uint32_t r[2][4];                  // [chunk pair][row g chunk 0, row g + 8 chunk 0, row g chunk 1, row g + 8 chunk 1]
    ldmatrix_x4(r[0], st + m * 64 + ((hi ^ sw) << 4));
    ldmatrix_x4(r[1], st + m * 64 + (((2 + hi) ^ sw) << 4));
    const uint32_t sc = st + 1024 + (g & 3) * 16 + (g >> 2) * 4;     // scales of row g; those of row g + 8 lie 8 bytes on
    if constexpr (FMT == kGemmMxfp4) {
      const uint32_t sa = lds32(sc), sb = lds32(sc + 8);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 fa = ue8m0x2(sa >> (16 * h)), fb = ue8m0x2(sb >> (16 * h));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t u[4], v[4];
          decode8(r[h][2 * q], u);
          decode8(r[h][2 * q + 1], v);
          const uint4 x = b(2 * h + q, 0);
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816<false>(part, u[0], v[0], u[1], v[1], x.x, x.y);
          mma_16816<false>(part, u[2], v[2], u[3], v[3], x.z, x.w);
          const float ga = q ? fa.y : fa.x, gb = q ? fb.y : fb.x;
          acc[0] = fmaf(part[0], ga, acc[0]);
          acc[1] = fmaf(part[1], ga, acc[1]);
          acc[2] = fmaf(part[2], gb, acc[2]);
          acc[3] = fmaf(part[3], gb, acc[3]);
        }
      }
    } else {
      // NVFP4: words 0 and 1 of a chunk belong to one block of 16, words 2 and 3 to the next; the scale (4 significant bits
      // times 2 of the value, down to 2^-24: exact) is multiplied in before the product
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t sa = lds32(sc + h * 64) >> (8 * (t >> 1)), sb = lds32(sc + h * 64 + 8) >> (8 * (t >> 1));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t fa = e4m3_h2(sa >> (16 * q)), fb = e4m3_h2(sb >> (16 * q));
          uint32_t u[4], v[4];
          decode8(r[h][2 * q], u);
          decode8(r[h][2 * q + 1], v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] = hmul2(u[i], fa);
            v[i] = hmul2(v[i], fb);
          }
          const uint4 x = b(2 * h + q, 0);
          mma_16816<false>(acc, u[0], v[0], u[1], v[1], x.x, x.y);
          mma_16816<false>(acc, u[2], v[2], u[3], v[3], x.z, x.w);
        }
      }
    }
  }
}

// Entries of the routing in plan.ids, by a whole CTA. Everything is bit masks over the experts, so nothing depends on timing.
__device__ __forceinline__ void make_plan(Plan& plan, int tokens, int experts, int topk) {
  const int tid = threadIdx.x, lane = tid & 31, pairs = tokens * topk;
  static_assert(THREADS == MAX_TOKENS * MAX_EXPERTS / 32, "one mask word a thread");
  plan.chosen[tid >> 5][lane] = 0;
  __syncthreads();
  const int my_token = tid / topk, e = tid < pairs ? plan.ids[tid] : 0;
  if (tid < pairs) atomicOr(&plan.chosen[my_token][e >> 5], 1u << (e & 31));
  __syncthreads();
  if (tid < 32) {
    uint32_t c[5] = {0, 0, 0, 0, 0};           // how many tokens chose each of this word's experts, bit by bit
    for (int t = 0; t < tokens; ++t) {
      uint32_t carry = plan.chosen[t][lane];
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const uint32_t both = c[i] & carry;
        c[i] ^= carry;
        carry = both;
      }
    }
    const uint32_t any = c[0] | c[1] | c[2] | c[3] | c[4], two = c[4] | (c[3] & (c[0] | c[1] | c[2]));
    const int mine = __popc(any) + __popc(two);
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    plan.any[lane] = any;
    plan.two[lane] = two;
    plan.before[lane] = inc - mine;
    if (lane == 31) plan.entries = inc;
  }
  __syncthreads();
  if (tid < pairs) {
    const int w = e >> 5, b = e & 31;
    const uint32_t below = (1u << b) - 1u;
    int slot = 0, all = 0;                     // tokens before this one that chose the expert, and all that did
    for (int t = 0; t < tokens; ++t) {
      const int in = (plan.chosen[t][w] >> b) & 1;
      all += in;
      slot += t < my_token ? in : 0;
    }
    const int entry = plan.before[w] + __popc(plan.any[w] & below) + __popc(plan.two[w] & below) + slot / COLS;
    plan.pair[entry * COLS + slot % COLS] = static_cast<unsigned short>(tid);
    if (slot % COLS == 0) {
      plan.expert[entry] = static_cast<unsigned short>(e);
      plan.count[entry] = static_cast<unsigned short>(min(COLS, all - slot));
    }
  }
  __syncthreads();
}

__device__ __forceinline__ uint32_t order_key(float v) {          // orders floats as unsigned numbers; never 0
  const uint32_t b = __float_as_uint(v);
  return max((b & 0x80000000u) ? ~b : (b | 0x80000000u), 1u);
}

// Top-k of one token by one warp. `score` holds the logits on entry, `key` and `cand` [experts] are scratch. Lane j < topk returns id
// and weight; scores, order and weights are those of moe_route_kernel (moe.cu). No lane whose best key is below the topk-th
// largest of the 32 lanes' best keys can hold a chosen expert, so a few candidates are left, which rank themselves.
__device__ __forceinline__ void warp_topk(const FewParams& p, float* score, uint32_t* key, unsigned short* cand, int& id, float& weight) {
  const int lane = threadIdx.x & 31, E = p.experts, K = p.topk;
  uint32_t best = 0;
  if (p.sigmoid) {
#pragma unroll 4
    for (int e = lane; e < E; e += 32) {
      const float s = 1.f / (1.f + __expf(-score[e]));
      score[e] = s;
      const uint32_t k = order_key(s + (p.sel_bias != nullptr ? __ldg(p.sel_bias + e) : 0.f));
      key[e] = k;
      best = max(best, k);
    }
  } else {
    float mx = -INFINITY;
#pragma unroll 4
    for (int e = lane; e < E; e += 32) mx = fmaxf(mx, score[e]);
    mx = warp_max(mx);
    float sum = 0.f;
#pragma unroll 4
    for (int e = lane; e < E; e += 32) {
      const float s = __expf(score[e] - mx);
      score[e] = s;
      sum += s;
    }
    const float inv = 1.f / warp_sum(sum);
#pragma unroll 4
    for (int e = lane; e < E; e += 32) {
      const float s = score[e] * inv;
      score[e] = s;
      key[e] = order_key(s);
      best = max(best, order_key(s));
    }
  }
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t other = __shfl_sync(0xffffffffu, best, i);
    rank += other > best || (other == best && i < lane);
  }
  const uint32_t thr = max(__shfl_sync(0xffffffffu, best, __ffs(__ballot_sync(0xffffffffu, rank == K - 1)) - 1), 1u);
  __syncwarp();
  int n = 0, ties = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {               // ascending experts; of equal keys at the threshold the first K will do
    const int e = e0 + lane;
    const uint32_t k = e < E ? key[e] : 0u;
    const uint32_t eq = __ballot_sync(0xffffffffu, k == thr);
    const uint32_t below = (1u << lane) - 1u;
    const bool take = k > thr || (k == thr && ties + __popc(eq & below) < K);
    const uint32_t taken = __ballot_sync(0xffffffffu, take);
    if (take) cand[n + __popc(taken & below)] = static_cast<unsigned short>(e);
    n += __popc(taken);
    ties += __popc(eq);
  }
  __syncwarp();
  // place of every candidate among them (the list ascends, so of equal keys the earlier one goes first); `key` takes the places
  id = 0;
  weight = 0.f;
  for (int c0 = 0; c0 < n; c0 += 32) {
    const int c = c0 + lane;
    const uint32_t mine = c < n ? key[cand[c]] : 0u;
    int place = 0;
    for (int i = 0; i < n; ++i) {
      const uint32_t k = key[cand[i]];
      place += k > mine || (k == mine && i < c);
    }
    for (int j = 0; j < K; ++j) {                     // lane j picks up the candidate of place j
      const uint32_t at = __ballot_sync(0xffffffffu, c < n && place == j);
      if (lane == j && at != 0) id = cand[c0 + __ffs(at) - 1];
    }
  }
  if (lane < K) weight = score[id];
  float sum = 0.f;
  for (int j = 0; j < K; ++j) sum += __shfl_sync(0xffffffffu, weight, j);
  weight = (p.renorm ? weight / fmaxf(sum, 1e-20f) : weight) * p.scale;
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__host__ __device__ constexpr int align16(int v) { return (v + 15) & ~15; }
// Shared memory of fc1: plan | logits, keys and candidates of this CTA's tokens | exponents | activations | rings (the router's partial
// sums, 16 KB, before them)
__host__ __device__ inline int x_pitch(int k, int step_k) { return (k + step_k - 1) / step_k * step_k * 2 + 64; }
__host__ __device__ inline int route_bytes(int tokens, int experts, int cluster) {
  return align16((tokens + cluster - 1) / cluster * experts * 10);
}
__host__ __device__ inline int fc1_fixed_bytes(int tokens, int experts, int cluster) {
  return align16(sizeof(Plan)) + route_bytes(tokens, experts, cluster) + MAX_TOKENS * 4 + WARPS * 512;
}

template <int FMT, int D>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_fc1_kernel(const __grid_constant__ FewParams p) {
  using T = Traits<FMT>;
  extern __shared__ __align__(128) uint8_t sm[];
  uint32_t cluster_n;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cluster_n));
  const int cluster = static_cast<int>(cluster_n), rank = static_cast<int>(cluster_ctarank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  Plan& plan = *reinterpret_cast<Plan*>(sm);
  const int lrows = (p.tokens + cluster - 1) / cluster;
  float* logit = reinterpret_cast<float*>(sm + align16(sizeof(Plan)));          // [lrows][experts]
  uint32_t* key = reinterpret_cast<uint32_t*>(logit + lrows * p.experts);
  unsigned short* cand = reinterpret_cast<unsigned short*>(key + lrows * p.experts);
  uint8_t* at_sm = sm + align16(sizeof(Plan)) + route_bytes(p.tokens, p.experts, cluster);
  int* row_exp = reinterpret_cast<int*>(at_sm);
  float* split_sums = reinterpret_cast<float*>(at_sm + MAX_TOKENS * 4);        // [warps][128]
  uint8_t* xs = sm + fc1_fixed_bytes(p.tokens, p.experts, cluster);
  const int pitch = x_pitch(p.hidden, T::STEP_K);
  uint8_t* rings = xs + align16(p.tokens * pitch);
  const uint32_t xs_addr = smem_u32(xs);

  cluster_arrive();                       // peers' shared memory is there from the first wait below on
  grid_dep_wait();
  grid_dep_launch();

  // ---- activations as they are (whole 16-byte pieces; what pads the last step is zero)
  const int pieces = (pitch - 64) / 16;
  for (int i = tid; i < p.tokens * pieces; i += THREADS) {
    const int tok = i / pieces, c = i - tok * pieces;
    const bool in = c * 8 < p.hidden;
    cp_async16(xs_addr + tok * pitch + c * 16, p.x + tok * p.ldx + (in ? c * 8 : 0), in);
  }
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
  if (T::kFp4 && warp < p.tokens) {
    uint32_t m = 0;
    for (int c = lane; c < pieces; c += 32) {
      const uint4 v = lds128(xs_addr + warp * pitch + c * 16);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max(m, max((w[i] << 16) & 0x7FFF0000u, w[i] & 0x7FFF0000u));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) row_exp[warp] = range_exp(m);
  }

  // ---- router: a warp takes sixteen experts and one of `parts` shares of K; tiles of experts go round the cluster's CTAs
  {
    const int e_tiles = (p.experts + 15) / 16, my_tiles = max(0, (e_tiles - rank + cluster - 1) / cluster);
    float* part = reinterpret_cast<float*>(rings);                  // [tile][part][16 tokens][16 experts] of a round
    const int blocks = (p.route_k + 31) / 32;
    for (int round = 0; round < my_tiles; round += WARPS) {
      const int tiles = min(my_tiles - round, WARPS), parts = WARPS / tiles;
      const int tile = warp / parts, share = warp % parts;
      if (tile < tiles) {
        const int e0 = (rank + (round + tile) * cluster) * 16;
        const __nv_bfloat16* ra = p.router + static_cast<long long>(min(e0 + g, p.experts - 1)) * p.ld_router;
        const __nv_bfloat16* rb = p.router + static_cast<long long>(min(e0 + g + 8, p.experts - 1)) * p.ld_router;
        const bool two = p.tokens > 8;
        float acc[2][4] = {};
        constexpr int U = 5;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        for (int b0 = share; b0 < blocks; b0 += parts * U) {
          uint4 wa[U], wb[U];
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int k = (b0 + i * parts) * 32 + t * 8;
            const bool in = k < p.route_k;
            wa[i] = in ? __ldg(reinterpret_cast<const uint4*>(ra + k)) : zero;
            wb[i] = in ? __ldg(reinterpret_cast<const uint4*>(rb + k)) : zero;
          }
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int k = (b0 + i * parts) * 32 + t * 8;
            const bool in = k < p.route_k;
            uint4 xa = zero, xb = zero;
            if (p.route_x == nullptr) {
              if (in && g < p.tokens) xa = lds128(xs_addr + g * pitch + k * 2);
              if (two && in && g + 8 < p.tokens) xb = lds128(xs_addr + (g + 8) * pitch + k * 2);
            } else {
              if (in && g < p.tokens) xa = ld_step(reinterpret_cast<const uint4*>(p.route_x + g * p.ld_route + k));
              if (two && in && g + 8 < p.tokens) xb = ld_step(reinterpret_cast<const uint4*>(p.route_x + (g + 8) * p.ld_route + k));
            }
            mma_16816<true>(acc[0], wa[i].x, wb[i].x, wa[i].y, wb[i].y, xa.x, xa.y);
            mma_16816<true>(acc[0], wa[i].z, wb[i].z, wa[i].w, wb[i].w, xa.z, xa.w);
            if (two) {
              mma_16816<true>(acc[1], wa[i].x, wb[i].x, wa[i].y, wb[i].y, xb.x, xb.y);
              mma_16816<true>(acc[1], wa[i].z, wb[i].z, wa[i].w, wb[i].w, xb.z, xb.w);
            }
          }
        }
        float* mine = part + warp * 256;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          mine[(n * 8 + 2 * t) * 16 + g] = acc[n][0];
          mine[(n * 8 + 2 * t + 1) * 16 + g] = acc[n][1];
          mine[(n * 8 + 2 * t) * 16 + g + 8] = acc[n][2];
          mine[(n * 8 + 2 * t + 1) * 16 + g + 8] = acc[n][3];
        }
      }
      __syncthreads();
      if (round == 0) cluster_wait();
      for (int i = tid; i < tiles * 256; i += THREADS) {
        const int tl = i >> 8, tok = (i >> 4) & 15, e = (rank + (round + tl) * cluster) * 16 + (i & 15);
        if (tok < p.tokens && e < p.experts) {
          float s = 0.f;
          for (int w = 0; w < parts; ++w) s += part[(tl * parts + w) * 256 + (i & 255)];
          st_cluster(map_to_cta(smem_u32(logit + (tok / cluster) * p.experts + e), tok % cluster), __float_as_uint(s));
        }
      }
      __syncthreads();
    }
    if (my_tiles == 0) cluster_wait();
  }
  cluster_arrive();
  if constexpr (T::kFp4) {                // meanwhile: fp16, scaled by a power of two per row, in the order of the decoded weights
    __syncthreads();
    for (int i = tid; i < p.tokens * pieces; i += THREADS) {
      const int tok = i / pieces;
      const uint32_t at = xs_addr + tok * pitch + (i - tok * pieces) * 16;
      float e[8];
      unpack8(lds128(at), e);
      sts128(at, pack_pairs(e, range_in(row_exp[tok])));
    }
  }
  cluster_wait();
  // ---- top-k: token `rank + i * cluster` by warp i; everybody gets the result
  for (int i = warp; i < lrows; i += WARPS) {
    const int tok = rank + i * cluster;
    if (tok < p.tokens) {
      int id;
      float w;
      warp_topk(p, logit + i * p.experts, key + i * p.experts, cand + i * p.experts, id, w);
      if (lane < p.topk) {
        const int at = tok * p.topk + lane;
        for (int r = 0; r < cluster; ++r) {
          st_cluster(map_to_cta(smem_u32(&plan.ids[at]), r), static_cast<uint32_t>(id));
          st_cluster(map_to_cta(smem_u32(&plan.weights[at]), r), __float_as_uint(w));
        }
        if (static_cast<int>(blockIdx.x) == rank) {        // the first cluster: fc2 makes the same plan
          p.ids[at] = id;
          p.weights[at] = w;
        }
      }
    }
  }
  cluster_sync_all();
  make_plan(plan, p.tokens, p.experts, p.topk);

  // ---- first product: a unit is (entry, 16 weight rows), one warp's work, or `split` warps' that share its K where the units are
  // too few for all warps of the chip; units go round the CTAs
  const int n1 = p.swiglu ? 2 * p.inter : p.inter, tiles = n1 / 16, units = plan.entries * tiles;
  const int steps = (p.hidden + T::STEP_K - 1) / T::STEP_K;
  const int row_bytes = T::kFp4 ? p.hidden / 2 : p.hidden * 2;
  const int grid = static_cast<int>(gridDim.x);
  const int split = units * 4 <= grid * WARPS && steps >= 8 ? 4 : units * 2 <= grid * WARPS && steps >= 4 ? 2 : 1;
  const int share = warp % split, group = warp / split, stride = grid * (WARPS / split);
  const int s0 = steps * share / split, s1 = steps * (share + 1) / split;
  Feed<FMT, D> feed;
  feed.init(smem_u32(rings) + warp * D * T::STAGE, row_bytes, lane);
  int iu = static_cast<int>(blockIdx.x) + group * grid, is = s0, islot = 0;
  auto aim = [&] {
    if (iu < units) {
      const int entry = iu / tiles;
      feed.set(p.w1, p.sf1, static_cast<long long>(plan.expert[entry]) * n1, iu - entry * tiles, row_bytes, p.ka1, lane);
    }
  };
  auto issue = [&] {
    if (iu < units) {
      feed.issue(islot, is, lane);
      if (++is == s1) {
        is = s0;
        iu += stride;
        aim();
      }
    }
    cp_async_commit();
    islot = islot + 1 == D ? 0 : islot + 1;
  };
  int unit = iu, slot = 0;
  aim();
#pragma unroll 1
  for (int d = 0; d < D; ++d) issue();
  while (unit < units) {
    const int entry = unit / tiles, tile = unit - entry * tiles;
    const int n = plan.count[entry];
    const unsigned short* pairs = plan.pair + entry * COLS;
    const bool live = g < n;
    const uint32_t xrow = xs_addr + (live ? pairs[g] / p.topk : 0) * pitch + t * 16;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = s0; s < s1; ++s) {
      cp_async_wait<D - 1>();
      __syncwarp();
      const uint32_t xat = xrow + s * (T::STEP_K * 2);
      step_mma<FMT, 1>(acc, feed.ring + slot * T::STAGE, lane, [&](int blk, int) {
        return live ? lds128(xat + blk * 64) : make_uint4(0, 0, 0, 0);
      });
      __syncwarp();
      issue();
      slot = slot + 1 == D ? 0 : slot + 1;
    }
    if (split > 1) {                       // the shares' sums meet in shared memory, in order
      float4* mine = reinterpret_cast<float4*>(split_sums) + warp * 32 + lane;
      *mine = make_float4(acc[0], acc[1], acc[2], acc[3]);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(split * 32) : "memory");
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < split; ++w) {
        const float4 v = reinterpret_cast<const float4*>(split_sums)[(group * split + w) * 32 + lane];
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
      acc[0] = sum.x; acc[1] = sum.y; acc[2] = sum.z; acc[3] = sum.w;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(split * 32) : "memory");
    }
    if (share == 0) {
      // lane (g, t) holds rows g and g + 8 of columns 2 t and 2 t + 1
      const float gs = p.gs1 != nullptr ? __ldg(p.gs1 + plan.expert[entry]) : 1.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 2 * t + c, pr = col < n ? pairs[col] : -1;
        const float f = pr < 0 ? 0.f : T::kFp4 ? range_out(row_exp[pr / p.topk]) : 1.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v = acc[2 * h + c] * f * gs;
          int row = tile_row<FMT>(tile, g + 8 * h);
          if (p.swiglu) {
            const float up = __shfl_xor_sync(0xffffffffu, v, 4);      // rows come in pairs: gate, up
            v = v / (1.f + __expf(-v)) * up;
            row >>= 1;
          } else {
            v = v <= 0.f ? 0.f : v * v;                               // (a NaN stays one)
          }
          if (pr >= 0 && (!p.swiglu || (g & 1) == 0)) p.mid[static_cast<long long>(pr) * p.inter + row] = v;
        }
      }
    }
    unit += stride;
  }
  cp_async_wait<0>();
}

// Shared memory of fc2: plan | partial sums [warps][tokens][16] | exponents of the rows of a batch | rings | rows of a batch
__host__ __device__ inline int fc2_fixed_bytes(int tokens) { return align16(sizeof(Plan)) + WARPS * tokens * 64 + MAX_PAIRS * 4; }

template <int FMT, int D>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_fc2_kernel(const __grid_constant__ FewParams p) {
  using T = Traits<FMT>;
  extern __shared__ __align__(128) uint8_t sm[];
  uint32_t cluster_n;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cluster_n));
  const int cluster = static_cast<int>(cluster_n), rank = static_cast<int>(cluster_ctarank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  Plan& plan = *reinterpret_cast<Plan*>(sm);
  float* sums = reinterpret_cast<float*>(sm + align16(sizeof(Plan)));
  int* row_exp = reinterpret_cast<int*>(sums + WARPS * p.tokens * 16);
  uint8_t* rings = sm + fc2_fixed_bytes(p.tokens);
  const uint32_t rows_addr = smem_u32(rings) + WARPS * D * T::STAGE;
  const int pitch = x_pitch(p.inter, T::STEP_K) * T::PARTS, part_bytes = x_pitch(p.inter, T::STEP_K);
  const int pairs = p.tokens * p.topk;

  for (int i = tid; i < WARPS * p.tokens * 16; i += THREADS) sums[i] = 0.f;
  grid_dep_wait();
  grid_dep_launch();
  if (tid < pairs) {
    plan.ids[tid] = ld_step(p.ids + tid);
    plan.weights[tid] = ld_step(p.weights + tid);
  }
  make_plan(plan, p.tokens, p.experts, p.topk);

  // A CTA has `row_tiles` tiles of 16 output rows and, of the entries, those that are `rank` modulo the cluster's size. Warp w works on
  // tile w % row_tiles and on every phases-th of the CTA's entries.
  const int tile = static_cast<int>(blockIdx.x) / cluster * p.row_tiles + warp % p.row_tiles;
  const int phases = WARPS / p.row_tiles, phase = warp / p.row_tiles;
  const bool works = phase < phases && tile * 16 < p.h_out;
  const int steps = (p.inter + T::STEP_K - 1) / T::STEP_K;
  const int row_bytes = T::kFp4 ? p.inter / 2 : p.inter * 2;
  const int stride = cluster * phases;
  Feed<FMT, D> feed;
  feed.init(smem_u32(rings) + warp * D * T::STAGE, row_bytes, lane);
  int iu = works ? rank + phase * cluster : plan.entries, is = 0, islot = 0;
  auto aim = [&] {
    if (iu < plan.entries)
      feed.set(p.w2, p.sf2, static_cast<long long>(plan.expert[iu]) * p.h_out, tile, row_bytes, p.ka2, lane);
  };
  auto issue = [&] {
    if (iu < plan.entries) {
      feed.issue(islot, is, lane);
      if (++is == steps) {
        is = 0;
        iu += stride;
        aim();
      }
    }
    cp_async_commit();
    islot = islot + 1 == D ? 0 : islot + 1;
  };
  int entry = iu, slot = 0;
  aim();
#pragma unroll 1
  for (int d = 0; d < D; ++d) issue();
  float* mine = sums + warp * p.tokens * 16;

  // Batches of the CTA's entries whose rows of mid fit: converted once for all tiles, the weights of the first steps on their way.
  for (int lo = rank; lo < plan.entries;) {
    int hi = lo, rows = 0;
    for (; hi < plan.entries && rows + plan.count[hi] <= p.batch; hi += cluster) rows += plan.count[hi];
    for (int i = warp, e = lo, first = 0; i < rows; i += WARPS) {
      while (first + plan.count[e] <= i) {
        first += plan.count[e];
        e += cluster;
      }
      const float* row = p.mid + static_cast<long long>(plan.pair[e * COLS + i - first]) * p.inter;
      const uint32_t dst = rows_addr + i * pitch;
      const int pieces = (part_bytes - 64) / 16;
      float f = 1.f;
      if constexpr (T::kFp4) {
        uint32_t m = 0;
#pragma unroll 4
        for (int k = lane * 4; k < p.inter; k += 128) {
          const float4 v = ld_step(reinterpret_cast<const float4*>(row + k));
          m = max(max(m, __float_as_uint(v.x) & 0x7FFFFFFFu), __float_as_uint(v.y) & 0x7FFFFFFFu);
          m = max(max(m, __float_as_uint(v.z) & 0x7FFFFFFFu), __float_as_uint(v.w) & 0x7FFFFFFFu);
        }
        const int ex = range_exp(__reduce_max_sync(0xffffffffu, m));
        if (lane == 0) row_exp[i] = ex;
        f = range_in(ex);
      }
#pragma unroll 2
      for (int c = lane; c < pieces; c += 32) {
        float e8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (c * 8 < p.inter) {
          const float4 u = ld_step(reinterpret_cast<const float4*>(row + c * 8)), v = ld_step(reinterpret_cast<const float4*>(row + c * 8 + 4));
          e8[0] = u.x; e8[1] = u.y; e8[2] = u.z; e8[3] = u.w; e8[4] = v.x; e8[5] = v.y; e8[6] = v.z; e8[7] = v.w;
        }
        if constexpr (T::kFp4) {
          sts128(dst + c * 16, pack_pairs(e8, f));
        } else {                            // two bf16 numbers: 16 significant bits (an infinity stays one)
          const uint4 top = pack8(e8);
          float h8[8];
          unpack8(top, h8);
#pragma unroll
          for (int j = 0; j < 8; ++j) h8[j] = fabsf(h8[j]) == INFINITY ? 0.f : e8[j] - h8[j];
          sts128(dst + c * 16, top);
          sts128(dst + part_bytes + c * 16, pack8(h8));
        }
      }
    }
    __syncthreads();
    int row0 = 0, at = lo;                  // row of the batch where entry `at` begins
    while (entry < hi) {
      while (at < entry) {
        row0 += plan.count[at];
        at += cluster;
      }
      const int n = plan.count[entry];
      const bool live = g < n;
      const uint32_t xrow = rows_addr + (row0 + (live ? g : 0)) * pitch + t * 16;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        cp_async_wait<D - 1>();
        __syncwarp();
        const uint32_t xat = xrow + s * (T::STEP_K * 2);
        step_mma<FMT, T::PARTS>(acc, feed.ring + slot * T::STAGE, lane, [&](int blk, int part) {
          return live ? lds128(xat + blk * 64 + part * part_bytes) : make_uint4(0, 0, 0, 0);
        });
        __syncwarp();
        issue();
        slot = slot + 1 == D ? 0 : slot + 1;
      }
      const float gs = p.gs2 != nullptr ? __ldg(p.gs2 + plan.expert[entry]) : 1.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 2 * t + c;
        if (col < n) {
          const int pr = plan.pair[entry * COLS + col], tok = pr / p.topk;
          const float w = plan.weights[pr] * gs, back = T::kFp4 ? range_out(row_exp[row0 + col]) : 1.f;
          mine[tok * 16 + g] += acc[c] * back * w;
          mine[tok * 16 + g + 8] += acc[2 + c] * back * w;
        }
      }
      __syncwarp();
      entry += stride;
    }
    __syncthreads();                        // before the next batch takes these rows' place
    lo = hi;
  }
  cp_async_wait<0>();
  __syncthreads();
  // ---- sums over the phases, then over the cluster, in order
  const int n_out = p.tokens * 16, all = p.row_tiles * n_out;
  for (int i = tid; i < all; i += THREADS) {
    float s = sums[i];
    for (int f = 1; f < phases; ++f) s += sums[f * all + i];
    sums[i] = s;
  }
  if (cluster > 1) cluster_sync_all();
  else __syncthreads();
  for (int i = tid + rank * THREADS; i < all; i += THREADS * cluster) {
    float s = 0.f;
    const uint32_t at = smem_u32(sums + i);
    for (int r = 0; r < cluster; ++r) s += cluster > 1 ? ld_dsmem_f32(map_to_cta(at, r)) : sums[i];
    const int tl = static_cast<int>(blockIdx.x) / cluster * p.row_tiles + i / n_out, tok = i % n_out / 16;
    if (tl * 16 >= p.h_out) continue;
    const int row = tile_row<FMT>(tl, i & 15);
    if (p.shared != nullptr) s += __bfloat162float(p.shared[tok * p.ld_shared + row]);
    p.out[tok * p.ldo + row] = __float2bfloat16(s);
  }
  if (cluster > 1) cluster_sync_all();       // nobody leaves while a peer may still read its sums
}

constexpr int stage_bytes(int kind) { return kind == kGemmBf16 ? 1024 : kind == kGemmMxfp4 ? 1088 : 1152; }
constexpr int FC2_DEPTH = 4;

// Clusters of `size` CTAs that the chip holds at once, one CTA an SM (0: none).
template <int FMT, int D>
int resident(int size) {
  static int known[17] = {};              // + 1
  if (known[size] == 0) {
    auto k1 = moe_few_fc1_kernel<FMT, D>;
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
    if (cudaOccupancyMaxActiveClusters(&n, k1, &q) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    known[size] = n + 1;
  }
  return known[size] - 1;
}

template <int FMT, int D>
cudaError_t launch_few(const FewParams& p, int cluster1, int cluster2, cudaStream_t st) {
  auto k1 = moe_few_fc1_kernel<FMT, D>;
  auto k2 = moe_few_fc2_kernel<FMT, FC2_DEPTH>;
  static const cudaError_t ready = [&] {
    cudaError_t e = cudaFuncSetAttribute(k1, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k1, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k2, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    return e;
  }();
  if (ready != cudaSuccess) return ready;
  const int clusters = resident<FMT, D>(cluster1);
  if (clusters < 1) return cudaErrorInvalidConfiguration;
  cudaError_t e = launch_dep_cluster(k1, dim3(clusters * cluster1), dim3(THREADS), cluster1, MAX_SMEM, st, p);
  if (e != cudaSuccess) return e;
  const int blocks = (p.h_out / 16 + p.row_tiles - 1) / p.row_tiles;
  return launch_dep_cluster(k2, dim3(blocks * cluster2), dim3(THREADS), cluster2, MAX_SMEM, st, p);
}

int fc1_room(int kind, int tokens, int hidden, int experts, int cluster) {      // for the rings
  return MAX_SMEM - fc1_fixed_bytes(tokens, experts, cluster) - align16(tokens * x_pitch(hidden, kind == kGemmBf16 ? 32 : 128));
}
int fc2_batch(int kind, int tokens, int inter) {
  const int pitch = x_pitch(inter, kind == kGemmBf16 ? 32 : 128) * (kind == kGemmBf16 ? 2 : 1);
  return min((MAX_SMEM - fc2_fixed_bytes(tokens) - WARPS * FC2_DEPTH * stage_bytes(kind)) / pitch, MAX_PAIRS);
}

}  // namespace
}  // namespace hb

extern "C" {

// Most tokens that one call takes at these widths (0: none).
int hb_moe_few_tokens(int kind, int hidden, int inter, int experts, int cluster) {
  using namespace hb;
  if (fc2_batch(kind, MAX_TOKENS, inter) < COLS) return 0;
  for (int t = MAX_TOKENS; t > 0; --t)
    if (fc1_room(kind, t, hidden, experts, cluster) >= WARPS * 4 * stage_bytes(kind)) return t;
  return 0;
}

int hb_moe_few(int kind, const void* x, long long ldx, const void* route_x, long long ld_route, const void* router,
               long long ld_router, int route_k, const void* sel_bias, int tokens, int experts, int topk, int sigmoid, int renorm,
               float scale, int hidden, int inter, int h_out, int swiglu, const void* w1, const void* sf1, const void* gs1, int ka1,
               const void* w2, const void* sf2, const void* gs2, int ka2, const void* shared, long long ld_shared, void* out,
               long long ldo, void* ws, int cluster1, int row_tiles, int cluster2, void* stream) {
  using namespace hb;
  const bool fp4 = is_fp4(kind);
  if (!fp4 && kind != kGemmBf16) return 1;
  if (cluster1 < 1 || cluster1 > 16 || cluster2 < 1 || cluster2 > 8 || row_tiles < 1 || row_tiles > WARPS) return 1;
  if (tokens < 1 || experts < 1 || experts > MAX_EXPERTS || topk < 1 || topk > MAX_TOPK || topk > experts) return 1;
  if (tokens > hb_moe_few_tokens(kind, hidden, inter, experts, cluster1)) return 1;
  const int n1 = swiglu ? 2 * inter : inter, rows = fp4 ? 128 : 16, k_of = fp4 ? 32 : 8;
  if (n1 < 1 || n1 % rows || h_out < 1 || h_out % rows || hidden % k_of || inter % k_of) return 1;
  if (router == nullptr || route_k < 8 || route_k % 8 || (route_x == nullptr && route_k != hidden)) return 1;
  FewParams p;
  p.x = static_cast<const __nv_bfloat16*>(x); p.route_x = static_cast<const __nv_bfloat16*>(route_x);
  p.router = static_cast<const __nv_bfloat16*>(router);
  p.sel_bias = static_cast<const float*>(sel_bias); p.shared = static_cast<const __nv_bfloat16*>(shared);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldx = ldx; p.ld_route = ld_route; p.ld_router = ld_router; p.ld_shared = ld_shared; p.ldo = ldo;
  p.tokens = tokens; p.experts = experts; p.topk = topk; p.hidden = hidden; p.inter = inter; p.h_out = h_out; p.route_k = route_k;
  p.sigmoid = sigmoid; p.renorm = renorm; p.swiglu = swiglu; p.scale = scale;
  p.w1 = static_cast<const uint8_t*>(w1); p.w2 = static_cast<const uint8_t*>(w2);
  p.sf1 = static_cast<const uint8_t*>(sf1); p.sf2 = static_cast<const uint8_t*>(sf2);
  p.gs1 = static_cast<const float*>(gs1); p.gs2 = static_cast<const float*>(gs2);
  p.ka1 = ka1; p.ka2 = ka2;
  const long long pairs = (static_cast<long long>(tokens) * topk + 15) / 16 * 16;
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.ids = reinterpret_cast<int*>(w);
  p.weights = reinterpret_cast<float*>(w + pairs * 4);
  p.mid = reinterpret_cast<float*>(w + pairs * 8);
  p.row_tiles = row_tiles;
  p.batch = fc2_batch(kind, tokens, inter);
  const int depth = fc1_room(kind, tokens, hidden, experts, cluster1) / (WARPS * stage_bytes(kind));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define HB_FEW(K)                                                   \
  e = depth >= 8   ? launch_few<K, 8>(p, cluster1, cluster2, st)    \
      : depth >= 6 ? launch_few<K, 6>(p, cluster1, cluster2, st)    \
                   : launch_few<K, 4>(p, cluster1, cluster2, st)
  if (kind == kGemmMxfp4) HB_FEW(kGemmMxfp4);
  else if (kind == kGemmNvfp4) HB_FEW(kGemmNvfp4);
  else HB_FEW(kGemmBf16);
#undef HB_FEW
  return e == cudaSuccess ? 0 : 2;
}

}  // extern "C"
