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
constexpr int FC1_WARPS = 12;
constexpr int FC2_WARPS = 8;
constexpr int COLS = 8;                  // tokens of a unit: the N side of mma.m16n8k16
constexpr int MAX_SMEM = 227 * 1024;

struct FewParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* route_x;
  const __nv_bfloat16* router;
  const float* logits;                   // instead of route_x / router: computed by another kernel
  const float* sel_bias;
  const __nv_bfloat16* shared;
  __nv_bfloat16* out;
  long long ldx, ld_route, ld_router, ld_logits, ld_shared, ldo;
  int tokens, experts, topk, hidden, inter, h_out, route_k;
  int sigmoid, renorm;
  float scale;
  const uint8_t *w1, *w2, *sf1, *sf2;
  const float *gs1, *gs2;
  int ka1, ka2;
  int* ids;                              // workspace: what fc1 leaves for fc2
  float* weights;
  float* mid;                            // [pairs][inter]
  uint8_t* mid_exp;                      // [pairs][exp_ld]: biased exponent of the largest number of each fc1 tile
  int exp_ld;
};

// The routing as every CTA holds it: entries (an expert and up to eight of its tokens) in ascending order of experts.
struct Plan {
  int entries;
  int ids[MAX_PAIRS];
  float weights[MAX_PAIRS];
  uint32_t tokens_of[MAX_EXPERTS];       // bit t: token t chose the expert
  unsigned short expert[MAX_PAIRS], first[MAX_PAIRS], count[MAX_PAIRS];   // of entries; `first` indexes `pair`
  unsigned short pair[MAX_PAIRS];        // token * topk + j, by expert, then token
  int warp_sum[32];
};

template <int FMT>
struct Traits {
  static constexpr bool kFp4 = FMT != kGemmBf16;
  static constexpr int STEP_K = kFp4 ? 128 : 32;            // K elements of 64 bytes of a row
  static constexpr int SC_BYTES = FMT == kGemmMxfp4 ? 64 : FMT == kGemmNvfp4 ? 128 : 0;
  static constexpr int STAGE = 16 * 64 + SC_BYTES;
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

// A row of largest magnitude m (its bits) goes to fp16 times 2^(141 - E), E the biased exponent of m: m lands in [2^14, 2^15).
// Rows of all but nothing keep E = 15, where factor and inverse are still normal numbers; an infinity or a NaN stays one.
__device__ __forceinline__ int range_exp(uint32_t bits) { return min(max(static_cast<int>(bits >> 23), 15), 254); }
__device__ __forceinline__ float range_in(int e) { return __int_as_float((268 - e) << 23); }
__device__ __forceinline__ float range_out(int e) { return __int_as_float((e - 14) << 23); }

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
  long long to_b;                  // from row m to row m + 8
  const uint8_t* s;
  int left;                        // bytes of the row from this lane's chunk on

  __device__ __forceinline__ void init(uint32_t ring_addr, int lane) {
    ring = ring_addr;
    const int m = lane >> 2, c = lane & 3;
    dst = m * 64 + ((c ^ ((m >> 1) & 3)) << 4);
    left = 0;
  }
  __device__ __forceinline__ void set(const uint8_t* w, const uint8_t* sf, long long row0, int tile, int row_bytes, int ka, int lane) {
    const int m = lane >> 2, c = lane & 3;
    a = w + (row0 + tile_row<FMT>(tile, m)) * row_bytes + c * 16;
    to_b = static_cast<long long>(T::kFp4 ? 64 : 8) * row_bytes;
    left = row_bytes - c * 16;
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
      if (lane < T::SC_BYTES / 16) cp_async16(st + 1024 + lane * 16, s + static_cast<long long>(step) * (T::SC_BYTES * 8), true);
  }
};

// One step: acc += W[16 rows][STEP_K] * b, where b(block) gives the lane's eight 16-bit activations at 32 * block + 8 * (lane % 4)
// of its column lane / 4. A lane holds those same K positions of its two weight rows, so K is permuted alike on both sides.
template <int FMT, typename B>
__device__ __forceinline__ void step_mma(float (&acc)[4], uint32_t st, int lane, B&& b) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (FMT == kGemmBf16) {
    const uint32_t at = st + g * 64 + ((t ^ ((g >> 1) & 3)) << 4);
    const uint4 u = lds128(at), v = lds128(at + 512), x = b(0);
    mma_16816<true>(acc, u.x, v.x, u.y, v.y, x.x, x.y);
    mma_16816<true>(acc, u.z, v.z, u.w, v.w, x.z, x.w);
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
          const uint32_t u = r[h][2 * q], v = r[h][2 * q + 1];
          const uint4 x = b(2 * h + q);
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816<false>(part, e2m1x2_to_half2(u & 255u), e2m1x2_to_half2(v & 255u), e2m1x2_to_half2((u >> 8) & 255u),
                           e2m1x2_to_half2((v >> 8) & 255u), x.x, x.y);
          mma_16816<false>(part, e2m1x2_to_half2((u >> 16) & 255u), e2m1x2_to_half2((v >> 16) & 255u), e2m1x2_to_half2(u >> 24),
                           e2m1x2_to_half2(v >> 24), x.z, x.w);
          const float ga = q ? fa.y : fa.x, gb = q ? fb.y : fb.x;
          acc[0] = fmaf(part[0], ga, acc[0]);
          acc[1] = fmaf(part[1], ga, acc[1]);
          acc[2] = fmaf(part[2], gb, acc[2]);
          acc[3] = fmaf(part[3], gb, acc[3]);
        }
      }
    } else {
      // NVFP4: words 0 and 1 of a chunk belong to one block of 16, words 2 and 3 to the next; the scale (4 significant bits
      // times 2 of the value: exact) is multiplied in before the product
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t sa = lds32(sc + h * 64) >> (8 * (t >> 1)), sb = lds32(sc + h * 64 + 8) >> (8 * (t >> 1));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t fa = e4m3_h2(sa >> (16 * q)), fb = e4m3_h2(sb >> (16 * q));
          const uint32_t u = r[h][2 * q], v = r[h][2 * q + 1];
          const uint4 x = b(2 * h + q);
          mma_16816<false>(acc, hmul2(e2m1x2_to_half2(u & 255u), fa), hmul2(e2m1x2_to_half2(v & 255u), fb),
                           hmul2(e2m1x2_to_half2((u >> 8) & 255u), fa), hmul2(e2m1x2_to_half2((v >> 8) & 255u), fb), x.x, x.y);
          mma_16816<false>(acc, hmul2(e2m1x2_to_half2((u >> 16) & 255u), fa), hmul2(e2m1x2_to_half2((v >> 16) & 255u), fb),
                           hmul2(e2m1x2_to_half2(u >> 24), fa), hmul2(e2m1x2_to_half2(v >> 24), fb), x.z, x.w);
        }
      }
    }
  }
}

// Entries of the routing in plan.ids, by a whole CTA. An expert's tokens are a mask, so their order does not depend on timing.
__device__ __forceinline__ void make_plan(Plan& plan, int tokens, int experts, int topk) {
  const int tid = threadIdx.x, n = blockDim.x, lane = tid & 31, warp = tid >> 5, pairs = tokens * topk;
  for (int e = tid; e < experts; e += n) plan.tokens_of[e] = 0;
  __syncthreads();
  for (int p = tid; p < pairs; p += n) atomicOr(&plan.tokens_of[plan.ids[p]], 1u << (p / topk));
  __syncthreads();
  // exclusive sums over the experts of (entries << 16 | pairs), `per` consecutive experts a thread
  const int per = (experts + n - 1) / n;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    const int c = e < experts ? __popc(plan.tokens_of[e]) : 0;
    mine += ((c + COLS - 1) / COLS) << 16 | c;
  }
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) plan.warp_sum[warp] = inc;
  __syncthreads();
  int at = inc - mine;
  for (int w = 0; w < warp; ++w) at += plan.warp_sum[w];
  if (tid == n - 1) plan.entries = (at + mine) >> 16;
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e >= experts) break;
    const uint32_t mask = plan.tokens_of[e];
    int left = __popc(mask), entry = at >> 16, first = at & 0xFFFF;
    at += ((left + COLS - 1) / COLS) << 16 | left;
    uint32_t m = mask;
    for (int c = 0; left > 0; ++c, ++entry, left -= COLS) {
      plan.expert[entry] = static_cast<unsigned short>(e);
      plan.first[entry] = static_cast<unsigned short>(first);
      plan.count[entry] = static_cast<unsigned short>(min(left, COLS));
      for (int j = 0; j < COLS && m != 0; ++j, ++first) {
        const int t = __ffs(m) - 1;
        m &= m - 1;
        int k = 0;
        while (plan.ids[t * topk + k] != e) ++k;            // (it is there: the mask says so)
        plan.pair[first] = static_cast<unsigned short>(t * topk + k);
      }
    }
  }
  __syncthreads();
}

__device__ __forceinline__ uint32_t order_key(float v) {          // orders floats as unsigned numbers; never 0
  const uint32_t b = __float_as_uint(v);
  return max((b & 0x80000000u) ? ~b : (b | 0x80000000u), 1u);
}

// Top-k of one token by one warp; `score` and `key` [experts] are its scratch, `score` holds the logits on entry. Lane j < topk
// returns id and weight. Same arithmetic and order as moe_route_kernel (moe.cu).
__device__ __forceinline__ void warp_topk(const FewParams& p, float* score, uint32_t* key, int& id, float& weight) {
  const int lane = threadIdx.x & 31, E = p.experts;
  if (p.sigmoid) {
    for (int e = lane; e < E; e += 32) {
      const float s = 1.f / (1.f + __expf(-score[e]));
      score[e] = s;
      key[e] = order_key(s + (p.sel_bias != nullptr ? p.sel_bias[e] : 0.f));
    }
  } else {
    float mx = -INFINITY;
    for (int e = lane; e < E; e += 32) mx = fmaxf(mx, score[e]);
    mx = warp_max(mx);
    float sum = 0.f;
    for (int e = lane; e < E; e += 32) {
      const float s = __expf(score[e] - mx);
      score[e] = s;
      sum += s;
    }
    const float inv = 1.f / warp_sum(sum);
    for (int e = lane; e < E; e += 32) {
      score[e] *= inv;
      key[e] = order_key(score[e]);
    }
  }
  uint32_t best = 0;
  int at = lane;
  auto rescan = [&] {
    best = 0;
    for (int e = lane; e < E; e += 32)
      if (key[e] > best) {
        best = key[e];
        at = e;
      }
  };
  rescan();
  __syncwarp();                       // scores of the other lanes' experts are read below
  float sum = 0.f;
  id = 0;
  weight = 0.f;
  for (int j = 0; j < p.topk; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const int win = static_cast<int>(__reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at) : 0x7FFFFFFFu));
    const float s = score[win];
    sum += s;
    if (lane == j) {
      id = win;
      weight = s;
    }
    if ((win & 31) == lane) {
      key[win] = 0;
      rescan();
    }
  }
  weight = (p.renorm ? weight / fmaxf(sum, 1e-20f) : weight) * p.scale;
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__host__ __device__ constexpr int align16(int v) { return (v + 15) & ~15; }
// Shared memory of fc1: plan | logits and keys of this CTA's tokens | largest magnitudes | activations | rings (the router's partial
// sums before they are used)
__host__ __device__ inline int fc1_x_pitch(int hidden, int step_k) { return (hidden + step_k - 1) / step_k * step_k * 2 + 64; }
__host__ __device__ inline int fc1_logit_rows(int tokens, int cluster) { return (tokens + cluster - 1) / cluster; }
__host__ __device__ inline int fc1_fixed_bytes(int tokens, int experts, int cluster) {
  return align16(sizeof(Plan)) + align16(fc1_logit_rows(tokens, cluster) * experts * 8) + MAX_TOKENS * 4;
}

template <int FMT, int D>
__global__ void __launch_bounds__(FC1_WARPS * 32, 1)
moe_few_fc1_kernel(const __grid_constant__ FewParams p, int swiglu) {
  using T = Traits<FMT>;
  extern __shared__ __align__(128) uint8_t sm[];
  uint32_t cluster;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(cluster));
  const uint32_t rank = cluster_ctarank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  Plan& plan = *reinterpret_cast<Plan*>(sm);
  const int lrows = fc1_logit_rows(p.tokens, cluster);
  float* logit = reinterpret_cast<float*>(sm + align16(sizeof(Plan)));          // [lrows][experts]
  uint32_t* key = reinterpret_cast<uint32_t*>(logit + lrows * p.experts);
  uint32_t* top_bits = reinterpret_cast<uint32_t*>(sm + fc1_fixed_bytes(p.tokens, p.experts, cluster) - MAX_TOKENS * 4);
  uint8_t* xs = sm + fc1_fixed_bytes(p.tokens, p.experts, cluster);
  const int pitch = fc1_x_pitch(p.hidden, T::STEP_K);
  uint8_t* rings = xs + align16(p.tokens * pitch);

  if (tid < MAX_TOKENS) top_bits[tid] = 0;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");    // peers' shared memory is there from the wait below on
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();

  // ---- activations: bf16 as they are, or fp16 scaled by a power of two per row
  const int segs = (p.hidden + 255) / 256;
  if constexpr (T::kFp4) {
    for (int u = warp; u < p.tokens * segs; u += FC1_WARPS) {
      const int tok = u / segs, k = (u % segs) * 256 + lane * 8;
      uint32_t m = 0;
      if (k < p.hidden) {
        const uint4 v = ld_step(reinterpret_cast<const uint4*>(p.x + tok * p.ldx + k));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max((w[i] << 16) & 0x7FFF0000u, w[i] & 0x7FFF0000u));
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == 0) atomicMax(&top_bits[tok], m);
    }
    __syncthreads();
  }
  for (int u = warp; u < p.tokens * segs; u += FC1_WARPS) {
    const int tok = u / segs, k = (u % segs) * 256 + lane * 8;
    if (k * 2 >= pitch - 64) continue;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k < p.hidden) v = ld_step(reinterpret_cast<const uint4*>(p.x + tok * p.ldx + k));
    if constexpr (T::kFp4) {
      const float f = range_in(range_exp(top_bits[tok]));
      float e[8];
      unpack8(v, e);
      __half2 h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(e[2 * i] * f, e[2 * i + 1] * f);
      v = *reinterpret_cast<const uint4*>(h);
    }
    *reinterpret_cast<uint4*>(xs + tok * pitch + k * 2) = v;
  }

  // ---- router: a warp takes sixteen experts and one of `parts` shares of K; tiles of experts go round the cluster's CTAs
  const int e_tiles = (p.experts + 15) / 16;
  const int my_tiles = (e_tiles - static_cast<int>(rank) + static_cast<int>(cluster) - 1) / static_cast<int>(cluster);
  if (p.logits == nullptr) {
    float* part = reinterpret_cast<float*>(rings);                  // [tile][part][16 tokens][16 experts] of a round
    for (int round = 0; round < my_tiles; round += FC1_WARPS) {
      const int tiles = min(my_tiles - round, FC1_WARPS), parts = FC1_WARPS / tiles;
      const int tile = warp / parts, share = warp % parts;
      if (tile < tiles) {
        const int e0 = (static_cast<int>(rank) + (round + tile) * static_cast<int>(cluster)) * 16;
        const int blocks = (p.route_k + 31) / 32;
        float acc[2][4] = {};
        constexpr int U = 4;
        for (int b0 = share; b0 < blocks; b0 += parts * U) {
          uint4 wa[U], wb[U], xa[U], xb[U];
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int k = (b0 + i * parts) * 32 + t * 8;
            const uint4 zero = make_uint4(0, 0, 0, 0);
            const bool in = k < p.route_k;
            wa[i] = in && e0 + g < p.experts ? __ldg(reinterpret_cast<const uint4*>(p.router + (e0 + g) * p.ld_router + k)) : zero;
            wb[i] = in && e0 + g + 8 < p.experts ? __ldg(reinterpret_cast<const uint4*>(p.router + (e0 + g + 8) * p.ld_router + k)) : zero;
            xa[i] = in && g < p.tokens ? ld_step(reinterpret_cast<const uint4*>(p.route_x + g * p.ld_route + k)) : zero;
            xb[i] = in && g + 8 < p.tokens ? ld_step(reinterpret_cast<const uint4*>(p.route_x + (g + 8) * p.ld_route + k)) : zero;
          }
#pragma unroll
          for (int i = 0; i < U; ++i) {
            mma_16816<true>(acc[0], wa[i].x, wb[i].x, wa[i].y, wb[i].y, xa[i].x, xa[i].y);
            mma_16816<true>(acc[0], wa[i].z, wb[i].z, wa[i].w, wb[i].w, xa[i].z, xa[i].w);
            mma_16816<true>(acc[1], wa[i].x, wb[i].x, wa[i].y, wb[i].y, xb[i].x, xb[i].y);
            mma_16816<true>(acc[1], wa[i].z, wb[i].z, wa[i].w, wb[i].w, xb[i].z, xb[i].w);
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
      if (round == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      for (int i = tid; i < tiles * 256; i += FC1_WARPS * 32) {
        const int tl = i >> 8, tok = (i >> 4) & 15, e = (static_cast<int>(rank) + (round + tl) * static_cast<int>(cluster)) * 16 + (i & 15);
        if (tok < p.tokens && e < p.experts) {
          float s = 0.f;
          for (int w = 0; w < parts; ++w) s += part[(tl * parts + w) * 256 + (i & 255)];
          const uint32_t at = smem_u32(logit + (tok / static_cast<int>(cluster)) * p.experts + e);
          st_cluster(map_to_cta(at, tok % cluster), __float_as_uint(s));
        }
      }
      __syncthreads();
    }
    if (my_tiles <= 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = tid; i < lrows * p.experts; i += FC1_WARPS * 32) {
      const int tok = static_cast<int>(rank) + (i / p.experts) * static_cast<int>(cluster);
      if (tok < p.tokens) logit[i] = ld_step(p.logits + tok * p.ld_logits + i % p.experts);
    }
    __syncthreads();
  }
  cluster_sync_all();
  // ---- top-k: token `rank + i * cluster` by warp i; everybody gets the result
  for (int i = warp; i < lrows; i += FC1_WARPS) {
    const int tok = static_cast<int>(rank) + i * static_cast<int>(cluster);
    if (tok < p.tokens) {
      int id;
      float w;
      warp_topk(p, logit + i * p.experts, key + i * p.experts, id, w);
      if (lane < p.topk) {
        const int at = tok * p.topk + lane;
        for (uint32_t r = 0; r < cluster; ++r) {
          st_cluster(map_to_cta(smem_u32(&plan.ids[at]), r), static_cast<uint32_t>(id));
          st_cluster(map_to_cta(smem_u32(&plan.weights[at]), r), __float_as_uint(w));
        }
        if (blockIdx.x == rank) {        // the first cluster: fc2 makes the same plan
          p.ids[at] = id;
          p.weights[at] = w;
        }
      }
    }
  }
  cluster_sync_all();
  make_plan(plan, p.tokens, p.experts, p.topk);

  // ---- first product: a unit is (entry, 16 weight rows); units go round all warps of the grid
  const int n1 = swiglu ? 2 * p.inter : p.inter, tiles = n1 / 16, units = plan.entries * tiles;
  const int steps = (p.hidden + T::STEP_K - 1) / T::STEP_K;
  const int row_bytes = T::kFp4 ? p.hidden / 2 : p.hidden * 2;
  const int stride = gridDim.x * FC1_WARPS;
  Feed<FMT, D> feed;
  feed.init(smem_u32(rings) + warp * D * T::STAGE, lane);
  // (CTA first: few units spread over all SMs)
  int iu = static_cast<int>(blockIdx.x) + warp * static_cast<int>(gridDim.x), is = 0, islot = 0;
  auto aim = [&] {
    if (iu < units) {
      const int entry = iu / tiles;
      feed.set(p.w1, p.sf1, static_cast<long long>(plan.expert[entry]) * n1, iu - entry * tiles, row_bytes, p.ka1, lane);
    }
  };
  auto issue = [&] {
    if (iu < units) {
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
  int unit = iu, slot = 0;
  aim();
#pragma unroll 1
  for (int d = 0; d < D; ++d) issue();
  const uint32_t xs_addr = smem_u32(xs);
  while (unit < units) {
    const int entry = unit / tiles, tile = unit - entry * tiles;
    const int n = plan.count[entry], first = plan.first[entry];
    const bool live = g < n;
    const uint32_t xrow = xs_addr + (live ? plan.pair[first + g] / p.topk : 0) * pitch + t * 16;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      cp_async_wait<D - 1>();
      __syncwarp();
      step_mma<FMT>(acc, feed.ring + slot * T::STAGE, lane, [&](int blk) {
        return live ? lds128(xrow + (s * T::STEP_K + blk * 32) * 2) : make_uint4(0, 0, 0, 0);
      });
      __syncwarp();
      issue();
      slot = slot + 1 == D ? 0 : slot + 1;
    }
    // lane (g, t) holds rows g and g + 8 of columns 2 t and 2 t + 1
    const float gs = p.gs1 != nullptr ? p.gs1[plan.expert[entry]] : 1.f;
    int pr[2];
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = 2 * t + c;
      pr[c] = col < n ? plan.pair[first + col] : -1;
      const float f = pr[c] < 0 ? 0.f : T::kFp4 ? gs * range_out(range_exp(top_bits[pr[c] / p.topk])) : gs;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = acc[2 * h + c] * f;
        int row = tile_row<FMT>(tile, g + 8 * h);
        if (swiglu) {
          const float up = __shfl_xor_sync(0xffffffffu, v, 4);      // rows come in pairs: gate, up
          v = v / (1.f + __expf(-v)) * up;
          row >>= 1;
        } else {
          v = v <= 0.f ? 0.f : v * v;                               // (a NaN stays one)
        }
        if (pr[c] >= 0 && (!swiglu || (g & 1) == 0)) {
          p.mid[static_cast<long long>(pr[c]) * p.inter + row] = v;
          top[c] = max(top[c], __float_as_uint(v) & 0x7FFFFFFFu);
        }
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
      if (g == 0 && pr[c] >= 0) p.mid_exp[static_cast<long long>(pr[c]) * p.exp_ld + tile] = static_cast<uint8_t>(top[c] >> 23);
    }
    unit += stride;
  }
  cp_async_wait<0>();
}

// Shared memory of fc2: plan | rows' exponents | partial sums [warps][tokens][16] | rings
__host__ __device__ inline int fc2_fixed_bytes(int tokens) {
  return align16(sizeof(Plan)) + MAX_PAIRS * 4 + FC2_WARPS * tokens * 16 * 4;
}

template <int FMT, int D>
__global__ void __launch_bounds__(FC2_WARPS * 32, 2)
moe_few_fc2_kernel(const __grid_constant__ FewParams p, int units1, int cluster) {
  using T = Traits<FMT>;
  extern __shared__ __align__(128) uint8_t sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0, tile = blockIdx.x / cluster;
  Plan& plan = *reinterpret_cast<Plan*>(sm);
  uint32_t* row_top = reinterpret_cast<uint32_t*>(sm + align16(sizeof(Plan)));
  float* sums = reinterpret_cast<float*>(row_top + MAX_PAIRS);
  uint8_t* rings = sm + fc2_fixed_bytes(p.tokens);
  const int pairs = p.tokens * p.topk;

  for (int i = tid; i < FC2_WARPS * p.tokens * 16; i += FC2_WARPS * 32) sums[i] = 0.f;
  for (int i = tid; i < pairs; i += FC2_WARPS * 32) row_top[i] = 0;
  grid_dep_wait();
  grid_dep_launch();
  for (int i = tid; i < pairs; i += FC2_WARPS * 32) {
    plan.ids[i] = ld_step(p.ids + i);
    plan.weights[i] = ld_step(p.weights + i);
  }
  __syncthreads();
  if constexpr (T::kFp4) {               // largest exponent of every pair's row, from those of its tiles
    const int chunks = p.exp_ld / 16;
    for (int i = tid; i < pairs * chunks; i += FC2_WARPS * 32) {
      const int pr = i / chunks, c = i - pr * chunks;
      const uint4 v = ld_step(reinterpret_cast<const uint4*>(p.mid_exp + static_cast<long long>(pr) * p.exp_ld + c * 16));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c * 16 + j < units1) m = max(m, (w[j >> 2] >> (8 * (j & 3))) & 255u);
      atomicMax(&row_top[pr], m);
    }
  }
  make_plan(plan, p.tokens, p.experts, p.topk);

  const int steps = (p.inter + T::STEP_K - 1) / T::STEP_K;
  const int row_bytes = T::kFp4 ? p.inter / 2 : p.inter * 2;
  const int stride = cluster * FC2_WARPS;
  Feed<FMT, D> feed;
  feed.init(smem_u32(rings) + warp * D * T::STAGE, lane);
  int iu = rank * FC2_WARPS + warp, is = 0, islot = 0;
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
  constexpr int BLOCKS = T::STEP_K / 32;
  while (entry < plan.entries) {
    const int n = plan.count[entry], first = plan.first[entry];
    const bool live = g < n;
    const int my_pair = live ? plan.pair[first + g] : 0;
    const float* row = p.mid + static_cast<long long>(my_pair) * p.inter;
    const float f = T::kFp4 ? range_in(range_exp(row_top[my_pair] << 23)) : 1.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float4 raw[BLOCKS][2];
    auto fetch = [&](int s) {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const int k = s * T::STEP_K + b * 32 + t * 8;
        const bool in = live && k < p.inter;
        raw[b][0] = in ? ld_step(reinterpret_cast<const float4*>(row + k)) : make_float4(0.f, 0.f, 0.f, 0.f);
        raw[b][1] = in ? ld_step(reinterpret_cast<const float4*>(row + k + 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    fetch(0);
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      uint4 x[BLOCKS];
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const float4 u = raw[b][0], v = raw[b][1];
        if constexpr (T::kFp4) {
          const __half2 h[4] = {__floats2half2_rn(u.x * f, u.y * f), __floats2half2_rn(u.z * f, u.w * f),
                                __floats2half2_rn(v.x * f, v.y * f), __floats2half2_rn(v.z * f, v.w * f)};
          x[b] = *reinterpret_cast<const uint4*>(h);
        } else {
          x[b] = make_uint4(pack_bf16(u.x, u.y), pack_bf16(u.z, u.w), pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        }
      }
      if (s + 1 < steps) fetch(s + 1);
      cp_async_wait<D - 1>();
      __syncwarp();
      step_mma<FMT>(acc, feed.ring + slot * T::STAGE, lane, [&](int blk) { return x[blk]; });
      __syncwarp();
      issue();
      slot = slot + 1 == D ? 0 : slot + 1;
    }
    const float gs = p.gs2 != nullptr ? p.gs2[plan.expert[entry]] : 1.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = 2 * t + c;
      if (col < n) {
        const int pr = plan.pair[first + col], tok = pr / p.topk;
        float w = plan.weights[pr] * gs;
        if constexpr (T::kFp4) {
          // two factors: the row's exponent alone can reach what one product with the weight would lose
          const float back = range_out(range_exp(row_top[pr] << 23));
          mine[tok * 16 + g] += acc[c] * back * w;
          mine[tok * 16 + g + 8] += acc[2 + c] * back * w;
        } else {
          mine[tok * 16 + g] += acc[c] * w;
          mine[tok * 16 + g + 8] += acc[2 + c] * w;
        }
      }
    }
    __syncwarp();
    entry += stride;
  }
  cp_async_wait<0>();
  __syncthreads();
  // ---- sums over the warps, then over the cluster, in order
  const int n_out = p.tokens * 16;
  for (int i = tid; i < n_out; i += FC2_WARPS * 32) {
    float s = sums[i];
    for (int w = 1; w < FC2_WARPS; ++w) s += sums[w * n_out + i];
    sums[i] = s;
  }
  if (cluster > 1) cluster_sync_all();
  else __syncthreads();
  for (int i = tid + rank * FC2_WARPS * 32; i < n_out; i += FC2_WARPS * 32 * cluster) {
    float s = 0.f;
    if (cluster > 1) {
      const uint32_t at = smem_u32(sums + i);
      for (int r = 0; r < cluster; ++r) s += ld_dsmem_f32(map_to_cta(at, r));
    } else {
      s = sums[i];
    }
    const int tok = i >> 4, row = tile_row<FMT>(tile, i & 15);
    if (p.shared != nullptr) s += __bfloat162float(p.shared[tok * p.ld_shared + row]);
    p.out[tok * p.ldo + row] = __float2bfloat16(s);
  }
  if (cluster > 1) cluster_sync_all();       // nobody leaves while a peer may still read its sums
}

template <int FMT, int D>
cudaError_t launch_few(const FewParams& p, int swiglu, int cluster1, int cluster2, size_t smem1, cudaStream_t st) {
  using T = Traits<FMT>;
  auto k1 = moe_few_fc1_kernel<FMT, D>;
  auto k2 = moe_few_fc2_kernel<FMT, 8>;
  static const cudaError_t ready = [&] {
    cudaError_t e = cudaFuncSetAttribute(k1, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k1, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k2, cudaFuncAttributeMaxDynamicSharedMemorySize, 113 * 1024);
    return e;
  }();
  if (ready != cudaSuccess) return ready;
  const int grid1 = kNumSms / cluster1 * cluster1;
  cudaError_t e = launch_dep_cluster(k1, dim3(grid1), dim3(FC1_WARPS * 32), cluster1, smem1, st, p, swiglu);
  if (e != cudaSuccess) return e;
  const size_t smem2 = fc2_fixed_bytes(p.tokens) + FC2_WARPS * 8 * T::STAGE;
  const int units1 = (swiglu ? 2 * p.inter : p.inter) / 16;
  return launch_dep_cluster(k2, dim3(p.h_out / 16 * cluster2), dim3(FC2_WARPS * 32), cluster2, smem2, st, p, units1, cluster2);
}

}  // namespace
}  // namespace hb

extern "C" {

// Workspace bytes of hb_moe_few.
long long hb_moe_few_ws(int tokens, int topk, int inter) {
  const long long pairs = (static_cast<long long>(tokens) * topk + 15) / 16 * 16;
  return pairs * (8 + 4ll * inter + (inter / 8 + 15) / 16 * 16);
}

// Most tokens that one call takes at this width (0: none).
int hb_moe_few_tokens(int kind, int hidden, int experts, int cluster) {
  using namespace hb;
  const int step = kind == kGemmBf16 ? 32 : 128, stage = kind == kGemmBf16 ? 1024 : kind == kGemmMxfp4 ? 1088 : 1152;
  for (int t = MAX_TOKENS; t > 0; --t)
    if (fc1_fixed_bytes(t, experts, cluster) + align16(t * fc1_x_pitch(hidden, step)) + FC1_WARPS * 4 * stage <= MAX_SMEM) return t;
  return 0;
}

int hb_moe_few(int kind, const void* x, long long ldx, const void* route_x, long long ld_route, const void* router,
               long long ld_router, int route_k, const void* logits, long long ld_logits, const void* sel_bias, int tokens,
               int experts, int topk, int sigmoid, int renorm, float scale, int hidden, int inter, int h_out, int swiglu,
               const void* w1, const void* sf1, const void* gs1, int ka1, const void* w2, const void* sf2, const void* gs2, int ka2,
               const void* shared, long long ld_shared, void* out, long long ldo, void* ws, int cluster1, int cluster2,
               void* stream) {
  using namespace hb;
  const bool fp4 = is_fp4(kind);
  if (!fp4 && kind != kGemmBf16) return 1;
  if (tokens < 1 || experts < 1 || experts > MAX_EXPERTS || topk < 1 || topk > MAX_TOPK || topk > experts) return 1;
  if (tokens > hb_moe_few_tokens(kind, hidden, experts, cluster1)) return 1;
  const int n1 = swiglu ? 2 * inter : inter, rows = fp4 ? 128 : 16, k_of = fp4 ? 32 : 8;
  if (n1 < 1 || n1 % rows || h_out < 1 || h_out % rows || hidden % k_of || inter % k_of || inter % 8) return 1;
  if (logits == nullptr && (route_x == nullptr || router == nullptr || route_k < 8 || route_k % 8)) return 1;
  if (cluster1 < 1 || cluster1 > 16 || cluster2 < 1 || cluster2 > 8) return 1;
  FewParams p;
  p.x = static_cast<const __nv_bfloat16*>(x); p.route_x = static_cast<const __nv_bfloat16*>(route_x);
  p.router = static_cast<const __nv_bfloat16*>(router); p.logits = static_cast<const float*>(logits);
  p.sel_bias = static_cast<const float*>(sel_bias); p.shared = static_cast<const __nv_bfloat16*>(shared);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldx = ldx; p.ld_route = ld_route; p.ld_router = ld_router; p.ld_logits = ld_logits; p.ld_shared = ld_shared; p.ldo = ldo;
  p.tokens = tokens; p.experts = experts; p.topk = topk; p.hidden = hidden; p.inter = inter; p.h_out = h_out; p.route_k = route_k;
  p.sigmoid = sigmoid; p.renorm = renorm; p.scale = scale;
  p.w1 = static_cast<const uint8_t*>(w1); p.w2 = static_cast<const uint8_t*>(w2);
  p.sf1 = static_cast<const uint8_t*>(sf1); p.sf2 = static_cast<const uint8_t*>(sf2);
  p.gs1 = static_cast<const float*>(gs1); p.gs2 = static_cast<const float*>(gs2);
  p.ka1 = ka1; p.ka2 = ka2;
  const long long pairs = (static_cast<long long>(tokens) * topk + 15) / 16 * 16;
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.ids = reinterpret_cast<int*>(w);
  p.weights = reinterpret_cast<float*>(w + pairs * 4);
  p.mid = reinterpret_cast<float*>(w + pairs * 8);
  p.mid_exp = w + pairs * (8 + 4ll * inter);
  p.exp_ld = (inter / 8 + 15) / 16 * 16;
  const int step = fp4 ? 128 : 32, stage = kind == kGemmBf16 ? 1024 : kind == kGemmMxfp4 ? 1088 : 1152;
  const int base = fc1_fixed_bytes(tokens, experts, cluster1) + align16(tokens * fc1_x_pitch(hidden, step));
  const bool deep = base + FC1_WARPS * 8 * stage <= MAX_SMEM;
  const size_t smem1 = base + FC1_WARPS * (deep ? 8 : 4) * stage;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define HB_FEW(K) e = deep ? launch_few<K, 8>(p, swiglu, cluster1, cluster2, smem1, st) : launch_few<K, 4>(p, swiglu, cluster1, cluster2, smem1, st)
  if (kind == kGemmMxfp4) HB_FEW(kGemmMxfp4);
  else if (kind == kGemmNvfp4) HB_FEW(kGemmNvfp4);
  else HB_FEW(kGemmBf16);
#undef HB_FEW
  return e == cudaSuccess ? 0 : 2;
}

}  // extern "C"
