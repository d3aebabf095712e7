// MXFP4 quantiser and its inverse for sm_100a.
//
// Format (OCP microscaling): blocks of 32 elements along K share a scale 2^(b - 127), b one byte (ue8m0); elements are e2m1.
//   b = max(floor(log2(max |x|)) - 2 + 127, 0)      (2 = exponent of e2m1's largest value; zeros: b = 0)
//   q = rne_e2m1(x * 2^(127 - b)), saturating at 6
// A block that holds an infinity or a NaN gets b = 255, the format's NaN: what reads it returns NaN, not a clipped number.
// The scale is a power of two, so x * 2^(127 - b) is exact and the only rounding is the one to e2m1.
//
// Packed values are row-major (low nibble first); scale bytes go to the 128 x 4 blocks that tcgen05.cp moves into TMEM, four
// of a row (128 elements) being one 32-bit word.
//
// Bound by bytes: 2 (bf16) or 4 in and 17/32 out per element. Two lanes share a block: each holds sixteen elements (one or two 32-byte
// loads), the maximum takes one shuffle, and eight lanes' scales make the word of an atom. A warp works on 1024 elements of a row at a
// time, all of its loads in flight at once.
//
// Measured, from memory: 2048 x 17408 bf16 quantised in 18.3 us (90 MB, 4.9 TB/s: bound by the instructions of the maxima and the packing;
// with eight elements a lane 21.7), back in 13.6; 17408 x 5120 fp32 68.9 (404 MB, 5.9 TB/s) and 62.0; one row of 5120 2.4 and 2.1, launch and
// latency. Half or twice as many elements a warp were slower (20.3, 18.9).
#include <type_traits>

#include "hb_api.h"
#include "hb_common.cuh"
#include "rownorm.cuh"

namespace hb {
namespace {

constexpr int QUANT_WARPS = 4;
constexpr int SEG = 1024;              // elements of a row per warp: 4 steps of 256
enum InType : int { kInBf16 = 0, kInF16 = 1, kInF32 = 2 };

// Sixteen consecutive elements, half a block; ALIGN: bytes that their address and the rows' pitch are multiples of (32, 16 or the type's).
template <int IN, int ALIGN>
struct Raw16 {
  static constexpr int WORDS = IN == kInF32 ? 16 : 8;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const void* x, long long i) {
    const uint8_t* at = static_cast<const uint8_t*>(x) + i * (IN == kInF32 ? 4 : 2);
    if constexpr (ALIGN == 32) {
#pragma unroll
      for (int j = 0; j < WORDS; j += 8)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[j]), "=r"(w[j + 1]), "=r"(w[j + 2]), "=r"(w[j + 3]), "=r"(w[j + 4]), "=r"(w[j + 5]), "=r"(w[j + 6]),
                       "=r"(w[j + 7])
                     : "l"(at + j * 4));
    } else if constexpr (ALIGN == 16) {
#pragma unroll
      for (int j = 0; j < WORDS; j += 4) {
        const uint4 v = ld_step(reinterpret_cast<const uint4*>(at + j * 4));
        w[j] = v.x; w[j + 1] = v.y; w[j + 2] = v.z; w[j + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        if constexpr (IN == kInF32) {
          w[j] = ld_step(reinterpret_cast<const uint32_t*>(at) + j);
        } else {
          const unsigned short* p = reinterpret_cast<const unsigned short*>(at) + 2 * j;
          w[j] = static_cast<uint32_t>(ld_step(p)) | static_cast<uint32_t>(ld_step(p + 1)) << 16;
        }
      }
    }
  }
  // Bits of the largest magnitude as a float (an order in which NaN comes last), 16-bit numbers compared two at a time.
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
    if constexpr (IN == kInF32) {
#pragma unroll
      for (int j = 0; j < WORDS; ++j) m = max(m, w[j] & 0x7FFFFFFFu);
      return m;
    } else {
#pragma unroll
      for (int j = 0; j < WORDS; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
      if constexpr (IN == kInBf16) return max(m << 16, m & 0xFFFF0000u);
      else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(max(m >> 16, m & 0xFFFFu)))));
    }
  }
  __device__ __forceinline__ void pair(int j, float& lo, float& hi) const {      // elements 2j, 2j + 1
    if constexpr (IN == kInF32) {
      lo = __uint_as_float(w[2 * j]);
      hi = __uint_as_float(w[2 * j + 1]);
    } else if constexpr (IN == kInBf16) {
      lo = bf16_lo(w[j]);
      hi = bf16_hi(w[j]);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      lo = t.x;
      hi = t.y;
    }
  }
};

// dst_rows (may be null; the expert-sorted buffers of a mixture-of-experts layer, m pairs of a token and one of its topk experts): pair r
// goes to row dst_rows[r], of token r / topk or, with topk 0, of the same row of x; an entry that is negative or not below dst_count (rows
// of the buffers, and with topk 0 of x) leaves the pair out. The other rows of the buffers (most of them, with few tokens: every expert's
// segment is padded to 128) are not touched.
template <int IN, int ALIGN>
__global__ void __launch_bounds__(QUANT_WARPS * 32, IN == kInF32 ? 9 : 12)
quant_mxfp4_kernel(const void* __restrict__ x, long long ldx, int m, int k, int ka, uint8_t* __restrict__ q,
                   uint8_t* __restrict__ sf, int segs, const int* __restrict__ dst_rows, int dst_count, int topk) {
  grid_dep_wait(x, dst_rows);
  grid_dep_launch();      // behind the wait: a grouped GEMM that follows reads the routing plan at once (see launch_dep)
  const uint32_t unit = blockIdx.x * QUANT_WARPS + (threadIdx.x >> 5);      // (the launch keeps it below 2^31)
  const int row = static_cast<int>(unit / static_cast<uint32_t>(segs)), seg = static_cast<int>(unit) - row * segs;
  const int lane = threadIdx.x & 31;
  if (row >= m) return;
  long long in_row = row;
  int dst = row;
  if (dst_rows != nullptr) {
    dst = dst_rows[row];
    if (static_cast<uint32_t>(dst) >= static_cast<uint32_t>(dst_count)) return;
    in_row = topk > 0 ? row / topk : dst;
  }
  const long long base = in_row * ldx;
  constexpr int STEP = 512, STEPS = SEG / STEP;
  const int k0 = seg * SEG + lane * 16;
  Raw16<IN, ALIGN> raw[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
    if (k0 + i * STEP < k) raw[i].load(x, base + k0 + i * STEP);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = k0 + i * STEP;                   // (k is a multiple of 32: a block is there as a whole or not at all)
    if (seg * SEG + i * STEP >= ka * 128) break;   // uniform
    uint32_t top = c < k ? raw[i].top() : 0u;
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    float inv;
    const uint32_t b = mx_scale(top, inv);
    if (c < k) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float lo, hi;
        raw[i].pair(j, lo, hi);
        w[j >> 2] |= e2m1x2(lo * inv, hi * inv) << (8 * (j & 3));
      }
      *reinterpret_cast<uint2*>(q + static_cast<size_t>(dst) * (k >> 1) + (c >> 1)) = make_uint2(w[0], w[1]);
    }
    // the four blocks of the eight lanes' atom as one word; blocks that pad the last K tile have b = 0
    uint32_t s = b << (8 * ((lane >> 1) & 3));
    s |= __shfl_xor_sync(0xffffffffu, s, 2);
    s |= __shfl_xor_sync(0xffffffffu, s, 4);
    const int g = c >> 5;
    if ((lane & 7) == 0 && (g >> 2) < ka) *reinterpret_cast<uint32_t*>(sf + row_sf_off(dst, g, ka)) = s;
  }
}

template <typename T>
__device__ __forceinline__ void store8(void* out, size_t i, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(void* out, size_t i, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + i) = pack8(v);
}
template <>
__device__ __forceinline__ void store8<__half>(void* out, size_t i, const float (&v)[8]) {
  __half2 h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<uint4*>(static_cast<__half*>(out) + i) = *reinterpret_cast<const uint4*>(h);
}
// Values of a packed matrix: e2m1 times 2^(b - 127). Both factors and (but for results past the largest float) the product are
// exact in 32 bits; 16-bit outputs are rounded once. The same split of a row as above.
template <typename T>
__global__ void __launch_bounds__(QUANT_WARPS * 32)
dequant_mxfp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf, int m, int k, int ka, void* __restrict__ out,
                     int segs) {
  grid_dep_wait(q, sf);
  grid_dep_launch();
  const uint32_t unit = blockIdx.x * QUANT_WARPS + (threadIdx.x >> 5);      // (the launch keeps it below 2^31)
  const int row = static_cast<int>(unit / static_cast<uint32_t>(segs)), seg = static_cast<int>(unit) - row * segs;
  const int lane = threadIdx.x & 31;
  if (row >= m) return;
  auto scale = [](uint32_t b) { return __uint_as_float(b == 255u ? 0x7FC00000u : b == 0u ? 0x00400000u : b << 23); };
  if constexpr (std::is_same<T, float>::value) {
    // four elements a lane, so that a store of the warp is 512 bytes in a row (of eight, two half-filled stores: 98 us instead of 62
    // for 17408 x 5120)
    uint32_t w[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = seg * SEG + i * 128 + lane * 4;
      if (c < k) {
        w[i] = ld_step(reinterpret_cast<const unsigned short*>(q + static_cast<size_t>(row) * (k >> 1) + (c >> 1)));
        b[i] = sf[row_sf_off(row, c >> 5, ka)];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = seg * SEG + i * 128 + lane * 4;
      if (c >= k) break;
      const float s = scale(b[i]);
      const float2 lo = e2m1x2_to_float2(w[i] & 255u), hi = e2m1x2_to_float2(w[i] >> 8);
      *reinterpret_cast<float4*>(static_cast<float*>(out) + static_cast<size_t>(row) * k + c) = make_float4(lo.x * s, lo.y * s, hi.x * s, hi.y * s);
    }
    return;
  } else {
    const int k0 = seg * SEG + lane * 8;
    uint32_t w[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = k0 + i * 256;
      if (c < k) {
        w[i] = ld_step(reinterpret_cast<const uint32_t*>(q + static_cast<size_t>(row) * (k >> 1) + (c >> 1)));
        b[i] = sf[row_sf_off(row, c >> 5, ka)];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = k0 + i * 256;
      if (c >= k) break;
      const float s = scale(b[i]);
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = e2m1x2_to_float2((w[i] >> (8 * j)) & 255u);
        v[2 * j] = t.x * s;
        v[2 * j + 1] = t.y * s;
      }
      store8<T>(out, static_cast<size_t>(row) * k + c, v);
    }
  }
}

template <int IN>
cudaError_t launch_quant(int align, const void* x, long long ldx, int m, int k, int ka, void* q, void* sf, const void* dst_rows,
                         int dst_count, int topk, cudaStream_t st) {
  const int segs = (ka * 128 + SEG - 1) / SEG;
  const long long units = static_cast<long long>(m) * segs, blocks = (units + QUANT_WARPS - 1) / QUANT_WARPS;
  if (units > 0x7FFFFFF0ll) return cudaErrorInvalidValue;
  auto kern = align == 32 ? quant_mxfp4_kernel<IN, 32> : align == 16 ? quant_mxfp4_kernel<IN, 16> : quant_mxfp4_kernel<IN, 0>;
  return launch_dep(kern, dim3(static_cast<unsigned>(blocks)),
                    dim3(QUANT_WARPS * 32), 0, st, x, ldx, m, k, ka, static_cast<uint8_t*>(q), static_cast<uint8_t*>(sf), segs,
                    static_cast<const int*>(dst_rows), dst_count, topk);
}

}  // namespace
}  // namespace hb

extern "C" {

int hb_quant_mxfp4(const void* x, int in_type, long long ldx, int m, int k, int ka, void* q, void* sf, const void* dst_rows,
                   int dst_count, int topk, void* stream) {
  using namespace hb;
  if (m < 1 || k < 32 || k % 32 != 0 || ka != (k + 255) / 256 * 2) return 1;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ldx * (in_type == kInF32 ? 4 : 2));
  const int align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (in_type) {
    case kInBf16: e = launch_quant<kInBf16>(align, x, ldx, m, k, ka, q, sf, dst_rows, dst_count, topk, st); break;
    case kInF16: e = launch_quant<kInF16>(align, x, ldx, m, k, ka, q, sf, dst_rows, dst_count, topk, st); break;
    case kInF32: e = launch_quant<kInF32>(align, x, ldx, m, k, ka, q, sf, dst_rows, dst_count, topk, st); break;
    default: return 1;
  }
  return e == cudaSuccess ? 0 : 2;
}

int hb_dequant_mxfp4(const void* q, const void* sf, int m, int k, int ka, void* out, int out_type, void* stream) {
  using namespace hb;
  if (m < 1 || k < 32 || k % 32 != 0 || ka != (k + 255) / 256 * 2) return 1;
  const int segs = (k + SEG - 1) / SEG;
  const long long blocks = (static_cast<long long>(m) * segs + QUANT_WARPS - 1) / QUANT_WARPS;
  if (static_cast<long long>(m) * segs > 0x7FFFFFF0ll) return 1;
  auto kern = out_type == kInBf16 ? dequant_mxfp4_kernel<__nv_bfloat16> : out_type == kInF16 ? dequant_mxfp4_kernel<__half>
                                                                                             : dequant_mxfp4_kernel<float>;
  if (out_type < 0 || out_type > 2) return 1;
  const cudaError_t e = launch_dep(kern, dim3(static_cast<unsigned>(blocks)), dim3(QUANT_WARPS * 32), 0,
                                   static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(q),
                                   static_cast<const uint8_t*>(sf), m, k, ka, out, segs);
  return e == cudaSuccess ? 0 : 2;
}

}  // extern "C"
