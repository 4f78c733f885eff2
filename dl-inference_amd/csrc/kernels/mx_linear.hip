// Linears on microscaled 4-bit weights on gfx950:
//   out[m, n] = sum_k x[m, k] * w[n, k] (+ bias[n]) (+ residual[m, n])
// on v_mfma_scale_f32_16x16x128_f8f6f4, which takes e4m3 or e2m1 elements with their blocks' scale
// codes and multiplies and scales in one instruction.
//
// Operand layout (lane l, g = l / 16): e2m1, 16 bytes: row l % 16, k = 32 g .. 32 g + 31; e4m3,
// 2 x 16 bytes: k = 16 g .. 16 g + 15, then the same + 64. The scale byte of lane l is that of row
// l % 16, block g of the 128 columns, for either element type. D[(l / 16) * 4 + i][l % 16].
#include "mx.h"

using namespace dk;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// The 16 or 32 bytes of one operand row that a lane feeds to one instruction (128 columns).
template <class F>
struct Frag {
  U32x4 q[F::kWords];
};

template <class F>
__device__ __forceinline__ i32x8 operand(const Frag<F>& f) {
  i32x8 v;
  const U32x4 lo = f.q[0], hi = f.q[F::kWords - 1];  // e2m1: the upper four registers are not read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = static_cast<int>(lo[i]);
    v[4 + i] = static_cast<int>(hi[i]);
  }
  return v;
}

// c + w x, w a fragment of 16 weight rows (e2m1), x one of 16 activation rows.
//
// Precision: the unit adds the products of 8 neighbouring columns after aligning them to the largest
// of the 8 and drops what lies below 2^-13 of it; further sums are fp32. Products of two e2m1
// values span less than that and are exact. With e4m3 the relative 2-norm error is 4e-6, far below
// the rounding of a 16-bit result. kSplit is for fp32 results: the e4m3 values of exponent fields
// 0..8 and 9..15 are multiplied by themselves; within each group the products of 8 columns span at
// most 13 bits, so nothing is dropped.
template <class F, bool kSplit>
__device__ __forceinline__ f32x4 mma(const Frag<MxFp4>& w, uint32_t sw, const Frag<F>& x,
                                     uint32_t sx, f32x4 c) {
  constexpr int kFp8 = 0, kFp4 = 4;
  constexpr int kX = F::kWords == 2 ? kFp8 : kFp4;
  if constexpr (kSplit && F::kWords == 2) {
    Frag<F> lo, hi;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // per byte: bit 7 of field + 0x38 is set from exponent field 9 (0x48) on
        const uint32_t top = ((x.q[j][i] & 0x78787878u) + 0x38383838u) & 0x80808080u;
        const uint32_t mask = (top - (top >> 7)) | top;
        hi.q[j][i] = x.q[j][i] & mask;
        lo.q[j][i] = x.q[j][i] & ~mask;
      }
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(lo), c, kFp4, kX, 0,
                                                         sw, 0, sx);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(hi), c, kFp4, kX,
                                                            0, sw, 0, sx);
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), c, kFp4, kX, 0,
                                                            sw, 0, sx);
  }
}

template <class F>
__device__ __forceinline__ Frag<F> loadFrag(const uint8_t* row, int64_t k0, int64_t k, int g) {
  Frag<F> f;
#pragma unroll
  for (int j = 0; j < F::kWords; ++j) {
    const int64_t at = k0 + (F::kWords == 2 ? j * 64 + g * 16 : g * 32);
    f.q[j] = at < k ? *gp(reinterpret_cast<const U32x4*>(row + at * F::kWords / 2))
                    : U32x4{0u, 0u, 0u, 0u};
  }
  return f;
}

// One wave per 16 x 16 tile of out.
template <class F, class T>
__device__ __forceinline__ void mx_linear_tile(const uint8_t* x, const uint8_t* xs,
                                               const uint8_t* w, const uint8_t* ws,
                                               const void* bias, const void* residual, void* out,
                                               int64_t M, int64_t N, int64_t K) {
  constexpr bool kSplit = sizeof(T) == 4;
  const int lane = threadIdx.x % kWave, g = lane / 16, r = lane % 16;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave) * 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 16;
  if (n0 >= N) return;
  const int64_t wr = n0 + r < N ? n0 + r : N - 1, xr = m0 + r < M ? m0 + r : M - 1;
  const int64_t blocks = K / kMxBlock;
  const uint8_t *pw = w + wr * (K / 2), *px = x + xr * (K * F::kWords / 2);
  const uint8_t *pws = ws + wr * blocks, *pxs = xs + xr * blocks;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int64_t k0 = 0; k0 < K; k0 += 128) {
    const int64_t b = k0 / kMxBlock + g;
    const uint32_t sw = b < blocks ? pws[b] : 127u, sx = b < blocks ? pxs[b] : 127u;
    acc = mma<F, kSplit>(loadFrag<MxFp4>(pw, k0, K, g), sw, loadFrag<F>(px, k0, K, g), sx, acc);
  }
  if (m0 + r >= M) return;
  T* po = static_cast<T*>(out) + (m0 + r) * N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + g * 4 + i;
    if (n >= N) break;
    float v = acc[i];
    if (bias != nullptr) v += ld(static_cast<const T*>(bias) + n);
    if (residual != nullptr) v += ld(static_cast<const T*>(residual) + (m0 + r) * N + n);
    st(po + n, v);
  }
}

}  // namespace

#define MX_LINEAR_KERNEL(name, F, T)                                                            \
  extern "C" __global__ void __launch_bounds__(256)                                             \
      name(const uint8_t* x, const uint8_t* xs, const uint8_t* w, const uint8_t* ws,            \
           const void* bias, const void* residual, void* out, int64_t M, int64_t N, int64_t K) { \
    mx_linear_tile<F, T>(x, xs, w, ws, bias, residual, out, M, N, K);                           \
  }
MX_LINEAR_KERNEL(mx_linear_tile_fp8_f32, MxFp8, float)
MX_LINEAR_KERNEL(mx_linear_tile_fp8_bf16, MxFp8, bf16)
MX_LINEAR_KERNEL(mx_linear_tile_fp8_f16, MxFp8, f16)
MX_LINEAR_KERNEL(mx_linear_tile_fp4_f32, MxFp4, float)
MX_LINEAR_KERNEL(mx_linear_tile_fp4_bf16, MxFp4, bf16)
MX_LINEAR_KERNEL(mx_linear_tile_fp4_f16, MxFp4, f16)
