// Operators around the microscaled linears on gfx950: quantisation, its inverse, RMSNorm with the
// residual's addition and a quantised output, and the gated activation with a quantised output.
// All are bound by the bytes they move. A lane takes 8 consecutive values (16 bytes of a 16-bit
// type), a quad of lanes one block of 32: the block's largest magnitude is two DPP steps away.
#include "mx.h"

using namespace dk;

namespace {

// Rows are a multiple of 32 long, so the tensor is one run of blocks.
template <class T, class F, bool kVec>
__device__ __forceinline__ void mx_quantize_impl(const void* x, uint8_t* codes, uint8_t* scales,
                                                 int64_t chunks) {
  const T* px = static_cast<const T*>(x);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  // chunks is a multiple of 4 and so are step and the block size: a quad stays together
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; c < chunks;
       c += step) {
    float y[8];
    mxLoad8<T, kVec>(px + c * 8, y);
    uint32_t w[F::kWords];
    const uint32_t code = mxQuantize8<F>(y, w);
    mxStoreCodes<F, kVec>(codes, c, w);
    if (threadIdx.x % 4 == 0) scales[c / 4] = static_cast<uint8_t>(code);
  }
}

template <class T, class F, bool kVec>
__device__ __forceinline__ void mx_dequantize_impl(const uint8_t* codes, const uint8_t* scales,
                                                   void* out, int64_t chunks) {
  T* po = static_cast<T*>(out);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; c < chunks;
       c += step) {
    uint32_t w[F::kWords];
    mxLoadCodes<F, kVec>(codes, c, w);
    const float s = mxScaleValue(scales[c / 4]);
    float v[8];
    F::unpack(w, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
    mxStore8<T, kVec>(po + c * 8, v);
  }
}

// Sum over the 256 threads of a block, the same in every thread.
__device__ __forceinline__ double blockSum64(double v, double* scratch) {
#pragma unroll
  for (int offset = kWave / 2; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  return (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
}

// h = x + residual of chunk i of a row, rounded to T as the add operator rounds it
template <class T, bool kVec>
__device__ __forceinline__ void hidden8(const T* x, const T* residual, int64_t i, float (&h)[8]) {
  mxLoad8<T, kVec>(x + i * 8, h);
  if (residual != nullptr) {
    float r[8];
    mxLoad8<T, kVec>(residual + i * 8, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = Num<T>::round(h[j] + r[j]);
  }
}

// One block per row, the row read twice. The sum of squares is held in 64 bits: the squares of
// 16-bit values are exact there and so, nearly always, is their sum, whatever its order. A scale is
// a step function of its block's largest value, and this keeps it from stepping with the order of a
// sum; it costs a conversion and an addition per value, hidden under the loads.
template <class T, class F, bool kVec>
__device__ __forceinline__ void rms_norm_mx_impl(const void* x, const void* residual,
                                                 const void* weight, void* hidden_out,
                                                 uint8_t* codes, uint8_t* scales, int64_t rows,
                                                 int64_t hidden, float eps) {
  FP_EXACT
  __shared__ double scratch[4];
  const T* pw = static_cast<const T*>(weight);
  const int64_t chunks = hidden / 8;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* px = static_cast<const T*>(x) + r * hidden;
    const T* pr = residual == nullptr ? nullptr : static_cast<const T*>(residual) + r * hidden;
    T* ph = hidden_out == nullptr ? nullptr : static_cast<T*>(hidden_out) + r * hidden;
    double sq = 0.0;
    for (int64_t i = threadIdx.x; i < chunks; i += blockDim.x) {
      float h[8];
      hidden8<T, kVec>(px, pr, i, h);
      if (ph != nullptr) mxStore8<T, kVec>(ph + i * 8, h);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq += static_cast<double>(h[j]) * static_cast<double>(h[j]);
    }
    const double mean = blockSum64(sq, scratch) / static_cast<double>(hidden);
    const float inv = static_cast<float>(1.0 / sqrt(mean + static_cast<double>(eps)));
    for (int64_t i = threadIdx.x; i < chunks; i += blockDim.x) {
      float h[8], g[8];
      if (ph != nullptr)  // the thread's own stores (hidden_out may be x or residual)
        mxLoad8<T, kVec>(ph + i * 8, h);
      else
        hidden8<T, kVec>(px, pr, i, h);
      mxLoad8<T, kVec>(pw + i * 8, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = h[j] * inv * g[j];
      uint32_t w[F::kWords];
      const uint32_t code = mxQuantize8<F>(h, w);
      const int64_t c = r * chunks + i;
      mxStoreCodes<F, kVec>(codes, c, w);
      if (threadIdx.x % 4 == 0) scales[c / 4] = static_cast<uint8_t>(code);
    }
  }
}

template <class T, class F, bool kVec>
__device__ __forceinline__ void silu_mul_mx_impl(const void* gate, const void* up, int64_t stride,
                                                 uint8_t* codes, uint8_t* scales, int64_t rows,
                                                 int64_t row_chunks) {
  const int64_t chunks = rows * row_chunks;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; c < chunks;
       c += step) {
    const int64_t r = c / row_chunks, at = r * stride + (c - r * row_chunks) * 8;
    float g[8], u[8];
    mxLoad8<T, kVec>(static_cast<const T*>(gate) + at, g);
    mxLoad8<T, kVec>(static_cast<const T*>(up) + at, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = g[j] / (1.f + expf(-g[j])) * u[j];
    uint32_t w[F::kWords];
    const uint32_t code = mxQuantize8<F>(g, w);
    mxStoreCodes<F, kVec>(codes, c, w);
    if (threadIdx.x % 4 == 0) scales[c / 4] = static_cast<uint8_t>(code);
  }
}

}  // namespace

DK_MX_KERNELS(mx_quantize, 256,
              (const void* x, uint8_t* codes, uint8_t* scales, int64_t chunks),
              (x, codes, scales, chunks))
DK_MX_KERNELS(mx_dequantize, 256,
              (const uint8_t* codes, const uint8_t* scales, void* out, int64_t chunks),
              (codes, scales, out, chunks))
DK_MX_KERNELS(rms_norm_mx, 256,
              (const void* x, const void* residual, const void* weight, void* hidden_out,
               uint8_t* codes, uint8_t* scales, int64_t rows, int64_t hidden, float eps),
              (x, residual, weight, hidden_out, codes, scales, rows, hidden, eps))
DK_MX_KERNELS(silu_mul_mx, 256,
              (const void* gate, const void* up, int64_t stride, uint8_t* codes, uint8_t* scales,
               int64_t rows, int64_t row_chunks),
              (gate, up, stride, codes, scales, rows, row_chunks))
