// Operators around the microscaled linears on gfx950: quantisation, its inverse, RMSNorm with the
// residual's addition and a quantised output, and the gated activation with a quantised output.
// All are bound by the bytes they move. A lane takes 8 consecutive values (16 bytes of a 16-bit
// type), a quad of lanes one block of 32: the block's largest magnitude is two DPP steps away.
// From memory: fp4 codes of 18944 x 3584 bf16 values 34 us, 5.1 TB/s (a large copy: 5.0); the gated
// activation of 4096 x 18944 into fp8 84 us, 4.7 TB/s.
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

template <int kControl>
__device__ __forceinline__ double addDpp(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(b), kControl, 0xF, 0xF, true);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(b >> 32), kControl, 0xF, 0xF, true);
  return v + __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}

// Sum over the threads of a block (up to 4 waves), the same in every thread. Inside a wave it stays
// in registers: rotations in rows of 16 lanes, then rows and halves exchanged (12 ds_bpermute and
// the waits for them otherwise).
__device__ __forceinline__ double blockSum64(double v, double* scratch) {
  v = addDpp<0x121>(v);  // row_ror 1, 2, 4, 8
  v = addDpp<0x122>(v);
  v = addDpp<0x124>(v);
  v = addDpp<0x128>(v);
  uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  uint32_t lo = static_cast<uint32_t>(b), hi = static_cast<uint32_t>(b >> 32);
  auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
  auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
  v = __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(h[0]) << 32 | l[0])) +
      __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(h[1]) << 32 | l[1]));
  b = static_cast<uint64_t>(__double_as_longlong(v));
  lo = static_cast<uint32_t>(b), hi = static_cast<uint32_t>(b >> 32);
  l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
  h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  v = __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(h[0]) << 32 | l[0])) +
      __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(h[1]) << 32 | l[1]));
  if (blockDim.x == kWave) return v;
  __syncthreads();
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
  __syncthreads();
  const double half = scratch[0] + scratch[1];
  return blockDim.x == 2 * kWave ? half : half + (scratch[2] + scratch[3]);
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

// The sum of squares is held in 64 bits: the squares of 16-bit values are exact there and so,
// nearly always, is their sum, whatever its order. A scale is a step function of its block's
// largest value, and this keeps it from stepping with the order of a sum; it costs a conversion and
// an addition per value, hidden under the loads.
__device__ __forceinline__ void addSquares(const float (&h)[8], double& sq) {
#pragma unroll
  for (int j = 0; j < 8; ++j) sq += static_cast<double>(h[j]) * static_cast<double>(h[j]);
}

// share: 1 / hidden. In 64 bits, as squares of large fp32 values leave the range of fp32.
__device__ __forceinline__ float inverseRms(double sq, double share, float eps) {
  return static_cast<float>(rsqrt(sq * share + static_cast<double>(eps)));
}

template <class F, bool kVec>
__device__ __forceinline__ void normStore8(float (&h)[8], const float (&g)[8], float inv,
                                           uint8_t* codes, uint8_t* scales, int64_t c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = h[j] * inv * g[j];
  uint32_t w[F::kWords];
  const uint32_t code = mxQuantize8<F>(h, w);
  mxStoreCodes<F, kVec>(codes, c, w);
  if (threadIdx.x % 4 == 0) scales[c / 4] = static_cast<uint8_t>(code);
}

// A row of at most kHeld chunks per thread: read once, all loads in flight together, and held over
// the sum as it is in memory (as floats it would take twice the registers, and the waves that a CU
// holds carry this kernel).
template <class T, class F, bool kVec, int kHeld>
__device__ __forceinline__ void normHeld(const T* px, const T* pr, const T* pw, T* ph,
                                         uint8_t* codes, uint8_t* scales, int64_t r, int64_t chunks,
                                         double share, float eps, double* scratch) {
  MxRaw8<T> held[kHeld];
  double sq = 0.0;
#pragma unroll
  for (int s = 0; s < kHeld; ++s) {
    const int64_t i = threadIdx.x + s * static_cast<int64_t>(blockDim.x);
    if (i >= chunks) break;
    float h[8];
    hidden8<T, kVec>(px, pr, i, h);
    if (ph != nullptr) mxStore8<T, kVec>(ph + i * 8, h);
    addSquares(h, sq);
    held[s] = mxPack8<T>(h);
  }
  const float inv = inverseRms(blockSum64(sq, scratch), share, eps);
#pragma unroll
  for (int s = 0; s < kHeld; ++s) {
    const int64_t i = threadIdx.x + s * static_cast<int64_t>(blockDim.x);
    if (i >= chunks) break;
    float h[8], g[8];
    mxUnpack8<T>(held[s], h);
    mxLoad8<T, kVec>(pw + i * 8, g);
    normStore8<F, kVec>(h, g, inv, codes, scales, r * chunks + i);
  }
}

// One block per row. With x, residual and hidden_out in bf16 and fp8 codes, 8192 rows of 3584: 45.8 us,
// 4.5 TB/s (50.7 us with the row held as floats, 57.7 with the mean's root and quotient in 64-bit
// library steps and the sum over ds_bpermute); one row of 896: about 4 us, the latency of a launch.
template <class T, class F, bool kVec>
__device__ __forceinline__ void rms_norm_mx_impl(const void* x, const void* residual,
                                                 const void* weight, void* hidden_out,
                                                 uint8_t* codes, uint8_t* scales, int64_t rows,
                                                 int64_t hidden, double share, float eps) {
  __shared__ double scratch[4];
  const T* pw = static_cast<const T*>(weight);
  const int64_t chunks = hidden / 8, held = (chunks + blockDim.x - 1) / blockDim.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* px = static_cast<const T*>(x) + r * hidden;
    const T* pr = residual == nullptr ? nullptr : static_cast<const T*>(residual) + r * hidden;
    T* ph = hidden_out == nullptr ? nullptr : static_cast<T*>(hidden_out) + r * hidden;
    if (held == 1) {
      normHeld<T, F, kVec, 1>(px, pr, pw, ph, codes, scales, r, chunks, share, eps, scratch);
    } else if (held == 2) {
      normHeld<T, F, kVec, 2>(px, pr, pw, ph, codes, scales, r, chunks, share, eps, scratch);
    } else if (held <= 4) {
      normHeld<T, F, kVec, 4>(px, pr, pw, ph, codes, scales, r, chunks, share, eps, scratch);
    } else {  // read twice
      double sq = 0.0;
      for (int64_t i = threadIdx.x; i < chunks; i += blockDim.x) {
        float h[8];
        hidden8<T, kVec>(px, pr, i, h);
        if (ph != nullptr) mxStore8<T, kVec>(ph + i * 8, h);
        addSquares(h, sq);
      }
      const float inv = inverseRms(blockSum64(sq, scratch), share, eps);
      for (int64_t i = threadIdx.x; i < chunks; i += blockDim.x) {
        float h[8], g[8];
        if (ph != nullptr)  // the thread's own stores (hidden_out may be x or residual)
          mxLoad8<T, kVec>(ph + i * 8, h);
        else
          hidden8<T, kVec>(px, pr, i, h);
        mxLoad8<T, kVec>(pw + i * 8, g);
        normStore8<F, kVec>(h, g, inv, codes, scales, r * chunks + i);
      }
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
               uint8_t* codes, uint8_t* scales, int64_t rows, int64_t hidden, double share, float eps),
              (x, residual, weight, hidden_out, codes, scales, rows, hidden, share, eps))
DK_MX_KERNELS(silu_mul_mx, 256,
              (const void* gate, const void* up, int64_t stride, uint8_t* codes, uint8_t* scales,
               int64_t rows, int64_t row_chunks),
              (gate, up, stride, codes, scales, rows, row_chunks))
