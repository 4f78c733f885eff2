#pragma once

// Microscaled (MX) tensors on gfx950: blocks of 32 values along a row share one scale, a power of
// two held as its biased exponent (one byte, 255 = NaN); elements are e4m3 (one byte) or e2m1
// (four bits, two to a byte, the lower index in the low half).
#include "common.h"

namespace dk {

constexpr int kMxBlock = 32;

typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef float F32x2 __attribute__((ext_vector_type(2)));

// An element type: the exponent and magnitude of its largest element, 8 elements in kWords words.
struct MxFp8 {
  static constexpr int kTop = 8;
  static constexpr float kLargest = 448.f;
  static constexpr int kWords = 2;
  // 8 values, already divided by their scale, rounded to nearest even (v_cvt_pk_fp8_f32 gives NaN
  // above 464, so the magnitude is limited first).
  static __device__ __forceinline__ void pack(const float (&v)[8], uint32_t (&w)[kWords]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int p = 0;
      p = __builtin_amdgcn_cvt_pk_fp8_f32(limit(v[4 * i]), limit(v[4 * i + 1]), p, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(limit(v[4 * i + 2]), limit(v[4 * i + 3]), p, true);
      w[i] = static_cast<uint32_t>(p);
    }
  }
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[kWords], float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const F32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
      const F32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
      v[4 * i] = lo[0];
      v[4 * i + 1] = lo[1];
      v[4 * i + 2] = hi[0];
      v[4 * i + 3] = hi[1];
    }
  }

 private:
  static __device__ __forceinline__ float limit(float v) {
    return __builtin_amdgcn_fmed3f(v, -kLargest, kLargest);
  }
};

struct MxFp4 {
  static constexpr int kTop = 2;
  static constexpr int kWords = 1;
  // v_cvt_scalef32_pk_fp4_f32 rounds to nearest even and saturates at 6
  static __device__ __forceinline__ void pack(const float (&v)[8], uint32_t (&w)[kWords]) {
    uint32_t p = 0;
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[0], v[1], 1.f, 0);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[2], v[3], 1.f, 1);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[4], v[5], 1.f, 2);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[6], v[7], 1.f, 3);
    w[0] = p;
  }
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[kWords], float (&v)[8]) {
    const F32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 0);
    const F32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 1);
    const F32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 2);
    const F32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], 1.f, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
  }
};

// Largest magnitude of a value or an earlier one, as bits: integer order is the order of
// magnitudes, with infinity and then NaN above every finite value (fmaxf drops a NaN).
__device__ __forceinline__ uint32_t mxMax(uint32_t most, float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b > most ? b : most;
}

// The same over the 4 lanes of a quad, which hold one block between them.
__device__ __forceinline__ uint32_t mxQuadMax(uint32_t most) {
  const uint32_t a = __builtin_amdgcn_update_dpp(0, most, 0xB1, 0xF, 0xF, true);  // lane ^ 1
  most = a > most ? a : most;
  const uint32_t b = __builtin_amdgcn_update_dpp(0, most, 0x4E, 0xF, 0xF, true);  // lane ^ 2
  return b > most ? b : most;
}

// Scale code of a block: the exponent of its largest magnitude less that of the largest element,
// so that magnitudes reach the element type's top binade; at least 0 (2^-127); 255 where the
// block holds an infinity or a NaN.
template <class F>
__device__ __forceinline__ uint32_t mxScale(uint32_t most) {
  const int e = static_cast<int>(most >> 23);
  return e == 255 ? 255u : static_cast<uint32_t>(e > F::kTop ? e - F::kTop : 0);
}

// 1 / 2^(code - 127), an exact multiplier (code is at most 252); 0 for the NaN code.
__device__ __forceinline__ float mxInverse(uint32_t code) {
  return code == 255u ? 0.f : __uint_as_float((254u - code) << 23);
}

__device__ __forceinline__ float mxScaleValue(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7FC00000u)
                      : __uint_as_float(code == 0u ? 0x00400000u : code << 23);
}

// 8 values, the lane's quarter of a block -> words of elements; returns the block's scale code.
template <class F>
__device__ __forceinline__ uint32_t mxQuantize8(const float (&y)[8], uint32_t (&w)[F::kWords]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = mxMax(most, y[i]);
  const uint32_t code = mxScale<F>(mxQuadMax(most));
  const float inverse = mxInverse(code);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = y[i] * inverse;
  F::pack(v, w);
  if (code == 255u) {  // NaN * 0: the elements of a NaN block are zeros
#pragma unroll
    for (int i = 0; i < F::kWords; ++i) w[i] = 0u;
  }
  return code;
}

// 8 values of T as they lie in memory, for values that stay in registers: half the registers of
// floats where T has 16 bits.
template <class T>
struct MxRaw8 {
  uint32_t w[2 * sizeof(T)];
};

template <class T>
__device__ __forceinline__ void mxUnpack8(const MxRaw8<T>& raw, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(raw.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, bf16)) {
        v[2 * i] = __uint_as_float(raw.w[i] << 16);
        v[2 * i + 1] = __uint_as_float(raw.w[i] & 0xFFFF0000u);
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 h = __builtin_bit_cast(h2, raw.w[i]);
        v[2 * i] = static_cast<float>(h[0]);
        v[2 * i + 1] = static_cast<float>(h[1]);
      }
    }
  }
}

template <class T>
__device__ __forceinline__ MxRaw8<T> mxPack8(const float (&v)[8]) {
  MxRaw8<T> raw;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, bf16)) {
        raw.w[i] = packBf16x2(v[2 * i], v[2 * i + 1]);
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 h = {static_cast<_Float16>(v[2 * i]), static_cast<_Float16>(v[2 * i + 1])};
        raw.w[i] = __builtin_bit_cast(uint32_t, h);
      }
    }
  }
  return raw;
}

// 8 consecutive values as floats. kVec: p is 16-byte aligned.
template <class T, bool kVec>
__device__ __forceinline__ void mxLoad8(const T* p, float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ld(p + i);
  } else {
    MxRaw8<T> raw;
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j) {
      const U32x4 a = gp(reinterpret_cast<const U32x4*>(p))[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) raw.w[4 * j + i] = a[i];
    }
    mxUnpack8<T>(raw, v);
  }
}

template <class T, bool kVec>
__device__ __forceinline__ void mxStore8(T* p, const float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) st(p + i, v[i]);
  } else {
    const MxRaw8<T> raw = mxPack8<T>(v);
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j) {
      U32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = raw.w[4 * j + i];
      gp(reinterpret_cast<U32x4*>(p))[j] = a;
    }
  }
}

// Words of elements of chunk c (8 values) of a tensor. kVec: codes is 8-byte aligned.
template <class F, bool kVec>
__device__ __forceinline__ void mxStoreCodes(uint8_t* codes, int64_t c,
                                             const uint32_t (&w)[F::kWords]) {
  uint8_t* p = codes + c * (4 * F::kWords);
  if constexpr (!kVec) {
#pragma unroll
    for (int i = 0; i < 4 * F::kWords; ++i) p[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
  } else if constexpr (F::kWords == 2) {
    *gp(reinterpret_cast<U32x2*>(p)) = U32x2{w[0], w[1]};
  } else {
    *gp(reinterpret_cast<uint32_t*>(p)) = w[0];
  }
}

template <class F, bool kVec>
__device__ __forceinline__ void mxLoadCodes(const uint8_t* codes, int64_t c,
                                            uint32_t (&w)[F::kWords]) {
  const uint8_t* p = codes + c * (4 * F::kWords);
  if constexpr (!kVec) {
#pragma unroll
    for (int i = 0; i < F::kWords; ++i) w[i] = 0u;
#pragma unroll
    for (int i = 0; i < 4 * F::kWords; ++i) w[i / 4] |= static_cast<uint32_t>(p[i]) << (8 * (i % 4));
  } else if constexpr (F::kWords == 2) {
    const U32x2 v = *gp(reinterpret_cast<const U32x2*>(p));
    w[0] = v[0];
    w[1] = v[1];
  } else {
    w[0] = *gp(reinterpret_cast<const uint32_t*>(p));
  }
}

}  // namespace dk

// Instantiates `extern "C"` kernels base_<format>_<dtype> (16-byte data) and
// base_<format>_<dtype>_any (any alignment) from base_impl<T, F, kVec>.
#define DK_MX_KERNEL(base, bounds, suffix, T, F, VEC, ARGS, CALL)                        \
  extern "C" __global__ void __launch_bounds__(bounds) base##_##suffix ARGS {           \
    base##_impl<T, F, VEC> CALL;                                                        \
  }
#define DK_MX_KERNELS(base, bounds, ARGS, CALL)                                          \
  DK_MX_KERNEL(base, bounds, fp8_f32, float, dk::MxFp8, true, ARGS, CALL)               \
  DK_MX_KERNEL(base, bounds, fp8_bf16, dk::bf16, dk::MxFp8, true, ARGS, CALL)           \
  DK_MX_KERNEL(base, bounds, fp8_f16, dk::f16, dk::MxFp8, true, ARGS, CALL)             \
  DK_MX_KERNEL(base, bounds, fp4_f32, float, dk::MxFp4, true, ARGS, CALL)               \
  DK_MX_KERNEL(base, bounds, fp4_bf16, dk::bf16, dk::MxFp4, true, ARGS, CALL)           \
  DK_MX_KERNEL(base, bounds, fp4_f16, dk::f16, dk::MxFp4, true, ARGS, CALL)             \
  DK_MX_KERNEL(base, bounds, fp8_f32_any, float, dk::MxFp8, false, ARGS, CALL)          \
  DK_MX_KERNEL(base, bounds, fp8_bf16_any, dk::bf16, dk::MxFp8, false, ARGS, CALL)      \
  DK_MX_KERNEL(base, bounds, fp8_f16_any, dk::f16, dk::MxFp8, false, ARGS, CALL)        \
  DK_MX_KERNEL(base, bounds, fp4_f32_any, float, dk::MxFp4, false, ARGS, CALL)          \
  DK_MX_KERNEL(base, bounds, fp4_bf16_any, dk::bf16, dk::MxFp4, false, ARGS, CALL)      \
  DK_MX_KERNEL(base, bounds, fp4_f16_any, dk::f16, dk::MxFp4, false, ARGS, CALL)
