// Products of a few rows with weights that are read once: what the kernels of the few-token layer and of the adapters
// beside a shared projection have in common.
//
// A wave multiplies 16 NT weight rows by 16 MT input rows on the matrix cores, both operands straight from global memory
// into the registers that the instruction reads: lane l holds, of row l % 16, the 16 bytes number l / 16 of every 64.
// The order in which the contraction's elements meet is free as long as both operands use the same, so 16-byte pieces
// need no transposition and no LDS.  Rows may start at any multiple of the element's size; the last, partial pieces of a
// row are put together from single elements, so nothing is read behind a row's end.
#pragma once
#include "common.hpp"
#include <type_traits>

namespace smoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_by2 __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Few;
template <> struct Few<bf16_t> {
  static constexpr int PER = 8;                 // elements of a 16-byte piece
  static constexpr float LOW = 1.0f;            // what the second of two parts is held times (see split)
  static __device__ __forceinline__ f32x4 mma(i32x4 w, i32x4 x, f32x4 c) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, w), __builtin_bit_cast(v8, x), c, 0, 0, 0);
  }
};
template <> struct Few<f16_t> {
  static constexpr int PER = 8;
  static constexpr float LOW = 2048.0f;
  static __device__ __forceinline__ f32x4 mma(i32x4 w, i32x4 x, f32x4 c) {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, w), __builtin_bit_cast(v8, x), c, 0, 0, 0);
  }
};
template <> struct Few<float> {
  static constexpr int PER = 4;
  static constexpr float LOW = 1.0f;
  static __device__ __forceinline__ f32x4 mma(i32x4 w, i32x4 x, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(w[i]), __int_as_float(x[i]), c, 0, 0, 0);
    return c;
  }
};
// Contraction elements of a load instruction (64 bytes per row), and of the four that a wave issues side by side per row
template <typename T> static constexpr int FEW_STEP = 4 * Few<T>::PER;
template <typename T> static constexpr int FEW_BLOCK = 4 * FEW_STEP<T>;

// A float32 value as the sum of two of the operand's type: the first is it rounded, the second the rest times LOW,
// rounded.  bfloat16 has float32's exponents, so the rest needs no factor; float16's would be subnormal for a first part below
// 0.25 without one.  Together they are off by 2^-18 (2^-24) of the value.  A value that is infinite as float16 stays so.
template <typename T>
__device__ __forceinline__ void split(float v, T& first, T& rest) {
  first = from_f32<T>(v);
  const float r = v - to_f32(first);
  rest = __builtin_isinf(to_f32(first)) ? from_f32<T>(0.0f) : from_f32<T>(r * Few<T>::LOW);
}

// 16 bytes from an address that is a multiple of the element's size.  ONCE: nobody reads them again.
template <typename T, bool ONCE>
__device__ __forceinline__ i32x4 load_piece(const T* p) {
  typedef typename std::conditional<sizeof(T) == 2, i32x4_by2, i32x4_by4>::type piece;
  if constexpr (ONCE) return __builtin_nontemporal_load((const piece*)p);
  else return *(const piece*)p;
}
// The same of a row that has `left` more elements (any number), zeros behind them
template <typename T>
__device__ __forceinline__ i32x4 load_piece_of(const T* p, int left) {
  constexpr int PER = Few<T>::PER;
  if (left >= PER) return load_piece<T, false>(p);
  typedef T V __attribute__((ext_vector_type(PER)));
  V v;
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = i < left ? p[i] : from_f32<T>(0.0f);
  return __builtin_bit_cast(i32x4, v);
}

}  // namespace smoe
