// Products of a few rows with weights that are read once: what the kernels of the few-token layer and of the adapters
// beside a shared projection have in common.
//
// A wave multiplies weight rows by input rows on the matrix cores, 16 x 16 x 32 (float32: 16 x 16 x 4), both operands straight
// from global memory into the registers that the instruction reads.  The order in which the contraction's elements meet is free
// as long as both operands use the same, so pieces of 16 bytes need no transposition and no LDS.  A lane's place in the instruction
// is (row l % 16, piece l / 16); 16 weight rows would take 64 bytes each per load, half a line.  Instead the 16 rows are
// 16 / P rows in P parts of the contraction: one load takes 64 P bytes of each of 16 / P rows, of weights and of inputs
// alike, and of the 16 x 16 sums those count whose parts agree; the others cost nothing, since the instruction's
// rate is not what bounds a stream.  Rows may start at any multiple of the element's size; the last piece of a
// row ends with the row, so nothing is read behind it.
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
  static __device__ __forceinline__ f32x4 mma(i32x4 w, i32x4 x, f32x4 c) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, w), __builtin_bit_cast(v8, x), c, 0, 0, 0);
  }
};
template <> struct Few<f16_t> {
  static constexpr int PER = 8;
  static __device__ __forceinline__ f32x4 mma(i32x4 w, i32x4 x, f32x4 c) {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, w), __builtin_bit_cast(v8, x), c, 0, 0, 0);
  }
};
template <> struct Few<float> {
  static constexpr int PER = 4;
  static __device__ __forceinline__ f32x4 mma(i32x4 w, i32x4 x, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(w[i]), __int_as_float(x[i]), c, 0, 0, 0);
    return c;
  }
};
// This lane's place: sub-row, part, and the offset of its piece among the 64 P bytes of a row
template <typename T, int P>
struct FewLane {
  static constexpr int ROWS = 16 / P;                        // rows of a load
  static constexpr int STEP = 4 * P * Few<T>::PER;           // contraction elements of a load
  int sub, part, q, at;
  __device__ __forceinline__ FewLane() {
    const int l = lane_id();
    sub = (l & 15) / P;
    part = (l & 15) % P;
    q = l >> 4;
    at = (part * 4 + q) * Few<T>::PER;
  }
};
// The sums of a group: every lane of part 0 gets, of input row sub, its weight rows VALUES q and up.
template <int P>
struct FewSums {
  static constexpr int VALUES = 4 / P;
  static __device__ __forceinline__ void take(const f32x4& acc, int part, float (&v)[VALUES]) {
    static_assert(P == 1 || P == 2 || P == 4, "parts of a group of four sums");
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
      float x = acc[i * P];
#pragma unroll
      for (int p = 1; p < P; ++p) x = part == p ? acc[i * P + p] : x;
      if constexpr (P > 1) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xb1, 0xf, 0xf, true));     // lane ^ 1
      if constexpr (P == 4) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4e, 0xf, 0xf, true));   // lane ^ 2
      v[i] = x;
    }
  }
};

// A float32 value as the sum of two of the operand's type: it rounded, and the rest rounded.  Together they are off by 2^-18
// (float16: 2^-24, or half its smallest number) of the value.  A value that is infinite as float16 stays so.
template <typename T>
__device__ __forceinline__ void split(float v, T& first, T& rest) {
  first = from_f32<T>(v);
  rest = __builtin_isinf(to_f32(first)) ? from_f32<T>(0.0f) : from_f32<T>(v - to_f32(first));
}

// 16 bytes from an address that is a multiple of the element's size.  ONCE: nobody reads them again.
template <typename T, bool ONCE>
__device__ __forceinline__ i32x4 load_piece(const T* p) {
  typedef typename std::conditional<sizeof(T) == 2, i32x4_by2, i32x4_by4>::type piece;
  if constexpr (ONCE) return __builtin_nontemporal_load((const piece*)p);
  else return *(const piece*)p;
}
// The last pieces of rows of at least PER elements, of which `left` (any number) lie from p to the row's end: the piece that
// ends with the row, with zeros in place of the elements before p.  Both operands of a product are read this way, so the
// elements that count still meet.
template <typename T>
__device__ __forceinline__ i32x4 load_piece_of(const T* p, int left) {
  constexpr int PER = Few<T>::PER, PER_DWORD = PER / 4;
  const int n = min(max(PER - left, 0), PER);                // elements that do not count
  i32x4 v = load_piece<T, false>(p + min(left - PER, 0));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int none = n - i * PER_DWORD;
    v[i] &= none <= 0 ? -1 : none >= PER_DWORD ? 0 : (int)0xffff0000;
  }
  return v;
}

// What a tile of WROWS weight rows and G groups of input rows leaves in LDS: the sum of wave v for weight row n and input row m
// at few_at<..>(v, n, m).
template <int WROWS, int INPUTS>
__device__ __forceinline__ int few_at(int wave, int n, int m) { return (wave * WROWS + n) * (INPUTS + 1) + m; }
template <int NW, int WROWS, int INPUTS>
static constexpr int FEW_PART = NW * WROWS * (INPUTS + 1);

// Products of WROWS weight rows with G groups of 16 / P input rows over K >= PER contraction elements, by NW waves that take blocks
// of the contraction in turn.  `weight(n)` / `input(m)`: the first element of such a row.  Inputs of H parts: `apart` elements
// from one part of a row to the next.  ONCE: no other workgroup reads these weights.  MORE: loads of each
// row that are issued side by side, if not the usual number.  Leaves the waves' sums in `part` (see few_at), without a barrier.
template <typename T, int P, int G, int H, int NW, int WROWS, bool ONCE = true, int MORE = 0, class Weight, class Input>
__device__ __forceinline__ void few_tile(Weight weight, Input input, int apart, int K, float* part) {
  typedef FewLane<T, P> Lane;
  constexpr int NT = WROWS / Lane::ROWS, LOADS = NT + G * H, SIDE = MORE ? MORE : LOADS <= 3 ? 4 : LOADS <= 6 ? 2 : 1, STEP = Lane::STEP, BLOCK = SIDE * STEP;
  constexpr int INPUTS = G * Lane::ROWS, V = FewSums<P>::VALUES;
  const Lane l;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* w[NT];
  const T* x[G];
#pragma unroll
  for (int j = 0; j < NT; ++j) w[j] = weight(j * Lane::ROWS + l.sub) + l.at;
#pragma unroll
  for (int i = 0; i < G; ++i) x[i] = input(i * Lane::ROWS + l.sub) + l.at;
  f32x4 acc[G][NT];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // a block's products: all its loads ahead of the first wait
  auto block = [&](int k0, auto load) {
    i32x4 wv[NT][SIDE], xv[G][H][SIDE];
#pragma unroll
    for (int s = 0; s < SIDE; ++s) {
#pragma unroll
      for (int j = 0; j < NT; ++j) wv[j][s] = load(w[j], k0 + s * STEP, std::integral_constant<bool, ONCE>());
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int p = 0; p < H; ++p) xv[i][p][s] = load(x[i] + p * apart, k0 + s * STEP, std::false_type());
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < SIDE; ++s)
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int p = 0; p < H; ++p)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = Few<T>::mma(wv[j][s], xv[i][p][s], acc[i][j]);
  };
  const int whole = K / BLOCK;
#pragma unroll 1
  for (int b = wave; b < whole; b += NW) block(b * BLOCK, [&](const T* p, int k, auto once) { return load_piece<T, decltype(once)::value>(p + k); });
  if (whole * BLOCK < K && wave == whole % NW)
    block(whole * BLOCK, [&](const T* p, int k, auto) { return load_piece_of<T>(p + k, K - k - l.at); });
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float v[V];
      FewSums<P>::take(acc[i][j], l.part, v);
      if (l.part == 0) {
#pragma unroll
        for (int c = 0; c < V; ++c)
          part[few_at<WROWS, INPUTS>(wave, j * Lane::ROWS + V * l.q + c, i * Lane::ROWS + l.sub)] = v[c];
      }
    }
}
// The waves' sums of one value, in their order
template <int NW, int WROWS, int INPUTS>
__device__ __forceinline__ float few_sum(const float* part, int n, int m) {
  float v = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; ++w) v += part[few_at<WROWS, INPUTS>(w, n, m)];
  return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// The dot products of one input row with DOT_ROWS weight rows over K >= PER contiguous elements, by a workgroup of DOT_NW waves that
// take its pieces in turn.  Thread j < DOT_ROWS returns with the j-th; `part`: DOT_NW * DOT_ROWS floats of LDS.
static constexpr int DOT_NW = 4, DOT_ROWS = 4, DOT_SIDE = 2;
template <typename T>
__device__ __forceinline__ float dot_rows(const T* x, const T* const (&w)[DOT_ROWS], int K, float* part) {
  constexpr int PER = Few<T>::PER, PIECE = 64 * PER;
  typedef T V __attribute__((ext_vector_type(PER)));
  float v[DOT_ROWS] = {};
  for (int k0 = threadIdx.x * PER; k0 < K; k0 += DOT_NW * PIECE * DOT_SIDE) {
    i32x4 xv[DOT_SIDE], wv[DOT_ROWS][DOT_SIDE];
#pragma unroll
    for (int p = 0; p < DOT_SIDE; ++p) {
      const int k = k0 + DOT_NW * PIECE * p;
      xv[p] = load_piece_of<T>(x + k, K - k);
#pragma unroll
      for (int j = 0; j < DOT_ROWS; ++j) wv[j][p] = load_piece_of<T>(w[j] + k, K - k);
    }
#pragma unroll
    for (int p = 0; p < DOT_SIDE; ++p)
#pragma unroll
      for (int j = 0; j < DOT_ROWS; ++j)
#pragma unroll
        for (int i = 0; i < PER; ++i)
          v[j] = fmaf(to_f32(__builtin_bit_cast(V, xv[p])[i]), to_f32(__builtin_bit_cast(V, wv[j][p])[i]), v[j]);
  }
#pragma unroll
  for (int j = 0; j < DOT_ROWS; ++j) {
    v[j] = wave_sum(v[j]);
    if (lane_id() == 0) part[(threadIdx.x >> 6) * DOT_ROWS + j] = v[j];
  }
  __syncthreads();
  float sum = 0.0f;
  if (threadIdx.x < DOT_ROWS) {
#pragma unroll
    for (int u = 0; u < DOT_NW; ++u) sum += part[u * DOT_ROWS + threadIdx.x];
  }
  return sum;
}

}  // namespace smoe
