// Numbers in 8 bits: e4m3 (four significant bits, largest 448, no infinities) with one scale for each block of 128.
//
// Rows (activations, gradients) are cut into blocks of 128 columns.  A block's scale is the smallest power of two s >= 2^-126 with
// max |v| <= 448 s: dividing by it is exact, so that the 8 bits of a value depend on the value and its block's largest alone, and
// the matrix instruction applies it by itself (it takes a power of two, held as its exponent + 127 in 8 bits, per operand row).  A
// scale that is no power of two would use at most one more binade of e4m3's subnormals.  NaN and infinities become NaN; a block
// that holds an infinity keeps nothing of its other values.
// Rows are Kp = K rounded up to 16 bytes long, filled with zeros, so that they start where 16-byte pieces can; those that a product
// reads from a workspace are rounded up to whole blocks.  Their scales are rows of KB = ceil(K / 128) bytes, KB rounded up to 4 apart.
#pragma once
#include "common.hpp"

namespace smoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

static constexpr int QB = 128;                                     // columns (and, of weights, rows) that share a scale

__host__ __device__ static inline int64_t padded_row(int64_t k) { return (k + 15) / 16 * 16; }
__host__ __device__ static inline int64_t block_row(int64_t k) { return (k + QB - 1) / QB * QB; }
__host__ __device__ static inline int64_t scale_blocks(int64_t k) { return (k + QB - 1) / QB; }
__host__ __device__ static inline int64_t scale_row(int64_t k) { return (scale_blocks(k) + 3) / 4 * 4; }

// exponent + 127 of the scale of a block whose largest magnitude is `top`: 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_byte(float top) {
  const unsigned u = __builtin_bit_cast(unsigned, top);
  return max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
}
__device__ __forceinline__ float scale_of(int byte) { return __builtin_bit_cast(float, byte << 23); }
// of any byte of a weight's scale, its lowest (2^-127) and the one that is no number among them
__device__ __forceinline__ float weight_scale(int byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x400000 : byte == 255 ? 0x7fc00000 : byte << 23);
}

// four values divided by their scale, a power of two, to the nearest of e4m3 (ties to even); the conversion takes what is above
// 448 to NaN, and nothing finite is
__device__ __forceinline__ int to_e4m3x4(float a, float b, float c, float d, float scale) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  const i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(i16x2{0, 0}, a, b, scale, false);
  return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true));
}
// times a scale that is a power of two
__device__ __forceinline__ void from_e4m3x4_exact(int q, float s, float (&v)[4]) {
  const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q, s, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q, s, true);
  v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
}
__device__ __forceinline__ void from_e4m3x4(int q, float s, float (&v)[4]) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(q, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(q, true);
  v[0] = lo[0] * s, v[1] = lo[1] * s, v[2] = hi[0] * s, v[3] = hi[1] * s;
}

// The largest of 16 neighbouring lanes' values, in each of them (four rotations of a row of 16); not-a-numbers are passed over
__device__ __forceinline__ float max16(float v) {
#define SMOE_ROTATED(n) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + n, 0xf, 0xf, false))
  v = fmaxf(v, SMOE_ROTATED(1));
  v = fmaxf(v, SMOE_ROTATED(2));
  v = fmaxf(v, SMOE_ROTATED(4));
  v = fmaxf(v, SMOE_ROTATED(8));
#undef SMOE_ROTATED
  return v;
}

// 32 values of e4m3 as bfloat16, which holds every one of them: eight of each of four matrix instructions' operands
typedef __bf16 bf16x8_8b __attribute__((ext_vector_type(8)));
typedef int i32x4_8b __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void to_bf16x32(i32x8 q, bf16x8_8b (&v)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    i32x4_8b r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[2 * i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * u + i], 1.0f, false));
      r[2 * i + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * u + i], 1.0f, true));
    }
    v[u] = __builtin_bit_cast(bf16x8_8b, r);
  }
}

// 16 values times their scale, a power of two, which bfloat16 holds as well (values under 2^-126 may lose bits)
__device__ __forceinline__ void to_bf16x16(i32x4_8b q, float scale, bf16x8_8b (&v)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    i32x4_8b r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[2 * i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * u + i], scale, false));
      r[2 * i + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * u + i], scale, true));
    }
    v[u] = __builtin_bit_cast(bf16x8_8b, r);
  }
}

// How a product applies scales and adds up.  The matrix cores' sums of 8-bit products are short of float32's: of eight neighbouring products
// each loses what lies below 2^-13 of the largest one's binade before they are added (measured; the sums of eights are
// added, and kept, in 32 bits).  128 to 4096 products of normal values end up 1.3e-5 of the result's norm off, whatever the
// instruction: 1/130 of what rounding the result to bfloat16 costs, 1/16 of float16, and too much beside float32.  Rows that came in float32
// are multiplied as bfloat16, which holds e4m3 exactly, at half the rate; so are float16 rows where the results go to 8 bits again.
enum Scaling8 {
  SCALES_BYTES,                                                    // all by the matrix instruction
  SCALES_FLOAT,                                                    // the rows' by the instruction, the weights' on every slice's sums
  SCALES_EXACT                                                     // both on every slice's sums, of bfloat16 products
};

// ---- arguments ---------------------------------------------------------------------------------------
struct QuantRowsArgs {
  const void* X; int64_t sxm;                                      // columns contiguous
  const int64_t* idx; int fan;                                     // row n is source row idx[n] / fan; NULL: n, of n / fan with coeff
  const void* coeff;                                               // times coeff[idx[n]], coeff[n]; NULL: 1
  int64_t rows, K;                                                 // (rows: of the source where there is coeff, and no idx)
  uint8_t* Q; uint8_t* S;
  int64_t slots;                                                   // with idx: entries outside [0, slots) make a row of zeros
  int64_t ld;                                                      // bytes of a row of Q, a multiple of 16, zeros behind the last value
  // Rows that a later product writes by slot: those of slots that the routing dropped it leaves alone, and a sum over a token's slots reads
  // them.  All are set to zero where kept[0] < clear.rows, here, ahead of the product, since this launch is there anyway.
  struct Clear {
    char* at; int64_t rows, bytes, ld;
    const int64_t* kept;
  } clear;
};
int launch_quantize_rows(const QuantRowsArgs& a, int dtype, hipStream_t st);

// weights (E, N, K), contraction contiguous, -> Q (E, N, Kp), QT (E, K, Np) (NULL: not wanted), S (E, NB, KB): a scale per 128 x 128
struct QuantWeightsArgs {
  const void* W; int64_t swe, swn;
  int E; int64_t N, K;
  uint8_t* Q; uint8_t* QT; uint8_t* S;
};
int launch_quantize_weights(const QuantWeightsArgs& a, int dtype, hipStream_t st);
// Y (E, N, K) contiguous from Q and its scales, one for each `tall` (1 or 128) rows x 128 columns, 8 bits or float32
struct DequantArgs {
  const uint8_t* Q; int64_t sqe, sqn;
  const void* S; int64_t sse, ssn, ssk; int s_f32, tall;
  int E; int64_t N, K;
  void* Y;
};
int launch_dequantize(const DequantArgs& a, int dtype, hipStream_t st);

// gated unit, forward: pre (rows, 2F) in `pre_dtype` -> h in `dtype` or (H8, HS) in 8 bits; P8 (rows, 2, Fp), PS (rows, 2, FB): the linear half and the gate's
// of pre in 8 bits, each with blocks of its own (NULL: not wanted)
struct UnitArgs {
  const void* pre; int64_t spm;
  void* h; uint8_t* H8; uint8_t* HS;                               // rows of H8 are whole blocks long
  uint8_t* P8; uint8_t* PS;
  int64_t rows, F;
  int act;
};
int launch_unit_fwd(const UnitArgs& a, int dtype, hipStream_t st);
// ... backward: d(pre) from the halves of pre in 8 bits and dh, in `dtype` or (D8, DS) in 8 bits with blocks along all 2F columns
struct UnitBackArgs {
  const uint8_t* P8; const uint8_t* PS;
  const void* dh; int64_t sdh;
  void* dpre; uint8_t* D8; uint8_t* DS;                            // rows of D8 are whole blocks long
  void* h;                                                         // the unit's value of the halves in 8 bits, too (NULL: not wanted)
  int64_t rows, F;
  int act;
};
int launch_unit_bwd(const UnitBackArgs& a, int dtype, hipStream_t st);

// Y[dst(n)] = X[src(n)] W[e(n)]^T (+ b[e(n)]) over rows sorted by expert, X and W in 8 bits
struct Product8Args {
  const uint8_t* X; const uint8_t* XS;                            // rows of whole blocks, 128 bytes more behind the last; scales as above
  const uint8_t* W; int64_t swe, swn;                             // (E, N, K), contraction contiguous, K a multiple of 16
  const void* WS; int64_t sse, ssn, ssk; int ws_f32;              // a scale per 128 x 128: 8 bits or float32
  const void* b; int64_t sbe, sbn;
  void* Y; int64_t sym;                                           // `out_dtype`
  const int64_t* idx; const int64_t* off;
  int L, K, N, E, fan, x_grouped, y_grouped;
  // instead of Y, of a product whose rows come out by expert:
  //   the gated unit on its columns (two halves of F = N / 2): H8, HS, and the halves themselves, P8, PS, where wanted
  //   the gated unit's gradient, the product being dh (F = N), from P8, PS: H8, HS, blocks along all 2F columns
  uint8_t* H8 = nullptr; uint8_t* HS = nullptr; uint8_t* P8 = nullptr; uint8_t* PS = nullptr;
  int act = 0;
  float* partial = nullptr;                                        // product_8bit_floats() of them, or NULL
};
// floats with which a product can cut the contraction of the tiles of its last round (0: it would not)
int64_t product_8bit_floats(int64_t L, int64_t K, int64_t columns, int E, bool exact);
// whether a product can be followed by the unit, or by its gradient, within its tiles
bool unit_rides(int64_t d, int64_t F);
bool unit_grad_rides(int64_t F);
enum Epilogue8 { EPI_ROWS, EPI_UNIT, EPI_UNIT_GRAD };
// exact: sums of bfloat16 products (SCALES_EXACT; whose rows come out in float32); row_dtype: of the rows that were taken to 8 bits and of the bias
int launch_product_8bit(const Product8Args& a, bool exact, int row_dtype, int out_dtype, hipStream_t st, int epilogue = EPI_ROWS);

// The same for a few rows per expert (csrc/few_rows_8bit.hip)
struct Few8Args {
  const void* X; int64_t sxm;                                     // float rows, columns contiguous, or rows in 8 bits (whole blocks) with XS
  const uint8_t* XS; int x_vec;                                   // x_vec: float rows start at multiples of 16 bytes
  const uint8_t* W; int64_t swe;                                  // (E, N, K rounded up to 16)
  const void* WS; int64_t sse, ssn, ssk; int ws_f32;
  const void* b; int64_t sbe, sbn;
  void* Y; int64_t sym; int out_dtype;                            // EPI_UNIT: the unit's values, float32
  const int64_t* ids;                                             // (L) expert of every slot, L <= 64: rows are slots; or NULL:
  const int64_t* idx; const int64_t* off;                         // rows sorted by expert
  int L, K, N, E, fan, x_grouped, y_grouped, act;
};
int launch_few_rows_8bit(const Few8Args& a, int x_dtype, int dtype, int epilogue, hipStream_t st);      // x_dtype -1: 8 bits
// What follows the experts' float32 rows (csrc/slots_f32.hip): out[t] = sum_j G[t, j] Y[t k + j] (G NULL: the sum; ids, or NULL: slots outside [0, E) are left
// out), and the gates' gradient <Y[t k + j], D[t]>
int launch_slots_combine(const float* Y, int64_t sy, const void* G, int64_t sgt, int64_t sgk, const int64_t* ids, int E, void* O, int64_t so, int64_t Tn,
                         int k, int N, int dtype, hipStream_t st);
int launch_slots_gate_grad(const float* Y, int64_t sy, const void* D, int64_t sd, void* DG, int64_t sgt, int64_t sgk, int64_t Tn, int k, int N, int dtype,
                           hipStream_t st);
int launch_few_combine(const float* rows, const void* gates, const int64_t* ids, void* out, int T, int k, int d, int E, int dtype, hipStream_t st);
__device__ __forceinline__ float bias_value(const void* b, int64_t at, int dtype) {
  if (dtype == SMOE_BF16) return to_f32(((const bf16_t*)b)[at]);
  if (dtype == SMOE_F16) return to_f32(((const f16_t*)b)[at]);
  return ((const float*)b)[at];
}

}  // namespace smoe
