// Passes between rows and their 8-bit form (eight_bit.hpp).  All of them are bound by what they read and write; 16 lanes own a
// block of 128 columns, eight each, so that its largest magnitude is four lane rotations away and the block is read once.
#include "eight_bit.hpp"

namespace smoe {

typedef int q_i32x4 __attribute__((ext_vector_type(4)));

// Eight consecutive values of a row from column c on, as float32; zeros from column K on.  VEC: whole 16-byte pieces.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t c, int64_t K, float (&v)[8]) {
  if constexpr (VEC) {
    if (c < K) {
      constexpr int PER = 16 / (int)sizeof(T);
      T t[8];
#pragma unroll
      for (int p = 0; p < 8 / PER; ++p)
        __builtin_memcpy(t + p * PER, (const char*)__builtin_assume_aligned((const char*)(row + c) + p * 16, 16), 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f32(row[c + i]) : 0.0f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ row, int64_t c, int64_t K, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c < K) {
      constexpr int PER = 16 / (int)sizeof(T);
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(v[i]);
#pragma unroll
      for (int p = 0; p < 8 / PER; ++p)
        __builtin_memcpy(__builtin_assume_aligned((char*)(row + c) + p * 16, 16), t + p * PER, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) row[c + i] = from_f32<T>(v[i]);
  }
}
__device__ __forceinline__ float top8(const float (&v)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
  return max16(m);
}
// the lane's eight values of a block in 8 bits (rows end at Kp, a multiple of 16), and its scale
__device__ __forceinline__ void store_block(uint8_t* __restrict__ q, uint8_t* __restrict__ s, int64_t c, int64_t Kp, const float (&v)[8]) {
  const int byte = scale_byte(top8(v));
  const float scale = scale_of(byte);
  if (c < Kp) *(i32x2*)(q + c) = i32x2{to_e4m3x4(v[0], v[1], v[2], v[3], scale), to_e4m3x4(v[4], v[5], v[6], v[7], scale)};
  if ((threadIdx.x & 15) == 0) *s = (uint8_t)byte;
}
__device__ __forceinline__ void load_block(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s, int64_t c, int64_t Kp, float (&v)[8]) {
  float lo[4] = {0, 0, 0, 0}, hi[4] = {0, 0, 0, 0};
  if (c < Kp) {
    const i32x2 p = *(const i32x2*)(q + c);
    const float f = scale_of(*s);
    from_e4m3x4_exact(p[0], f, lo);
    from_e4m3x4_exact(p[1], f, hi);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
}

// A pass's units of work: blocks of 128 of its rows, 16 lanes each, 16 of them per workgroup
struct Unit {
  int64_t row; int block; int64_t c;
  bool there;
  __device__ __forceinline__ Unit(int64_t rows, int blocks) {
    const unsigned u = blockIdx.x * 16u + (threadIdx.x >> 4);
    row = u / (unsigned)blocks;
    block = (int)(u - (unsigned)row * (unsigned)blocks);
    c = (int64_t)block * QB + (threadIdx.x & 15) * 8;
    there = row < rows;
  }
};
// Rows of one launch: so many that its units can be counted in 31 bits
static int64_t rows_per_launch(int64_t rows, int64_t blocks) {
  const int64_t most = (0x7fffff00LL / 16 * 16) / blocks;
  return rows < most ? rows : most;
}

// zeros for rows that a product may leave alone (at a kernel's end: its own work does not wait for kept[0])
template <typename V>
__device__ __forceinline__ void clear_all(const QuantRowsArgs::Clear& c) {
  const int64_t wide = c.bytes / (int64_t)sizeof(V), total = c.rows * wide;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += gridDim.x * (int64_t)256) {
    const int64_t row = i / wide;
    ((V*)(c.at + row * c.ld))[i - row * wide] = V{};
  }
}
__device__ __forceinline__ void clear_rows(const QuantRowsArgs::Clear& c) {
  if (!c.at || c.kept[0] >= c.rows) return;
  if ((((uintptr_t)c.at | c.bytes | c.ld) & 15) == 0) clear_all<q_i32x4>(c);
  else clear_all<short>(c);
}

template <typename T, bool VEC>
__device__ __forceinline__ void quantize_unit(const QuantRowsArgs& a, const Unit& u) {
  int64_t src = u.row;
  float f = 1.0f;
  bool have = true;                                                // (a row that the routing dropped has no source)
  if (a.idx) {
    const int64_t i = a.idx[u.row];
    have = i >= 0 && i < a.slots;
    src = have ? i / a.fan : 0;
    if (a.coeff && have) f = to_f32(((const T*)a.coeff)[i]);
  }
  float v[8];
  load8<T, VEC>((const T*)a.X + src * a.sxm, have ? u.c : a.K, a.K, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= f;
  store_block(a.Q + u.row * a.ld, a.S + u.row * scale_row(a.K) + u.block, u.c, a.ld, v);
}
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantRowsArgs a, int blocks) {
  const Unit u(a.rows, blocks);
  if (u.there) quantize_unit<T, VEC>(a, u);
  clear_rows(a.clear);
}
// a source row once, times each of its fan coefficients (8192 rows of 2048, 8 each: 84 us by idx, 29 so)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quantize_times_kernel(QuantRowsArgs a, int blocks) {
  const Unit u(a.rows, blocks);
  if (u.there) {
    float v[8], x[8];
    load8<T, VEC>((const T*)a.X + u.row * a.sxm, u.c, a.K, v);
    for (int j = 0; j < a.fan; ++j) {
      const int64_t n = u.row * a.fan + j;
      const float f = to_f32(((const T*)a.coeff)[n]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = v[i] * f;
      store_block(a.Q + n * a.ld, a.S + n * scale_row(a.K) + u.block, u.c, a.ld, x);
    }
  }
  clear_rows(a.clear);
}

template <typename T>
static int quantize_rows(QuantRowsArgs a, hipStream_t st) {
  const int64_t blocks = scale_blocks(a.K), Sr = scale_row(a.K);
  const bool vec = ((uintptr_t)a.X & 15) == 0 && a.sxm * (int64_t)sizeof(T) % 16 == 0 && a.K % 8 == 0;
  const bool times = a.coeff && !a.idx;
  int64_t left = a.rows;
  while (left > 0) {
    a.rows = rows_per_launch(left, blocks);
    const dim3 grid((unsigned)((a.rows * blocks + 15) / 16));
    if (times && vec) quantize_times_kernel<T, true><<<grid, 256, 0, st>>>(a, (int)blocks);
    else if (times) quantize_times_kernel<T, false><<<grid, 256, 0, st>>>(a, (int)blocks);
    else if (vec) quantize_rows_kernel<T, true><<<grid, 256, 0, st>>>(a, (int)blocks);
    else quantize_rows_kernel<T, false><<<grid, 256, 0, st>>>(a, (int)blocks);
    left -= a.rows;
    if (a.idx) a.idx += a.rows;
    else a.X = (const T*)a.X + a.rows * a.sxm;
    const int64_t made = a.rows * (times ? a.fan : 1);
    if (times) a.coeff = (const T*)a.coeff + made;
    a.Q += made * a.ld;
    a.S += made * Sr;
    a.clear.at = nullptr;
  }
  return launch_status("quantize_rows");
}
int launch_quantize_rows(const QuantRowsArgs& a, int dtype, hipStream_t st) {
  if (dtype == SMOE_BF16) return quantize_rows<bf16_t>(a, st);
  if (dtype == SMOE_F16) return quantize_rows<f16_t>(a, st);
  return quantize_rows<float>(a, st);
}

// ---- weights ---------------------------------------------------------------------------------------------
// One workgroup per block of 128 x 128, which it holds in registers (rows 16 p + (t >> 4), eight columns a thread); the transposed
// bytes go through LDS.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quantize_weights_kernel(QuantWeightsArgs a, int nb, int kb) {
  __shared__ float tops[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[QB][QB + 16];            // [column][row]
  const unsigned b = blockIdx.x;
  const unsigned kblk = b % (unsigned)kb, rest = b / (unsigned)kb, nblk = rest % (unsigned)nb, e = rest / (unsigned)nb;
  const int t = threadIdx.x;
  const int64_t c = (int64_t)kblk * QB + (t & 15) * 8, Kp = padded_row(a.K), Np = padded_row(a.N);
  float v[8][8], top = 0.0f;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int64_t n = (int64_t)nblk * QB + p * 16 + (t >> 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
    if (n < a.N) load8<T, VEC>((const T*)a.W + (int64_t)e * a.swe + n * a.swn, c, a.K, v[p]);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[p][i]));
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
  if ((t & 63) == 0) tops[t >> 6] = top;
  __syncthreads();
  const int byte = scale_byte(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
  const float scale = scale_of(byte);
  if (t == 0) a.S[b] = (uint8_t)byte;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int r = p * 16 + (t >> 4);
    const int64_t n = (int64_t)nblk * QB + r;
    const i32x2 q = {to_e4m3x4(v[p][0], v[p][1], v[p][2], v[p][3], scale), to_e4m3x4(v[p][4], v[p][5], v[p][6], v[p][7], scale)};
    if (n < a.N && c < Kp) *(i32x2*)(a.Q + ((int64_t)e * a.N + n) * Kp + c) = q;
    if (a.QT) {
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[(t & 15) * 8 + i][r] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
    }
  }
  if (!a.QT) return;
  __syncthreads();
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int piece = p * 256 + t, col = piece >> 3;
    const int64_t k = (int64_t)kblk * QB + col, n = (int64_t)nblk * QB + (piece & 7) * 16;
    if (k < a.K && n < Np) *(q_i32x4*)(a.QT + ((int64_t)e * a.K + k) * Np + n) = *(const q_i32x4*)&tile[col][(piece & 7) * 16];
  }
}
template <typename T>
static int quantize_weights(const QuantWeightsArgs& a, hipStream_t st) {
  const int64_t nb = scale_blocks(a.N), kb = scale_blocks(a.K), total = a.E * nb * kb;
  if (total > 0x7fffffffLL) { set_error("quantize_weights: grid too large"); return SMOE_ERR_RANGE; }
  const bool vec = ((uintptr_t)a.W & 15) == 0 && (a.swn | a.swe) * (int64_t)sizeof(T) % 16 == 0 && a.K % 8 == 0;
  if (vec) quantize_weights_kernel<T, true><<<(unsigned)total, 256, 0, st>>>(a, (int)nb, (int)kb);
  else quantize_weights_kernel<T, false><<<(unsigned)total, 256, 0, st>>>(a, (int)nb, (int)kb);
  return launch_status("quantize_weights");
}
int launch_quantize_weights(const QuantWeightsArgs& a, int dtype, hipStream_t st) {
  if (dtype == SMOE_BF16) return quantize_weights<bf16_t>(a, st);
  if (dtype == SMOE_F16) return quantize_weights<f16_t>(a, st);
  return quantize_weights<float>(a, st);
}

// 16 values a thread: a 16-byte piece of a row, which lies in one block
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dequantize_kernel(DequantArgs a, unsigned pieces) {
  const int64_t u = blockIdx.x * (int64_t)256 + threadIdx.x, rows = (int64_t)a.E * a.N;
  if (u >= rows * pieces) return;
  const int64_t row = u / pieces, c = (u - row * pieces) * 16, e = row / a.N, n = row - e * a.N;
  const int64_t at = e * a.sse + n / a.tall * a.ssn + c / QB * a.ssk;
  const float s = a.s_f32 ? ((const float*)a.S)[at] : weight_scale(((const uint8_t*)a.S)[at]);
  const uint8_t* q = a.Q + e * a.sqe + n * a.sqn + c;
  T* y = (T*)a.Y + row * a.K;
  if (c + 16 <= a.K && ((uintptr_t)q & 15) == 0) {
    const q_i32x4 p = *(const q_i32x4*)q;
    float v[2][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
      from_e4m3x4(p[i], s, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i >> 1][(i & 1) * 4 + j] = f[j];
    }
    store8<T, VEC>(y, c, a.K, v[0]);
    store8<T, VEC>(y, c + 8, a.K, v[1]);
    return;
  }
  for (int i = 0; i < 16 && c + i < a.K; ++i) y[c + i] = from_f32<T>(__builtin_amdgcn_cvt_f32_fp8(q[i], 0) * s);
}
template <typename T>
static int dequantize(const DequantArgs& a, hipStream_t st) {
  const int64_t pieces = (a.K + 15) / 16, grid = ((int64_t)a.E * a.N * pieces + 255) / 256;
  if (grid > 0x7fffffffLL) { set_error("dequantize: grid too large"); return SMOE_ERR_RANGE; }
  const bool vec = ((uintptr_t)a.Y & 15) == 0 && a.K % 8 == 0;
  if (vec) dequantize_kernel<T, true><<<(unsigned)grid, 256, 0, st>>>(a, (unsigned)pieces);
  else dequantize_kernel<T, false><<<(unsigned)grid, 256, 0, st>>>(a, (unsigned)pieces);
  return launch_status("dequantize");
}
int launch_dequantize(const DequantArgs& a, int dtype, hipStream_t st) {
  if (dtype == SMOE_BF16) return dequantize<bf16_t>(a, st);
  if (dtype == SMOE_F16) return dequantize<f16_t>(a, st);
  return dequantize<float>(a, st);
}

// ---- gated unit ------------------------------------------------------------------------------------------
// TI: type of pre; TH: type of h, or void: 8 bits
template <typename TI, bool QUANT, bool VEC>
__global__ __launch_bounds__(256) void unit_fwd_kernel(UnitArgs a, int blocks) {
  const Unit u(a.rows, blocks);
  if (!u.there) return;
  const int64_t F = a.F, Fp = padded_row(F);
  const TI* pre = (const TI*)a.pre + u.row * a.spm;
  float lin[8], gat[8], h[8];
  load8<TI, VEC>(pre + (a.act & 1 ? F : 0), u.c, F, lin);
  load8<TI, VEC>(pre + (a.act & 1 ? 0 : F), u.c, F, gat);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = glu_h(a.act, gat[i], lin[i]);
  if constexpr (QUANT) store_block(a.H8 + u.row * block_row(F), a.HS + u.row * scale_row(F) + u.block, u.c, block_row(F), h);
  else store8<TI, VEC>((TI*)a.h + u.row * F, u.c, F, h);
  if (a.P8) {
    store_block(a.P8 + u.row * 2 * Fp, a.PS + u.row * 2 * blocks + u.block, u.c, Fp, lin);
    store_block(a.P8 + (u.row * 2 + 1) * Fp, a.PS + (u.row * 2 + 1) * blocks + u.block, u.c, Fp, gat);
  }
}
template <typename TI, bool QUANT>
static int unit_fwd(UnitArgs a, hipStream_t st) {
  const int64_t blocks = scale_blocks(a.F), Fp = padded_row(a.F);
  const bool vec = (((uintptr_t)a.pre | (QUANT ? 0 : (uintptr_t)a.h)) & 15) == 0 && a.spm * (int64_t)sizeof(TI) % 16 == 0 && a.F % 8 == 0;
  int64_t left = a.rows;
  while (left > 0) {
    a.rows = rows_per_launch(left, blocks);
    const dim3 grid((unsigned)((a.rows * blocks + 15) / 16));
    if (vec) unit_fwd_kernel<TI, QUANT, true><<<grid, 256, 0, st>>>(a, (int)blocks);
    else unit_fwd_kernel<TI, QUANT, false><<<grid, 256, 0, st>>>(a, (int)blocks);
    left -= a.rows;
    a.pre = (const TI*)a.pre + a.rows * a.spm;
    if (a.h) a.h = (TI*)a.h + a.rows * a.F;
    if (a.H8) a.H8 += a.rows * block_row(a.F), a.HS += a.rows * scale_row(a.F);
    if (a.P8) a.P8 += a.rows * 2 * Fp, a.PS += a.rows * 2 * blocks;
  }
  return launch_status("unit_fwd");
}
int launch_unit_fwd(const UnitArgs& a, int dtype, hipStream_t st) {
  if (a.H8) return unit_fwd<float, true>(a, st);
  if (dtype == SMOE_BF16) return unit_fwd<bf16_t, false>(a, st);
  if (dtype == SMOE_F16) return unit_fwd<f16_t, false>(a, st);
  return unit_fwd<float, false>(a, st);
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void unit_bwd_kernel(UnitBackArgs a, int blocks) {
  const Unit u(a.rows, blocks);
  if (!u.there) return;
  const int64_t F = a.F, Fp = padded_row(F);
  float lin[8], gat[8], dh[8];
  load_block(a.P8 + u.row * 2 * Fp, a.PS + u.row * 2 * blocks + u.block, u.c, Fp, lin);
  load_block(a.P8 + (u.row * 2 + 1) * Fp, a.PS + (u.row * 2 + 1) * blocks + u.block, u.c, Fp, gat);
  load8<T, VEC>((const T*)a.dh + u.row * a.sdh, u.c, F, dh);
  if (a.h) {
    float h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = glu_h(a.act, gat[i], lin[i]);
    store8<T, VEC>((T*)a.h + u.row * F, u.c, F, h);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float dl, dg;
    glu_grad(a.act, dh[i], gat[i], lin[i], dl, dg);
    lin[i] = dl, gat[i] = dg;
  }
  T* out = (T*)a.dpre + u.row * 2 * F;
  store8<T, VEC>(out + (a.act & 1 ? F : 0), u.c, F, lin);
  store8<T, VEC>(out + (a.act & 1 ? 0 : F), u.c, F, gat);
}
// In 8 bits the blocks run along all 2F columns, the contraction of the product that reads them: with F no multiple of 128 one of them
// holds columns of both halves, and its values are read one by one.
// A block of the first half and the one of the second half that reads the same columns lie side by side in a workgroup: in the order of the columns
// both would come from memory twice (8204 rows of 2 x 2880: 59 us, 55 so; its arithmetic bounds it, 47 million exponentials).
__global__ __launch_bounds__(256) void unit_bwd_8bit_kernel(UnitBackArgs a, int blocks) {
  Unit u(a.rows, blocks);
  if (!u.there) return;
  u.block = u.block & 1 ? (blocks + 1) / 2 + u.block / 2 : u.block / 2;
  u.c = (int64_t)u.block * QB + (threadIdx.x & 15) * 8;
  const int64_t F = a.F, Fp = padded_row(F), D = 2 * F, Dp = block_row(D);
  const int hb = (int)scale_blocks(F);
  const uint8_t* p8 = a.P8 + u.row * 2 * Fp;
  const uint8_t* ps = a.PS + u.row * 2 * hb;
  const float* dh = (const float*)a.dh + u.row * a.sdh;
  float v[8];
  const bool first = u.c < F;
  const int64_t j0 = first ? u.c : u.c - F;
  const bool gate_half = first == ((a.act & 1) != 0);
  if ((F & 7) == 0 && u.c < D) {                                // eight columns of one half, within one block of it
    float lin[8], gat[8], d[8];
    load_block(p8, ps + j0 / QB, j0, Fp, lin);
    load_block(p8 + Fp, ps + hb + j0 / QB, j0, Fp, gat);
    load8<float, true>(dh, j0, F, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float dl, dg;
      glu_grad(a.act, d[i], gat[i], lin[i], dl, dg);
      v[i] = gate_half ? dg : dl;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t c = u.c + i;
      v[i] = 0.0f;
      if (c < D) {
        const bool head = c < F;
        const int64_t j = head ? c : c - F;
        const float lin = __builtin_amdgcn_cvt_f32_fp8(p8[j], 0) * scale_of(ps[j / QB]);
        const float gat = __builtin_amdgcn_cvt_f32_fp8(p8[Fp + j], 0) * scale_of(ps[hb + j / QB]);
        float dl, dg;
        glu_grad(a.act, dh[j], gat, lin, dl, dg);
        v[i] = head == ((a.act & 1) != 0) ? dg : dl;
      }
    }
  }
  store_block(a.D8 + u.row * Dp, a.DS + u.row * scale_row(D) + u.block, u.c, Dp, v);
}
template <typename T>
static int unit_bwd(UnitBackArgs a, hipStream_t st) {
  const bool quant = a.D8 != nullptr;
  const int64_t F = a.F, Fp = padded_row(F), hb = scale_blocks(F), blocks = quant ? scale_blocks(2 * F) : hb;
  const bool vec = (((uintptr_t)a.dh | (uintptr_t)a.dpre | (uintptr_t)a.h) & 15) == 0 && a.sdh * (int64_t)sizeof(T) % 16 == 0 && F % 8 == 0;
  int64_t left = a.rows;
  while (left > 0) {
    a.rows = rows_per_launch(left, blocks);
    const dim3 grid((unsigned)((a.rows * blocks + 15) / 16));
    if (quant) unit_bwd_8bit_kernel<<<grid, 256, 0, st>>>(a, (int)blocks);
    else if (vec) unit_bwd_kernel<T, true><<<grid, 256, 0, st>>>(a, (int)blocks);
    else unit_bwd_kernel<T, false><<<grid, 256, 0, st>>>(a, (int)blocks);
    left -= a.rows;
    a.P8 += a.rows * 2 * Fp, a.PS += a.rows * 2 * hb;
    a.dh = (const T*)a.dh + a.rows * a.sdh;
    if (quant) a.D8 += a.rows * block_row(2 * F), a.DS += a.rows * scale_row(2 * F);
    else a.dpre = (T*)a.dpre + a.rows * 2 * F;
    if (a.h) a.h = (T*)a.h + a.rows * F;
  }
  return launch_status("unit_bwd");
}
int launch_unit_bwd(const UnitBackArgs& a, int dtype, hipStream_t st) {
  if (a.D8) return unit_bwd<float>(a, st);
  if (dtype == SMOE_BF16) return unit_bwd<bf16_t>(a, st);
  if (dtype == SMOE_F16) return unit_bwd<f16_t>(a, st);
  return unit_bwd<float>(a, st);
}

}  // namespace smoe
