// scatter2scatter on 8-bit weights for a few rows per expert: a stream over the weights.
//
// A workgroup has CF groups of 16 output columns and up to 16 MF rows of one expert; its eight waves share the contraction, each a run of
// slices of 128, and add their sums up through LDS, in the order of the waves.  A wave's fragments go from memory to registers, two
// slices of them on their way (16 KB per wave at CF = 4), since nobody else reads them.  Products are of bfloat16, which holds e4m3 exactly,
// with both scales on every slice's sums (Scaling8): the matrix cores have time for it, a slice's 2 KB of weights take about 900 cycles
// to come from memory and 64 MF + 64 to multiply.
// Rows come as they are (float32, bfloat16, float16) and are taken to 8 bits on the way, a block's largest of four lanes, or from
// a workspace where there are so many that each column group would do it again.
#include "eight_bit.hpp"

namespace smoe {

typedef int w_i32x4 __attribute__((ext_vector_type(4)));
typedef float w_f32x4 __attribute__((ext_vector_type(4)));
static constexpr int FEW_NW = 8, FEW_NT = FEW_NW * 64;

// What lane l has of a row's slice: its 16 values from 16 (l / 16) on, and the 16 that are 64 further
template <typename T>
__device__ __forceinline__ void load_values(const T* __restrict__ row, int k0, int K, bool vec, float (&v)[32]) {
  const int g = (lane_id() >> 4) << 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = k0 + h * 64 + g;
    if (vec && c + 16 <= K) {
      constexpr int PER = 16 / (int)sizeof(T);
      T t[16];
#pragma unroll
      for (int p = 0; p < 16 / PER; ++p) __builtin_memcpy(t + p * PER, (const char*)__builtin_assume_aligned((const char*)(row + c) + p * 16, 16), 16);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[h * 16 + i] = to_f32(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[h * 16 + i] = c + i < K ? to_f32(row[c + i]) : 0.0f;
    }
  }
}

template <typename TX, int MF, int CF, int EPI>
__global__ __launch_bounds__(FEW_NT, 2) void few_rows_8bit_kernel(Few8Args a, int dtype, int per) {
  constexpr bool FROM_8BIT = sizeof(TX) == 1;
  constexpr int ROWS = 16 * MF;
  __shared__ __attribute__((aligned(16))) w_f32x4 sums[FEW_NW][MF * CF][64];
  __shared__ int s_src[64], s_dst[64];
  const int t = threadIdx.x, l = lane_id(), wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // ---- whose rows
  int e, rows, row0 = 0;
  if (a.ids) {
    // up to 64 slots: one per lane, the blockIdx.y-th of the experts that they name
    const int64_t id = l < a.L ? a.ids[l] : -1;
    bool again = id < 0 || id >= a.E;
    const int ide = again ? -1 : (int)id;
    for (int j = 0; j + 1 < a.L; ++j) again = again || (l > j && ide == __builtin_amdgcn_readlane(ide, j));
    const unsigned long long firsts = __ballot(!again);
    if ((int)blockIdx.y >= __popcll(firsts)) return;
    const unsigned long long below = (1ull << l) - 1;
    const unsigned long long hit = __ballot(!again && __popcll(firsts & below) == (int)blockIdx.y);
    e = __builtin_amdgcn_readlane(ide, __ffsll((long long)hit) - 1);
    const unsigned long long mine = __ballot(ide == e);
    rows = __popcll(mine);
    if (wave == 0 && ide == e) {
      const int m = __popcll(mine & below);
      s_src[m] = l / a.fan;
      s_dst[m] = l;
    }
  } else {
    if (!find_tile<ROWS>(a.off, a.E, blockIdx.y, e, row0, rows)) return;
    if (t < rows) {
      const int r = row0 + t;
      const int slot = a.x_grouped && a.y_grouped ? 0 : (int)a.idx[r];
      s_src[t] = a.x_grouped ? r : (int)((unsigned)slot / (unsigned)a.fan);
      s_dst[t] = a.y_grouped ? r : slot;
    }
  }
  __syncthreads();
  // ---- this wave's weight rows and scales
  const int F = a.N / 2;
  constexpr int HALF = EPI == EPI_UNIT ? CF / 2 : CF;              // groups of neighbouring columns
  const int n0 = blockIdx.x * (HALF * 16);
  const int64_t Kp = padded_row(a.K);
  const char* W = (const char*)a.W + e * a.swe;
  const char* wrow[CF];
  const char* wscale[CF];
  const int WSB = a.ws_f32 ? 4 : 1;
#pragma unroll
  for (int j = 0; j < CF; ++j) {
    int n = min(n0 + (j % HALF) * 16 + (l & 15), (EPI == EPI_UNIT ? F : a.N) - 1);
    if (EPI == EPI_UNIT && j >= HALF) n += F;
    wrow[j] = W + n * Kp;
    wscale[j] = (const char*)a.WS + (e * a.sse + n / QB * a.ssn) * WSB;
  }
  const int nk = (int)scale_blocks(a.K), first = wave * per, last = min(first + per, nk);
  const int g16 = (l >> 4) << 4;
  // a slice's fragment: 16 bytes and those 64 further; pieces behind the row's end are the row's first, and zeros
  auto load_cols = [&](int kt, int j, i32x8& f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = kt * QB + h * 64 + g16;
      const bool there = c < Kp;
      const w_i32x4 v = __builtin_nontemporal_load((const w_i32x4*)(wrow[j] + (there ? c : 0)));
#pragma unroll
      for (int i = 0; i < 4; ++i) f[h * 4 + i] = there ? v[i] : 0;
    }
  };
  auto scale_at = [&](int kt, int j) {
    const char* p = wscale[j] + kt * a.ssk * WSB;
    return a.ws_f32 ? *(const float*)p : scale_of(*(const uint8_t*)p);
  };
  for (int base = 0; base < rows; base += ROWS) {                  // (by ids, an expert may have more rows than ROWS)
    const int here = min(ROWS, rows - base);
    w_f32x4 acc[MF][CF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < CF; ++j) acc[i][j] = w_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const TX* xrow[MF];
    const uint8_t* xs[MF];
    bool have[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int m = i * 16 + (l & 15);
      have[i] = m < here;
      const int64_t src = s_src[base + (have[i] ? m : 0)];
      xrow[i] = (const TX*)a.X + src * a.sxm;
      xs[i] = FROM_8BIT ? a.XS + src * scale_row(a.K) : nullptr;
    }
    const bool vec = a.x_vec != 0;
    i32x8 w[2][CF];
    float ws[2][CF];
    auto fetch = [&](int kt, int p) {
#pragma unroll
      for (int j = 0; j < CF; ++j) load_cols(kt, j, w[p][j]);
#pragma unroll
      for (int j = 0; j < CF; ++j) ws[p][j] = scale_at(kt, j);
    };
    auto multiply = [&](int kt, int p) {
      bf16x8_8b x[MF][4];
      float fx[MF];
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        i32x8 q = {0, 0, 0, 0, 0, 0, 0, 0};
        fx[i] = 0.0f;
        if constexpr (FROM_8BIT) {
          // (the workspace's rows are whole slices long)
          if (have[i]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const w_i32x4 v = *(const w_i32x4*)(xrow[i] + kt * QB + h * 64 + g16);
#pragma unroll
              for (int c = 0; c < 4; ++c) q[h * 4 + c] = v[c];
            }
            fx[i] = scale_of(xs[i][kt]);
          }
        } else {
          float v[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = 0.0f;
          if (have[i]) load_values<TX>(xrow[i], kt * QB, a.K, vec, v);
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < 32; ++c) top = fmaxf(top, fabsf(v[c]));
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const int byte = scale_byte(top);
          const float inv = inverse_scale(byte);
#pragma unroll
          for (int c = 0; c < 8; ++c) q[c] = to_e4m3x4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3], inv);
          fx[i] = scale_of(byte);
        }
        to_bf16x32(q, x[i]);
      }
#pragma unroll
      for (int j = 0; j < CF; ++j) {
        bf16x8_8b wv[4];
        to_bf16x32(w[p][j], wv);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          w_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int u = 0; u < 4; ++u) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i][u], wv[u], s, 0, 0, 0);
          // (rows down the lanes' four values, columns across them: a column's scale is the lane's own)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = fmaf(s[c] * ws[p][j], __shfl(fx[i], 4 * (l >> 4) + c), acc[i][j][c]);
        }
      }
    };
    if (first < last) fetch(first, 0);
    for (int kt = first; kt < last; kt += 2) {
      if (kt + 1 < last) fetch(kt + 1, 1);
      multiply(kt, 0);
      if (kt + 2 < last) fetch(kt + 2, 0);
      if (kt + 1 < last) multiply(kt + 1, 1);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < CF; ++j) sums[wave][i * CF + j][l] = acc[i][j];
    __syncthreads();
    // ---- the waves' sums, one value per thread and step: row 16 i + 4 (lane / 16) + c, column 16 j + lane % 16
    constexpr int VALUES = ROWS * HALF * 16;
    for (int v = t; v < VALUES; v += FEW_NT) {
      const int m = v / (HALF * 16), n = v % (HALF * 16), i = m >> 4, j = n >> 4;
      const int lane = ((m >> 2) & 3) * 16 + (n & 15), c = m & 3;
      const int col = n0 + n;
      if (m >= here || col >= (EPI == EPI_UNIT ? F : a.N)) continue;
      auto total = [&](int jj) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < FEW_NW; ++k) s += ((const float*)&sums[k][i * CF + jj][lane])[c];
        return s;
      };
      auto biased = [&](float s, int at) { return a.b ? s + bias_value(a.b, e * a.sbe + at * a.sbn, dtype) : s; };
      const float one = biased(total(j), col);
      const int64_t dst = s_dst[base + m];
      if constexpr (EPI == EPI_UNIT) {
        const float two = biased(total(j + HALF), F + col);
        ((float*)a.Y)[dst * a.sym + col] = a.act & 1 ? glu_h(a.act, one, two) : glu_h(a.act, two, one);
      } else {
        const int64_t at = dst * a.sym + col;
        if (a.out_dtype == SMOE_F32) ((float*)a.Y)[at] = one;
        else if (a.out_dtype == SMOE_BF16) ((bf16_t*)a.Y)[at] = from_f32<bf16_t>(one);
        else ((f16_t*)a.Y)[at] = from_f32<f16_t>(one);
      }
    }
    __syncthreads();
  }
}

// out[t] = sum_j gates[t, j] rows[t k + j] of float32 rows, slots whose id lies outside [0, E) left out
template <typename T>
__global__ __launch_bounds__(256) void few_combine_kernel(const float* rows, const T* gates, const int64_t* ids, T* out, int T_, int k, int d, int E) {
  const int64_t v = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (v >= (int64_t)T_ * d) return;
  const int tok = (int)(v / d), c = (int)(v - (int64_t)tok * d);
  float s = 0.0f;
  for (int j = 0; j < k; ++j) {
    const int64_t id = ids[tok * k + j];
    if (id >= 0 && id < E) s = fmaf(to_f32(gates[tok * k + j]), rows[((int64_t)tok * k + j) * d + c], s);
  }
  out[v] = from_f32<T>(s);
}
int launch_few_combine(const float* rows, const void* gates, const int64_t* ids, void* out, int T, int k, int d, int E, int dtype, hipStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)T * d + 255) / 256);
  if (dtype == SMOE_BF16) few_combine_kernel<bf16_t><<<grid, 256, 0, st>>>(rows, (const bf16_t*)gates, ids, (bf16_t*)out, T, k, d, E);
  else if (dtype == SMOE_F16) few_combine_kernel<f16_t><<<grid, 256, 0, st>>>(rows, (const f16_t*)gates, ids, (f16_t*)out, T, k, d, E);
  else few_combine_kernel<float><<<grid, 256, 0, st>>>(rows, (const float*)gates, ids, (float*)out, T, k, d, E);
  return launch_status("few_combine");
}

template <typename TX, int MF, int CF, int EPI>
static int launch_few(const Few8Args& a, int dtype, hipStream_t st) {
  const int cols = EPI == EPI_UNIT ? a.N / 2 : a.N, group = (EPI == EPI_UNIT ? CF / 2 : CF) * 16;
  const int64_t segments = a.ids ? (a.L < a.E ? a.L : a.E) : max_tiles(a.L, a.E, 16 * MF);
  const int per = (int)((scale_blocks(a.K) + FEW_NW - 1) / FEW_NW);
  if (segments > 65535) { set_error("few_rows_8bit: too many rows"); return SMOE_ERR_RANGE; }
  few_rows_8bit_kernel<TX, MF, CF, EPI><<<dim3((cols + group - 1) / group, (unsigned)segments), FEW_NT, 0, st>>>(a, dtype, per);
  return launch_status("few_rows_8bit");
}
template <typename TX, int MF>
static int launch_few(const Few8Args& a, int dtype, int epilogue, hipStream_t st) {
  if (epilogue == EPI_UNIT) return launch_few<TX, MF, 4, EPI_UNIT>(a, dtype, st);
  return launch_few<TX, MF, 4, EPI_ROWS>(a, dtype, st);
}
int launch_few_rows_8bit(const Few8Args& a, int x_dtype, int dtype, int epilogue, hipStream_t st) {
  if (x_dtype == SMOE_BF16) return launch_few<bf16_t, 1>(a, dtype, epilogue, st);
  if (x_dtype == SMOE_F16) return launch_few<f16_t, 1>(a, dtype, epilogue, st);
  if (x_dtype == SMOE_F32) return launch_few<float, 1>(a, dtype, epilogue, st);
  return launch_few<uint8_t, 1>(a, dtype, epilogue, st);
}

}  // namespace smoe
