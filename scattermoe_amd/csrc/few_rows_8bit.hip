// scatter2scatter on 8-bit weights for a few rows per expert: a stream over the weights.
//
// Products are of bfloat16, which holds e4m3 times a power of two exactly (Scaling8): the matrix cores have time for it.  Scales of
// float32 multiply every slice's sums.
// 16 weight rows in an instruction would take 64 bytes each per load, half a line.  Instead its 16 rows are 8 rows in two parts of a
// slice of 128: a load takes whole lines of 8 weight rows, rows and weights alike, and of the 16 x 16 sums those count whose parts
// agree (few_rows.hpp).  A workgroup has GROUPS groups of 8 columns and 8 MF rows of one expert; its waves share the
// contraction, each a run of slices, two of them on their way from memory to registers, and add their sums up through LDS, in
// the order of the waves.
// Rows come as they are (float32, bfloat16, float16) and are taken to 8 bits on the way, a block's largest of eight lanes, or from
// a workspace where there are so many that each column group would do it again.
#include "eight_bit.hpp"

namespace smoe {

typedef int w_i32x4 __attribute__((ext_vector_type(4)));
typedef float w_f32x4 __attribute__((ext_vector_type(4)));
static constexpr int FEW_NW = 4, FEW_NT = FEW_NW * 64, GROUPS = 8;

// `bytes` of memory from one address for the wave on, with 32-bit offsets; behind them is nothing (zeros).  Plain pointers would have two
// registers per offset.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t from_here(const void* p, int64_t bytes) {
  const uint64_t v = (uint64_t)p;
  const uint64_t u = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
  const int range = __builtin_amdgcn_readfirstlane(bytes < 0xffffffffLL ? (int)(unsigned)bytes : -1);
  return __builtin_amdgcn_make_buffer_rsrc((void*)u, 0, range, 0x00020000);
}

template <typename TX, int MF, int EPI, bool SF>
__global__ __launch_bounds__(FEW_NT, 2) void few_rows_8bit_kernel(Few8Args a, int dtype, int per) {
  constexpr bool FROM_8BIT = sizeof(TX) == 1;
  constexpr int ROWS = 8 * MF;
  __shared__ __attribute__((aligned(16))) w_f32x4 sums[FEW_NW][MF * GROUPS][64];
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
  constexpr int HALF = EPI == EPI_UNIT ? GROUPS / 2 : GROUPS;      // groups of neighbouring columns
  const int n0 = blockIdx.x * (HALF * 8);
  const int Kp = (int)padded_row(a.K);
  // 32-bit offsets from the first row of either half: at most 64 rows of 2^21 bytes (product_checks in capi_8bit.hip refuses longer ones)
  e = __builtin_amdgcn_readfirstlane(e);
  const char* We = (const char*)a.W + e * a.swe;
  const int64_t n1 = n0 + (EPI == EPI_UNIT ? F : 0);
  const __amdgpu_buffer_rsrc_t W[2] = {from_here(We + (int64_t)n0 * Kp, (a.N - n0) * (int64_t)Kp), from_here(We + n1 * Kp, (a.N - n1) * Kp)};
  const int sub = (l & 15) >> 1, at = (l & 1) * 64 + (l >> 4) * 16;  // row of a group, and this lane's 16 values of a slice
  unsigned woff[HALF];
#pragma unroll
  for (int j = 0; j < HALF; ++j) woff[j] = (unsigned)(min(n0 + j * 8 + sub, (EPI == EPI_UNIT ? F : a.N) - 1) - n0) * (unsigned)Kp + at;
  // A slice's scales: one for these columns, which lie in one block of 128; in the unit one for the first half's and two for the second's, whose
  // columns start anywhere.  A byte comes as the dword it lies in and is taken out where it is used: loaded as a byte, it is converted
  // where it was loaded, and every slice waits for its own scales (8 experts, 4096 -> 14336, 32 rows: 90 us, 72 so).
  constexpr int SCALES = EPI == EPI_UNIT ? 3 : 1, WSB = SF ? 4 : 1;
  const char* ws_at = (const char*)a.WS + e * a.sse * WSB;
  const int ws_rem = (int)((uintptr_t)ws_at & 3);
  const __amdgpu_buffer_rsrc_t WS = from_here(ws_at - ws_rem, 0xffffffffLL);
  int sfirst[SCALES];
  sfirst[0] = ws_rem + (int)(n0 / QB * a.ssn) * WSB;
  if constexpr (EPI == EPI_UNIT) {
    const int b = (F + n0) / QB;
    sfirst[1] = ws_rem + (int)(b * a.ssn) * WSB;
    sfirst[2] = ws_rem + (int)(min(b + 1, (a.N - 1) / QB) * a.ssn) * WSB;
  }
  const int nk = (int)scale_blocks(a.K), first = wave * per, last = min(first + per, nk);
  auto load_scale = [&](int kt, int h) { return (int)__builtin_amdgcn_raw_buffer_load_b32(WS, 0, (sfirst[h] + (int)(kt * a.ssk) * WSB) & ~3, 0); };
  auto scale_in = [&](int v, int kt, int h) {
    return SF ? __builtin_bit_cast(float, v) : weight_scale((v >> (((sfirst[h] + (int)(kt * a.ssk)) & 3) * 8)) & 255);
  };
  for (int base = 0; base < rows; base += ROWS) {                  // (by ids, an expert may have more rows than ROWS)
    const int here = min(ROWS, rows - base);
    w_f32x4 acc[MF][GROUPS];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) acc[i][j] = w_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const TX* xrow[MF];
    const uint8_t* xs[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int m = i * 8 + sub;
      const int64_t src = s_src[base + (m < here ? m : 0)];          // (what a lane without a row multiplies is not looked at)
      xrow[i] = (const TX*)a.X + src * a.sxm + at;
      xs[i] = FROM_8BIT ? a.XS + src * scale_row(a.K) : nullptr;
    }
    // rows of a slice: 8 bits and their scale (the dword of four slices), or values on their way to that
    constexpr int XV = FROM_8BIT ? 4 : 4 * (int)sizeof(TX);
    typedef int XRegs __attribute__((ext_vector_type(XV)));
    w_i32x4 w[2][GROUPS];
    int ws[2][SCALES];
    XRegs xv[2][MF];
    int xb[2][MF];
    // slices that go two at a time: all of rows in 8 bits, which are whole slices long, whole ones of aligned float rows
    const int whole = FROM_8BIT ? max(first, last) : a.x_vec ? max(first, min(last, a.K / QB)) : first;
    auto fetch = [&](int slice, int p) {
      const int kt = min(slice, whole - 1);
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        w[p][j] = __builtin_bit_cast(w_i32x4, __builtin_amdgcn_raw_buffer_load_b128(W[j / HALF], (int)woff[j % HALF], kt * QB, 0));
      }
#pragma unroll
      for (int h = 0; h < SCALES; ++h) ws[p][h] = load_scale(kt, h);
#pragma unroll
      for (int i = 0; i < MF; ++i) {
#pragma unroll
        for (int u = 0; u < XV / 4; ++u) {
          const w_i32x4 v = *(const w_i32x4*)((const char*)(xrow[i] + kt * QB) + u * 16);
#pragma unroll
          for (int c = 0; c < 4; ++c) xv[p][i][u * 4 + c] = v[c];
        }
        if constexpr (FROM_8BIT) xb[p][i] = *(const int*)(xs[i] + (kt & ~3));
      }
    };
    auto fetch_some = [&](int kt) {                                // a slice that ends before its 128th value, or of other rows
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        w[0][j] = __builtin_bit_cast(w_i32x4, __builtin_amdgcn_raw_buffer_load_b128(W[j / HALF], (int)woff[j % HALF], kt * QB, 0));
      }
#pragma unroll
      for (int h = 0; h < SCALES; ++h) ws[0][h] = load_scale(kt, h);
      if constexpr (!FROM_8BIT) {
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          TX v[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) v[c] = kt * QB + at + c < a.K ? xrow[i][kt * QB + c] : from_f32<TX>(0.0f);
          __builtin_memcpy(&xv[0][i], v, sizeof(v));
        }
      }
    };
    auto multiply = [&](int slice, int p, int end) {
      bf16x8_8b x[MF][2];
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        w_i32x4 q;
        int byte;
        if constexpr (FROM_8BIT) asm volatile("" : "+v"(xb[p][i]));
        if constexpr (FROM_8BIT) {
          q = xv[p][i];
          byte = (xb[p][i] >> (8 * (min(slice, last - 1) & 3))) & 255;
        } else {
          TX v[16];
          __builtin_memcpy(v, &xv[p][i], sizeof(v));
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < 16; ++c) top = fmaxf(top, fabsf(to_f32(v[c])));
          top = fmaxf(top, __shfl_xor(top, 1));
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          byte = scale_byte(top);
          const float scale = scale_of(byte);
#pragma unroll
          for (int c = 0; c < 4; ++c) q[c] = to_e4m3x4(to_f32(v[4 * c]), to_f32(v[4 * c + 1]), to_f32(v[4 * c + 2]), to_f32(v[4 * c + 3]), scale);
        }
        to_bf16x16(q, scale_of(byte), x[i]);
      }
      // (behind a row's end is the next one's, which may be no number; behind the last slice, that one again)
      const bool there = slice < end && slice * QB + at < Kp;
      float scales[SCALES];
#pragma unroll
      for (int h = 0; h < SCALES; ++h) {
        asm volatile("" : "+v"(ws[p][h]));
        scales[h] = scale_in(ws[p][h], min(slice, end - 1), h);
      }
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        bf16x8_8b wv[2];
        w_i32x4 q = w[p][j];
        float scale = scales[0];
        if constexpr (EPI == EPI_UNIT) {
          if (j >= HALF) scale = (F + n0 + (j - HALF) * 8 + sub) / QB == (F + n0) / QB ? scales[1] : scales[2];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) q[c] = there ? q[c] : 0;
        to_bf16x16(q, SF ? 1.0f : scale, wv);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          w_f32x4 s = SF ? w_f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[i][j];
#pragma unroll
          for (int u = 0; u < 2; ++u) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i][u], wv[u], s, 0, 0, 0);
          // (columns across the lanes: a column's scale is the lane's own)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = SF ? fmaf(s[c], scale, acc[i][j][c]) : s[c];
        }
        if (j & 1) __builtin_amdgcn_sched_barrier(0);              // (all groups' conversions at once take too many registers)
      }
    };
    // (pairs of slices; one behind the last is the last again, its weights zeros: no branches, whose joins cost registers)
    if (first < whole) {
      // (in this order: the waits inside the loop are for what is on its way in either of its entries)
      fetch(first, 0);
      __builtin_amdgcn_sched_barrier(0);
      fetch(first + 1, 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma nounroll
      for (int kt = first; kt < whole; kt += 2) {
        multiply(kt, 0, whole);
        __builtin_amdgcn_sched_barrier(0);
        fetch(kt + 2, 0);
        __builtin_amdgcn_sched_barrier(0);
        multiply(kt + 1, 1, whole);
        __builtin_amdgcn_sched_barrier(0);
        fetch(kt + 3, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    for (int kt = whole; kt < last; ++kt) {
      fetch_some(kt);
      multiply(kt, 0, last);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) sums[wave][i * GROUPS + j][l] = acc[i][j];
    __syncthreads();
    // ---- the waves' sums, one value per thread and step: row r of a fragment in part p is instruction row 2 r + p, columns alike
    constexpr int VALUES = ROWS * HALF * 8;
    for (int v = t; v < VALUES; v += FEW_NT) {
      const int m = v / (HALF * 8), n = v % (HALF * 8), i = m >> 3, j = n >> 3;
      const int col = n0 + n;
      if (m >= here || col >= (EPI == EPI_UNIT ? F : a.N)) continue;
      auto total = [&](int jj) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < FEW_NW; ++k)
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const int row = 2 * (m & 7) + part;
            s += ((const float*)&sums[k][i * GROUPS + jj][(row >> 2) * 16 + 2 * (n & 7) + part])[row & 3];
          }
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

template <typename TX, int MF, int EPI>
static int launch_few(const Few8Args& a, int dtype, hipStream_t st) {
  const int cols = EPI == EPI_UNIT ? a.N / 2 : a.N, group = (EPI == EPI_UNIT ? GROUPS / 2 : GROUPS) * 8;
  const int64_t segments = a.ids ? (a.L < a.E ? a.L : a.E) : max_tiles(a.L, a.E, 8 * MF);
  const int per = (int)((scale_blocks(a.K) + FEW_NW - 1) / FEW_NW);
  if (segments > 65535) { set_error("few_rows_8bit: too many rows"); return SMOE_ERR_RANGE; }
  const dim3 grid((cols + group - 1) / group, (unsigned)segments);
  if (a.ws_f32) few_rows_8bit_kernel<TX, MF, EPI, true><<<grid, FEW_NT, 0, st>>>(a, dtype, per);
  else few_rows_8bit_kernel<TX, MF, EPI, false><<<grid, FEW_NT, 0, st>>>(a, dtype, per);
  return launch_status("few_rows_8bit");
}
template <typename TX, int MF>
static int launch_few(const Few8Args& a, int dtype, int epilogue, hipStream_t st) {
  return epilogue == EPI_UNIT ? launch_few<TX, MF, EPI_UNIT>(a, dtype, st) : launch_few<TX, MF, EPI_ROWS>(a, dtype, st);
}
int launch_few_rows_8bit(const Few8Args& a, int x_dtype, int dtype, int epilogue, hipStream_t st) {
  if (x_dtype == SMOE_BF16) return launch_few<bf16_t, 1>(a, dtype, epilogue, st);
  if (x_dtype == SMOE_F16) return launch_few<f16_t, 1>(a, dtype, epilogue, st);
  if (x_dtype == SMOE_F32) return launch_few<float, 1>(a, dtype, epilogue, st);
  // (8 or 16 rows of an expert at a time, us at 2, 4, 8 rows per expert, loads as 1 / rank^0.5: 8 experts, 4096 -> 14336 71, 77, 89 or 73, 74, 80;
  // 128 experts, 2048 -> 1536 63, 66, 80 or 69, 71, 77)
  return a.L <= 4 * (int64_t)a.E ? launch_few<uint8_t, 1>(a, dtype, epilogue, st) : launch_few<uint8_t, 2>(a, dtype, epilogue, st);
}

}  // namespace smoe
