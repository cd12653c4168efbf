// scatter2scatter on 8-bit operands (eight_bit.hpp): Y[dst(n)] = X[src(n)] W[e(n)]^T over rows sorted by expert, in tiles of
// 128 rows x 256 columns that never straddle two experts.
//
// A slice of the contraction is 128 values, 128 bytes a row, one block of both operands' scales and one v_mfma_scale_f32_16x16x128:
// byte for byte the slice of 64 16-bit values of gemm_mfma.hpp, whose operand tiles (DirectOp), tile lookup and order are used as they
// are (offsets there count pairs of bytes).  The instruction multiplies by a power of two per operand row: the rows' scales always,
// the weights' where they are held in 8 bits.  Scales in float32 are applied to each slice's sums: four multiply-adds per
// instruction of 32 cycles, in the vector unit beside the matrix cores.
// Two workgroups of four waves per CU, as in mainloop_pair: what one does outside its loop the other's products hide.  The row
// operand has two stages of 16 KB, the column operand one of 32 KB, whose fragments of a slice are read into registers ahead of the
// products, so that the next slice's pieces can be on their way into it meanwhile.
#include "gemm_mfma.hpp"
#include "eight_bit.hpp"

namespace smoe {

typedef Tile<128, 256, 1, 4, 2, false, 2, true> Tile8;
typedef DirectOp<Tile8::BM, Tile8::NT> Rows8;
typedef DirectOp<Tile8::BN, Tile8::NT> Cols8;
static constexpr int LDS8_B = 2 * Rows8::LDS_BYTES, LDS8 = LDS8_B + Cols8::LDS_BYTES;

__device__ __forceinline__ f32x4 mfma8(i32x8 w, i32x8 x, f32x4 c, int w_scale, int x_scale) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, w_scale, 0, x_scale);
}
template <class Op>
__device__ __forceinline__ i32x8 fragment8(const char* tile, int base) {
  const i32x4 a = Op::frag(tile, base, 0), b = Op::frag(tile, base, 1);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// What a wave multiplies a slice's products with: the weights' scales of its columns, in two halves of 32 (one and the same where the tile's
// columns are neighbours)
template <int SC>
struct WeightScales {
  typedef typename std::conditional<SC == SCALES_BYTES, int, float>::type V;
  const char* at[2];
  int64_t step;
  bool f32;
  __device__ __forceinline__ void load(int kt, V (&v)[2]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* p = at[h] + kt * step;
      if constexpr (SC == SCALES_BYTES) v[h] = *(const uint8_t*)p;
      else if constexpr (SC == SCALES_FLOAT) v[h] = *(const float*)p;
      else v[h] = f32 ? *(const float*)p : scale_of(*(const uint8_t*)p);
    }
  }
};

// sx: this thread's (t < 128) dwords of its row's scales; s_scale: [2][128] dwords of LDS, four slices each
template <int SC>
__device__ __forceinline__ void mainloop_8bit(Rows8& A, Cols8& B, const WeightScales<SC>& W, const uint8_t* sx, int K, char* lds,
                                              unsigned* s_scale, Block (&acc)[Tile8::FM][Tile8::FN]) {
  typedef Tile8 TL;
  typedef typename WeightScales<SC>::V V;
  constexpr int LOADS = Rows8::R + Cols8::R, PER_STEP = LOADS / 3;
  static_assert(LOADS % 3 == 0, "the loads of the next slice go with three quarters of a slice's products");
  const int wave = threadIdx.x >> 6, l = lane_id(), t = threadIdx.x;
  const int klen = K / 2, nfull = K / 128, nk = (K + 127) / 128;       // (pieces are counted in pairs of bytes)
  const bool tail = nk > nfull;
  const unsigned lds_u = lds_address(lds);
  unsigned fetched = 0;
  V ws[2];
  W.load(0, ws);
  if (t < TL::BM) s_scale[t] = *(const unsigned*)sx;
#pragma unroll
  for (int j = 0; j < Cols8::R; ++j) {
    if (nfull > 0) B.issue_one(lds_u + LDS8_B, 0, j);
    else B.issue_tail_one(lds_u + LDS8_B, 0, klen, j);
  }
#pragma unroll
  for (int j = 0; j < Rows8::R; ++j) {
    if (nfull > 0) A.issue_one(lds_u, 0, j);
    else A.issue_tail_one(lds_u, 0, klen, j);
  }
  unsigned xs[2 * TL::FM];
  // MORE: 0 the last slice, 1 a whole one follows, 2 a partial one
  auto slice = [&](int kt, auto more) {
    constexpr int MORE = decltype(more)::value;
    const unsigned par = (unsigned)(kt & 1) * Rows8::LDS_BYTES;
    char* ta = lds + par;
    char* tb = lds + LDS8_B;
    const unsigned na = lds_u + (Rows8::LDS_BYTES - par);
    // this thread's pieces of slice kt have landed, everyone's have, and everyone is done with slice kt - 1
    if (MORE == 0 && tail) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      A.zero_tail(ta, kt * 64, klen);
      B.zero_tail(tb, kt * 64, klen);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // (taken here, where nothing is on its way: a wait for them further down would be one for the next slice's pieces)
    asm volatile("" : "+v"(ws[0]), "+v"(ws[1]), "+v"(fetched));
    __builtin_amdgcn_sched_barrier(0);
    if ((kt & 3) == 0) {
#pragma unroll
      for (int i = 0; i < 2 * TL::FM; ++i) xs[i] = s_scale[((kt >> 2) & 1) * TL::BM + i * 16 + (l & 15)];
    }
    if ((kt & 3) == 3 && t < TL::BM) s_scale[(((kt >> 2) + 1) & 1) * TL::BM + t] = fetched;
    i32x8 fa[2][2], fb[2 * TL::FN];
#pragma unroll
    for (int j = 0; j < 2 * TL::FN; ++j) fb[j] = fragment8<Cols8>(tb, wave * TL::WTN + j * 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) fa[0][i] = fragment8<Rows8>(ta, i * 16);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // everyone has the column operand's fragments
    __builtin_amdgcn_sched_barrier(0);
    V now[2] = {ws[0], ws[1]};
    if constexpr (MORE != 0) {
      W.load(kt + 1, ws);
      if ((kt & 3) == 1 && kt + 3 < nk && t < TL::BM) fetched = *(const unsigned*)(sx + (kt + 3));
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < TL::FM; ++s) {
      const int c = s & 1, n = c ^ 1;
      if constexpr (MORE != 0) {
#pragma unroll
        for (int q = s * PER_STEP; q < (s + 1) * PER_STEP && q < LOADS; ++q) {
          if (q < Cols8::R) {
            if constexpr (MORE == 1) B.issue_one(lds_u + LDS8_B, (kt + 1) * 64, q);
            else B.issue_tail_one(lds_u + LDS8_B, (kt + 1) * 64, klen, q);
          } else {
            if constexpr (MORE == 1) A.issue_one(na, (kt + 1) * 64, q - Cols8::R);
            else A.issue_tail_one(na, (kt + 1) * 64, klen, q - Cols8::R);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (SC != SCALES_EXACT && s + 1 < TL::FM) {
#pragma unroll
        for (int i = 0; i < 2; ++i) fa[n][i] = fragment8<Rows8>(ta, (2 * (s + 1) + i) * 16);
      }
      if constexpr (SC == SCALES_EXACT) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          bf16x8_8b va[4];
          to_bf16x32(s == 0 ? fa[0][i] : fragment8<Rows8>(ta, (2 * s + i) * 16), va);
          const float fx = scale_of((int)(xs[2 * s + i] & 255u));
#pragma unroll
          for (int j = 0; j < 2 * TL::FN; ++j) {
            bf16x8_8b vb[4];
            to_bf16x32(fb[j], vb);
            f32x4& d = acc[s][j >> 1].q[2 * i + (j & 1)];
            f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < 4; ++u) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[u], va[u], p, 0, 0, 0);
            const float f = now[j >> 1] * fx;
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = fmaf(p[e], f, d[e]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2 * TL::FN; ++j) {
            f32x4& d = acc[s][j >> 1].q[2 * i + (j & 1)];
            const int x = (int)xs[2 * s + i];
            if constexpr (SC == SCALES_FLOAT) {
              const f32x4 p = mfma8(fb[j], fa[c][i], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 127, x);
#pragma unroll
              for (int e = 0; e < 4; ++e) d[e] = fmaf(p[e], now[j >> 1], d[e]);
            } else {
              d = mfma8(fb[j], fa[c][i], d, now[j >> 1], x);
            }
          }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) xs[2 * s + i] >>= 8;
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  for (int kt = 0; kt + 1 < nfull; ++kt) slice(kt, std::integral_constant<int, 1>());
  if (tail && nfull > 0) slice(nfull - 1, std::integral_constant<int, 2>());
  slice(nk - 1, std::integral_constant<int, 0>());
}

__device__ __forceinline__ float bias_value(const void* b, int64_t at, int dtype) {
  if (dtype == SMOE_BF16) return to_f32(((const bf16_t*)b)[at]);
  if (dtype == SMOE_F16) return to_f32(((const f16_t*)b)[at]);
  return ((const float*)b)[at];
}

// (float32 rows: the operands as bfloat16 take the registers of a second workgroup)
template <typename TO, int SC>
__global__ __launch_bounds__(Tile8::NT, SC == SCALES_EXACT ? 1 : 2) void product_8bit_kernel(Product8Args a, int bias_dtype, Raster rast) {
  typedef Tile8 TL;
  __shared__ __attribute__((aligned(16))) char lds[LDS8];
  __shared__ unsigned s_scale[2 * TL::BM];
  __shared__ int64_t s_dst[TL::BM];
  __shared__ int s_src[TL::BM];
  int m_tile, n_tile, m_loc, n_loc, e, row0, rows;
  if (!rast.map<2 * Raster::SN>(blockIdx.x, m_tile, n_tile, m_loc, n_loc)) return;
  if (!find_tile<TL::BM>(a.off, a.E, m_tile, e, row0, rows)) return;
  const int n0 = n_tile * TL::BN, t = threadIdx.x;
  const uint8_t* sx = nullptr;
  if (t < TL::BM) {
    const int row = row0 + (t < rows ? t : rows - 1);                  // rows behind the last one repeat it
    int slot = 0;
    if (!a.x_grouped || !a.y_grouped) slot = (int)a.idx[row];
    const int src = a.x_grouped ? row : (int)((unsigned)slot / (unsigned)a.fan);
    s_src[t] = src;
    s_dst[t] = t < rows ? (int64_t)(a.y_grouped ? row : slot) * a.sym : -1;
    sx = a.XS + src * scale_row(a.K);
  }
  __syncthreads();
  Rows8 A;
  A.rot = (n_loc * Rows8::R / (2 * Raster::SN)) % Rows8::R;
  const int src0 = a.x_grouped ? row0 : 0;
  const int64_t K = a.K;
  A.init((const char*)a.X + src0 * K, [&](int row) { return (int64_t)(s_src[row] - src0) * K; });
  Cols8 B;
  B.rot = (m_loc * Cols8::R / Raster::SM) % Cols8::R;
  const int64_t swn = a.swn;
  const int last = a.N - 1 - n0;
  B.init((const char*)a.W + e * a.swe + n0 * swn, [&](int row) { return (int64_t)min(row, last) * swn; });
  WeightScales<SC> W;
  const int WSB = SC == SCALES_BYTES ? 1 : SC == SCALES_FLOAT || a.ws_f32 ? 4 : 1;
  const int nb = min(n0 + (int)wave_uniform_id() * TL::WTN, a.N - 1) / QB;
  W.at[0] = W.at[1] = (const char*)a.WS + (e * a.sse + nb * a.ssn) * WSB;
  W.step = a.ssk * WSB;
  W.f32 = a.ws_f32 != 0;
  Block acc[TL::FM][TL::FN];
#pragma unroll
  for (int i = 0; i < TL::FM; ++i)
#pragma unroll
    for (int j = 0; j < TL::FN; ++j) acc[i][j].clear();
  mainloop_8bit<SC>(A, B, W, sx, a.K, lds, s_scale, acc);
  __syncthreads();
  const int wave = t >> 6, l = lane_id();
  if (a.b) {
#pragma unroll
    for (int j = 0; j < 2 * TL::FN; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = n0 + wave * TL::WTN + j * 16 + 4 * (l >> 4) + c;
        const float b = n < a.N ? bias_value(a.b, e * a.sbe + n * a.sbn, bias_dtype) : 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * TL::FM; ++i) acc[i >> 1][j >> 1].q[2 * (i & 1) + (j & 1)][c] += b;
      }
  }
  TO* Y = (TO*)a.Y;
  if constexpr (sizeof(TO) == 2) {
    if (((uintptr_t)Y & 15) == 0 && ((a.sym | a.N) & 7) == 0) epilogue_staged<TO, TL>(acc, Y, s_dst, n0, a.N, nullptr, 0, lds);
    else epilogue<TO, TL>(acc, Y, s_dst, n0, a.N, nullptr, 0);
  } else {
    // 16 rows of 64 bytes per wave and store: whole sectors as they lie in the registers
    const bool whole = ((uintptr_t)Y & 15) == 0 && ((a.sym | a.N) & 3) == 0;
    auto walk = [&](auto put) {
#pragma unroll
      for (int i = 0; i < 2 * TL::FM; ++i) {
        const int64_t d = s_dst[i * 16 + (l & 15)];
        if (d >= 0) {
#pragma unroll
          for (int j = 0; j < 2 * TL::FN; ++j) put(d, n0 + wave * TL::WTN + j * 16 + 4 * (l >> 4), acc[i >> 1][j >> 1].q[2 * (i & 1) + (j & 1)]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (whole) {
      walk([&](int64_t d, int n, const f32x4& v) {
        if (n < a.N) *(f32x4*)(Y + d + n) = v;
      });
    } else {
      walk([&](int64_t d, int n, const f32x4& v) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n + c < a.N) Y[d + n + c] = v[c];
      });
    }
  }
}

template <typename TO, bool EXACT>
static int launch_product(const Product8Args& a, int bias_dtype, hipStream_t st) {
  const int64_t m_tiles = max_tiles(a.L, a.E, Tile8::BM);
  const int n_tiles = (a.N + Tile8::BN - 1) / Tile8::BN;
  const Raster r = a.L < (int64_t)STRIPE_BELOW * a.E ? make_striped(m_tiles, n_tiles, GM_RING)
                                                     : make_raster(m_tiles, n_tiles, GM_S2S, 2 * Raster::SN);
  if (r.grid() > 0x7fffffffLL) { set_error("product_8bit: grid too large"); return SMOE_ERR_RANGE; }
  const unsigned grid = (unsigned)r.grid();
  if constexpr (EXACT) product_8bit_kernel<TO, SCALES_EXACT><<<grid, Tile8::NT, 0, st>>>(a, bias_dtype, r);
  else if (a.ws_f32) product_8bit_kernel<TO, SCALES_FLOAT><<<grid, Tile8::NT, 0, st>>>(a, bias_dtype, r);
  else product_8bit_kernel<TO, SCALES_BYTES><<<grid, Tile8::NT, 0, st>>>(a, bias_dtype, r);
  return launch_status("product_8bit");
}

int launch_product_8bit(const Product8Args& a, int row_dtype, int out_dtype, hipStream_t st) {
  if (row_dtype == SMOE_F32) return launch_product<float, true>(a, row_dtype, st);
  if (out_dtype == SMOE_F32) return launch_product<float, false>(a, row_dtype, st);
  if (out_dtype == SMOE_BF16) return launch_product<bf16_t, false>(a, row_dtype, st);
  return launch_product<f16_t, false>(a, row_dtype, st);
}

}  // namespace smoe
