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
// products, so that the next slice's pieces can be on their way into it meanwhile.  (The weights' fragments, which no other wave reads, straight
// from memory into registers, 16 rows of 64 bytes per load: 32768 x 4096 x 28672 3447 -> 4478 us.)
#include "gemm_mfma.hpp"
#include "eight_bit.hpp"

namespace smoe {

typedef Tile<128, 256, 1, 4, 2, false, 2, true> Tile8;
typedef DirectOp<Tile8::BM, Tile8::NT> Rows8;
typedef DirectOp<Tile8::BN, Tile8::NT> Stage8;
static constexpr int LDS8_B = 2 * Rows8::LDS_BYTES, LDS8 = LDS8_B + Stage8::LDS_BYTES;
static_assert(LDS8 >= Tile8::BM * Tile8::BN * 2, "the epilogues' 16-bit tile");

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

// The tile's weight rows.  What a slice asks for behind a row's end is the next row's, or, behind the last one's, nothing (the
// descriptor ends there).
struct Cols8 {
  static constexpr int R = Stage8::R;
  i32x4 rsrc;
  unsigned off[R];
  template <typename F>
  __device__ __forceinline__ void init(const char* b, int64_t left, int rot, F row_off) {
    rsrc = buffer_rsrc(b, (unsigned)(left < 0xffffffffLL ? left : 0xffffffffLL));
    const int t = threadIdx.x;
    turn = rot;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int p = rnd(j) * Tile8::NT + t, row = p >> 3;
      off[j] = (unsigned)row_off(row) + (((p & 7) ^ direct_swz(row)) << 4);
    }
  }
  int turn = 0;            // (see DirectOp)
  __device__ __forceinline__ int rnd(int j) const { const int r = j + turn; return r >= R ? r - R : r; }
  __device__ __forceinline__ void issue_one(unsigned tile, int kt, int j) const {
    buffer_to_lds16(rsrc, off[j], (unsigned)kt * 128u, tile + wave_uniform_id() * 1024 + rnd(j) * Tile8::NT * 16);
  }
};

// The rows in 8 bits are whole slices long here (zeros behind the last value); sx: this thread's (t < 128) dwords of its row's scales;
// s_scale: [2][128] dwords of LDS, four slices each.  What is loaded ahead behind the last slice is not looked at.
template <int SC>
__device__ __forceinline__ void mainloop_8bit(const Rows8& A, const Cols8& B, const WeightScales<SC>& W, const uint8_t* sx, int K, int rows_in,
                                              char* lds, unsigned* s_scale, Block (&acc)[Tile8::FM][Tile8::FN]) {
  typedef Tile8 TL;
  typedef typename WeightScales<SC>::V V;
  constexpr int COLS = 2 * TL::FN, LOADS = Rows8::R + Cols8::R, PER_STEP = LOADS / 3;
  static_assert(LOADS % 3 == 0, "the loads of the next slice go with three quarters of a slice's products");
  const int l = lane_id(), t = threadIdx.x, wave = t >> 6;
  const int nk = (K + 127) / 128;
  const int steps = __builtin_amdgcn_readfirstlane((rows_in + 31) / 32);   // blocks of 32 rows that there are: an expert's last tile is lower
  const unsigned lds_u = lds_address(lds);
  unsigned fetched = 0;
  V ws[2];
  W.load(0, ws);
  if (t < TL::BM) s_scale[t] = *(const unsigned*)sx;
#pragma unroll
  for (int j = 0; j < Rows8::R; ++j) A.issue_one(lds_u, 0, j);
#pragma unroll
  for (int j = 0; j < Cols8::R; ++j) B.issue_one(lds_u + LDS8_B, 0, j);
  auto slice = [&](int kt) {
    const char* ta = lds + (kt & 1) * Rows8::LDS_BYTES;
    const unsigned na = lds_u + ((kt & 1) ^ 1) * Rows8::LDS_BYTES;
    // this thread's pieces of slice kt have landed, everyone's have, and everyone is done with slice kt - 1
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // (taken here, where nothing is on its way: a wait for them further down would be one for the next slice's pieces)
    asm volatile("" : "+v"(ws[0]), "+v"(ws[1]), "+v"(fetched));
    __builtin_amdgcn_sched_barrier(0);
    i32x8 fb[COLS];
#pragma unroll
    for (int j = 0; j < COLS; ++j) fb[j] = fragment8<Stage8>(lds + LDS8_B, wave * TL::WTN + j * 16);
    // (the dword of a fragment's rows is read again for each of its four slices: eight registers less)
    const unsigned* sc = s_scale + ((kt >> 2) & 1) * TL::BM + (l & 15);
    i32x8 fa[2][2];
    unsigned xs[2][2];
    auto rows = [&](int s, int i) {
      fa[s & 1][i] = fragment8<Rows8>(ta, (2 * s + i) * 16);
      xs[s & 1][i] = sc[(2 * s + i) * 16];
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) rows(0, i);
    if ((kt & 3) == 3 && t < TL::BM) s_scale[(((kt >> 2) + 1) & 1) * TL::BM + t] = fetched;
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // everyone has the column operand's fragments
    __builtin_amdgcn_sched_barrier(0);
    if ((kt + 1) * 128 > K) {
      // a partial slice: the rows are zeros there, but the next row's bytes may be no number
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool there = kt * 128 + h * 64 + ((l >> 4) << 4) < K;
#pragma unroll
        for (int j = 0; j < COLS; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) fb[j][h * 4 + e] = there ? fb[j][h * 4 + e] : 0;
      }
    }
    V now[2] = {ws[0], ws[1]};
    W.load(min(kt + 1, nk - 1), ws);
    if ((kt & 3) == 1 && kt + 3 < nk && t < TL::BM) fetched = *(const unsigned*)(sx + (kt + 3));
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < TL::FM; ++s) {
#pragma unroll
      for (int q = s * PER_STEP; q < (s + 1) * PER_STEP && q < LOADS; ++q) {
        if (q < Cols8::R) B.issue_one(lds_u + LDS8_B, kt + 1, q);
        else A.issue_one(na, (kt + 1) * 64, q - Cols8::R);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (s > 0 && s >= steps) continue;
      if (s + 1 < TL::FM) {
#pragma unroll
        for (int i = 0; i < 2; ++i) rows(s + 1, i);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int x = (int)(xs[s & 1][i] >> (8 * (kt & 3)));
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
          f32x4& d = acc[s][j >> 1].q[2 * i + (j & 1)];
          if constexpr (SC == SCALES_EXACT) {
            bf16x8_8b va[4], vb[4];
            to_bf16x32(fa[s & 1][i], va);
            to_bf16x32(fb[j], vb);
            f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < 4; ++u) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[u], va[u], p, 0, 0, 0);
            const float f = now[j >> 1] * scale_of(x & 255);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = fmaf(p[e], f, d[e]);
          } else if constexpr (SC == SCALES_FLOAT) {
            const f32x4 p = mfma8(fb[j], fa[s & 1][i], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 127, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = fmaf(p[e], now[j >> 1], d[e]);
          } else {
            d = mfma8(fb[j], fa[s & 1][i], d, now[j >> 1], x);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
#pragma nounroll
  for (int kt = 0; kt < nk; ++kt) slice(kt);
  // (what was loaded ahead lands in LDS, which the epilogue uses)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The largest of the lanes that hold one row of the accumulators (16 and 32 apart)
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
// A tile's bytes on their way through LDS: rows of WIDTH + 16, so that the 16 rows of a wave's four-byte writes meet 64 different banks
template <int WIDTH>
struct ByteTile {
  static constexpr int ROW = WIDTH + 16;
  static __device__ __forceinline__ void put(char* lds, int row, int col, int q) { *(int*)(lds + row * ROW + col) = q; }
  // ROWS rows to `out`, `ld` bytes apart, `rows` and `cols` (a multiple of 16) of them there
  template <int ROWS>
  static __device__ __forceinline__ void store(const char* lds, uint8_t* out, int64_t ld, int rows, int cols) {
#pragma unroll
    for (int p = 0; p < ROWS * (WIDTH / 16) / Tile8::NT; ++p) {
      const int piece = p * Tile8::NT + (int)threadIdx.x, r = piece / (WIDTH / 16), c = piece % (WIDTH / 16) * 16;
      const i32x4 v = *(const i32x4*)(lds + r * ROW + c);
      if (r < rows && c < cols) *(i32x4*)(out + r * ld + c) = v;
    }
  }
};

// The gated unit behind a product.  A tile holds 128 columns of the hidden rows, one block: a wave 32 of each half (accumulators [.][0],
// [.][1]), so that a lane has both halves of its values, and a row's largest magnitude is that of four lanes and four waves.  Against
// the product's float32 rows written, read and taken to 8 bits by a pass (4099 tokens, 4096 / 14336): see the launcher.
__device__ __forceinline__ void epilogue_unit(Block (&acc)[Tile8::FM][Tile8::FN], const Product8Args& a, int row0, int rows, int n_tile, char* lds) {
  typedef Tile8 TL;
  typedef ByteTile<QB> Bytes;
  const int t = threadIdx.x, wave = t >> 6, l = lane_id(), F = a.N / 2;
  const bool mine = n_tile * QB + wave * 32 < F;                   // (F is a multiple of 32)
  float* top = (float*)(lds + TL::BM * Bytes::ROW);               // [wave][row]
  const int fb = (int)scale_blocks(F);
  // one value per accumulator of half h (2: the unit's) to 8 bits, its rows to `out`
  auto write = [&](auto value, uint8_t* out, int64_t ld, int cols, uint8_t* scales, int64_t sld) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * TL::FM; ++i) {
      float m = 0.0f;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int c = 0; c < 4; ++c) m = fmaxf(m, fabsf(value(i, g, c)));
      m = row_max(mine ? m : 0.0f);
      if (l < 16) top[wave * TL::BM + i * 16 + l] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * TL::FM; ++i) {
      const int r = i * 16 + (l & 15);
      const int byte = scale_byte(fmaxf(fmaxf(top[r], top[TL::BM + r]), fmaxf(top[2 * TL::BM + r], top[3 * TL::BM + r])));
      const float inv = inverse_scale(byte);
#pragma unroll
      for (int g = 0; g < 2; ++g)
        Bytes::put(lds, r, wave * 32 + 16 * g + 4 * (l >> 4), to_e4m3x4(value(i, g, 0), value(i, g, 1), value(i, g, 2), value(i, g, 3), inv));
      if (wave == 0 && l < 16 && r < rows) scales[r * sld] = (uint8_t)byte;
    }
    __syncthreads();
    Bytes::template store<TL::BM>(lds, out, ld, rows, cols);
  };
  auto half = [&](int h) { return [&acc, h](int i, int g, int c) { return acc[i >> 1][h].q[2 * (i & 1) + g][c]; }; };
  if (a.P8) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      write(half(h), a.P8 + ((int64_t)row0 * 2 + h) * F + n_tile * QB, 2 * F, min(QB, F - n_tile * QB), a.PS + ((int64_t)row0 * 2 + h) * fb + n_tile, 2 * fb);
  }
  const bool gate_first = (a.act & 1) != 0;
#pragma unroll
  for (int i = 0; i < 2 * TL::FM; ++i)
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float one = acc[i >> 1][0].q[2 * (i & 1) + g][c], two = acc[i >> 1][1].q[2 * (i & 1) + g][c];
        acc[i >> 1][0].q[2 * (i & 1) + g][c] = gate_first ? glu_h(a.act, one, two) : glu_h(a.act, two, one);
      }
  // (hidden rows are whole slices long, zeros behind the last value)
  const int64_t ld = scale_blocks(F) * QB;
  if (!mine) {
#pragma unroll
    for (int i = 0; i < TL::FM; ++i) acc[i][0].clear();
  }
  write(half(0), a.H8 + (int64_t)row0 * ld + n_tile * QB, ld, QB, a.HS + (int64_t)row0 * scale_row(F) + n_tile, scale_row(F));
}

// The gated unit's gradient behind a product that is dh.  F is a multiple of 128, so that the blocks of both halves of d(pre) lie in a tile: 256
// columns of dh, two blocks of each half.  32 rows at a time: their gradients of the first half take dh's registers, those of the second 32 more.
__device__ __forceinline__ void epilogue_unit_grad(Block (&acc)[Tile8::FM][Tile8::FN], const Product8Args& a, int row0, int rows, int n0, char* lds) {
  typedef Tile8 TL;
  typedef ByteTile<TL::BN> Bytes;
  constexpr int PARTS = 4, ROWS = TL::BM / PARTS, FR = ROWS / 16;
  const int t = threadIdx.x, wave = t >> 6, l = lane_id(), F = a.N;
  float* top = (float*)(lds + 2 * ROWS * Bytes::ROW);             // [half][wave][row]
  const bool gate_first = (a.act & 1) != 0;
  const bool mine = n0 + wave * TL::WTN < F;
  const int n = mine ? n0 + wave * TL::WTN : 0, fb = F / QB;
  const int64_t Ds = scale_row(2 * F);
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    float second[FR][2 * TL::FN][4];
    if (part) __syncthreads();
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int r = part * ROWS + i * 16 + (l & 15), row = row0 + min(r, rows - 1);
      const uint8_t* p8 = a.P8 + (int64_t)row * 2 * F + n;
      const uint8_t* ps = a.PS + (int64_t)row * 2 * fb + n / QB;
      const float s1 = scale_of(ps[0]), s2 = scale_of(ps[fb]);
      float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j) {
        float one[4], two[4];
        from_e4m3x4(*(const int*)(p8 + j * 16 + 4 * (l >> 4)), s1, one);
        from_e4m3x4(*(const int*)(p8 + F + j * 16 + 4 * (l >> 4)), s2, two);
        f32x4& d = acc[(part * FR + i) >> 1][j >> 1].q[2 * ((part * FR + i) & 1) + (j & 1)];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float dl, dg;
          glu_grad(a.act, d[c], gate_first ? one[c] : two[c], gate_first ? two[c] : one[c], dl, dg);
          d[c] = gate_first ? dg : dl;
          second[i][j][c] = gate_first ? dl : dg;
          m1 = fmaxf(m1, fabsf(d[c])), m2 = fmaxf(m2, fabsf(second[i][j][c]));
        }
      }
      m1 = row_max(m1), m2 = row_max(m2);
      if (l < 16) top[wave * ROWS + i * 16 + l] = m1, top[(4 + wave) * ROWS + i * 16 + l] = m2;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int r = i * 16 + (l & 15), pair = wave & 2;            // the two waves that share this one's blocks
      const int b1 = scale_byte(fmaxf(top[pair * ROWS + r], top[(pair + 1) * ROWS + r]));
      const int b2 = scale_byte(fmaxf(top[(4 + pair) * ROWS + r], top[(5 + pair) * ROWS + r]));
      const float inv1 = inverse_scale(b1), inv2 = inverse_scale(b2);
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j) {
        const f32x4& d = acc[(part * FR + i) >> 1][j >> 1].q[2 * ((part * FR + i) & 1) + (j & 1)];
        const int col = wave * TL::WTN + j * 16 + 4 * (l >> 4);
        Bytes::put(lds, r, col, to_e4m3x4(d[0], d[1], d[2], d[3], inv1));
        Bytes::put(lds + ROWS * Bytes::ROW, r, col, to_e4m3x4(second[i][j][0], second[i][j][1], second[i][j][2], second[i][j][3], inv2));
      }
      if ((wave & 1) == 0 && l < 16 && part * ROWS + r < rows && mine) {
        uint8_t* s = a.HS + (int64_t)(row0 + part * ROWS + r) * Ds + n / QB;
        s[0] = (uint8_t)b1, s[fb] = (uint8_t)b2;
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      Bytes::template store<ROWS>(lds + h * ROWS * Bytes::ROW, a.H8 + (int64_t)(row0 + part * ROWS) * 2 * F + h * F + n0, 2 * F, rows - part * ROWS,
                                  min(TL::BN, F - n0));      // (whole slices: 2 F is a multiple of them)
  }
}

// (float32 rows: the operands as bfloat16 take the registers of a second workgroup)
template <typename TO, int SC, int EPI>
__global__ __launch_bounds__(Tile8::NT, SC == SCALES_EXACT ? 1 : 2) void product_8bit_kernel(Product8Args a, int bias_dtype, Raster rast) {
  typedef Tile8 TL;
  __shared__ __attribute__((aligned(16))) char lds[LDS8];
  __shared__ unsigned s_scale[2 * TL::BM];
  __shared__ int64_t s_dst[EPI == EPI_ROWS ? TL::BM : 1];
  __shared__ int s_src[TL::BM];
  int m_tile, n_tile, m_loc, n_loc, e, row0, rows;
  if (!rast.map<2 * Raster::SN>(blockIdx.x, m_tile, n_tile, m_loc, n_loc)) return;
  if (!find_tile<TL::BM>(a.off, a.E, m_tile, e, row0, rows)) return;
  const int t = threadIdx.x, F = a.N / 2;
  // first output column of the tile, and of this wave's two halves of 32
  const int n0 = n_tile * (EPI == EPI_UNIT ? QB : TL::BN);
  const uint8_t* sx = nullptr;
  if (t < TL::BM) {
    const int row = row0 + (t < rows ? t : rows - 1);                  // rows behind the last one repeat it
    int slot = 0;
    if (!a.x_grouped || (EPI == EPI_ROWS && !a.y_grouped)) slot = (int)a.idx[row];
    const int src = a.x_grouped ? row : (int)((unsigned)slot / (unsigned)a.fan);
    s_src[t] = src;
    if constexpr (EPI == EPI_ROWS) s_dst[t] = t < rows ? (int64_t)(a.y_grouped ? row : slot) * a.sym : -1;
    sx = a.XS + src * scale_row(a.K);
  }
  __syncthreads();
  Rows8 A;
  A.rot = (n_loc * Rows8::R / (2 * Raster::SN)) % Rows8::R;
  const int src0 = a.x_grouped ? row0 : 0;
  const int64_t ld = (a.K + QB - 1) / QB * QB;                         // the rows are whole slices long
  A.init((const char*)a.X + src0 * ld, [&](int row) { return (int64_t)(s_src[row] - src0) * ld; });
  Cols8 B;
  const int turn = (m_loc * Cols8::R / Raster::SM) % Cols8::R;
  const int64_t swn = a.swn;
  const int wave_u = (int)wave_uniform_id();
  int nb[2];
  if constexpr (EPI == EPI_UNIT) {
    // tile column -> weight row: wave, first 32 of its 64 from the first half of the rows, the others from the second
    B.init((const char*)a.W + e * a.swe, (int64_t)a.N * swn, turn,
           [&](int tc) { return (int64_t)(min(n0 + (tc >> 6) * 32 + (tc & 31), F - 1) + (tc & 32 ? F : 0)) * swn; });
    const int hc = min(n0 + wave_u * 32, F - 1);
    nb[0] = hc / QB, nb[1] = (F + hc) / QB;
  } else {
    const int last = a.N - 1 - n0;
    B.init((const char*)a.W + e * a.swe + n0 * swn, (a.N - n0) * swn, turn, [&](int row) { return (int64_t)min(row, last) * swn; });
    nb[0] = nb[1] = min(n0 + wave_u * TL::WTN, a.N - 1) / QB;
  }
  WeightScales<SC> W;
  const int WSB = SC == SCALES_BYTES ? 1 : SC == SCALES_FLOAT || a.ws_f32 ? 4 : 1;
#pragma unroll
  for (int h = 0; h < 2; ++h) W.at[h] = (const char*)a.WS + (e * a.sse + nb[h] * a.ssn) * WSB;
  W.step = a.ssk * WSB;
  W.f32 = a.ws_f32 != 0;
  Block acc[TL::FM][TL::FN];
#pragma unroll
  for (int i = 0; i < TL::FM; ++i)
#pragma unroll
    for (int j = 0; j < TL::FN; ++j) acc[i][j].clear();
  mainloop_8bit<SC>(A, B, W, sx, a.K, rows, lds, s_scale, acc);
  __syncthreads();
  const int wave = t >> 6, l = lane_id();
  if (EPI != EPI_UNIT_GRAD && a.b) {
#pragma unroll
    for (int j = 0; j < 2 * TL::FN; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        int n = n0 + wave * TL::WTN + j * 16 + 4 * (l >> 4) + c;
        bool there = n < a.N;
        if constexpr (EPI == EPI_UNIT) {
          n = n0 + wave * 32 + (j & 1) * 16 + 4 * (l >> 4) + c;
          there = n < F;
          n += j >= 2 ? F : 0;
        }
        const float b = there ? bias_value(a.b, e * a.sbe + n * a.sbn, bias_dtype) : 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * TL::FM; ++i) acc[i >> 1][j >> 1].q[2 * (i & 1) + (j & 1)][c] += b;
      }
  }
  if constexpr (EPI == EPI_UNIT) {
    epilogue_unit(acc, a, row0, rows, n_tile, lds);
    return;
  } else if constexpr (EPI == EPI_UNIT_GRAD) {
    epilogue_unit_grad(acc, a, row0, rows, n0, lds);
    return;
  } else {
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
}

template <typename TO, bool EXACT, int EPI>
static int launch_product(const Product8Args& a, int bias_dtype, hipStream_t st) {
  const int64_t m_tiles = max_tiles(a.L, a.E, Tile8::BM);
  const int n_tiles = EPI == EPI_UNIT ? (a.N / 2 + QB - 1) / QB : (a.N + Tile8::BN - 1) / Tile8::BN;
  const Raster r = a.L < (int64_t)STRIPE_BELOW * a.E ? make_striped(m_tiles, n_tiles, GM_RING)
                                                     : make_raster(m_tiles, n_tiles, GM_S2S, 2 * Raster::SN);
  if (r.grid() > 0x7fffffffLL) { set_error("product_8bit: grid too large"); return SMOE_ERR_RANGE; }
  const unsigned grid = (unsigned)r.grid();
  if constexpr (EXACT) product_8bit_kernel<TO, SCALES_EXACT, EPI><<<grid, Tile8::NT, 0, st>>>(a, bias_dtype, r);
  else if (a.ws_f32) product_8bit_kernel<TO, SCALES_FLOAT, EPI><<<grid, Tile8::NT, 0, st>>>(a, bias_dtype, r);
  else product_8bit_kernel<TO, SCALES_BYTES, EPI><<<grid, Tile8::NT, 0, st>>>(a, bias_dtype, r);
  return launch_status("product_8bit");
}

// The unit's blocks are 128 hidden columns, and a wave's 32 of either half have one scale of the weights; its weight rows are
// 32-bit offsets from the expert's first.  Else the product's float32 rows go through a pass of their own.
bool unit_rides(int64_t d, int64_t F) { return F % 32 == 0 && 2 * F * padded_row(d) < (1LL << 31); }
// The gradient's blocks run along both halves: they lie within one half where F is whole blocks.
bool unit_grad_rides(int64_t F) { return F % QB == 0; }

int launch_product_8bit(const Product8Args& a, int row_dtype, int out_dtype, hipStream_t st, int epilogue) {
  const bool exact = row_dtype == SMOE_F32;
  if (epilogue == EPI_UNIT) return exact ? launch_product<float, true, EPI_UNIT>(a, row_dtype, st) : launch_product<float, false, EPI_UNIT>(a, row_dtype, st);
  if (epilogue == EPI_UNIT_GRAD)
    return exact ? launch_product<float, true, EPI_UNIT_GRAD>(a, row_dtype, st) : launch_product<float, false, EPI_UNIT_GRAD>(a, row_dtype, st);
  if (exact) return launch_product<float, true, EPI_ROWS>(a, row_dtype, st);
  if (out_dtype == SMOE_F32) return launch_product<float, false, EPI_ROWS>(a, row_dtype, st);
  if (out_dtype == SMOE_BF16) return launch_product<bf16_t, false, EPI_ROWS>(a, row_dtype, st);
  return launch_product<f16_t, false, EPI_ROWS>(a, row_dtype, st);
}

}  // namespace smoe
