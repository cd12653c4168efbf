// scatter2scatter on 8-bit operands (eight_bit.hpp): Y[dst(n)] = X[src(n)] W[e(n)]^T over rows sorted by expert, in tiles of
// 128 (64) rows x 256 columns that never straddle two experts.
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

static constexpr int NT8 = 256, BN8 = 256;
// tiles of 128 rows, two workgroups per CU, or of 64, three (3 below: epilogues derive nothing from the thread's index ahead of the loop)
template <int BM> using Tile8 = Tile<BM, BN8, 1, 4, 2, false, 3, true>;
template <class TL> using Rows8 = DirectOp<TL::BM, NT8>;
typedef DirectOp<BN8, NT8> Stage8;
template <class TL> static constexpr int LDS8_B = 2 * Rows8<TL>::LDS_BYTES;
template <class TL> static constexpr int LDS8 = LDS8_B<TL> + Stage8::LDS_BYTES;      // (the epilogues' 16-bit tile is smaller)

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
      else v[h] = f32 ? *(const float*)p : weight_scale(*(const uint8_t*)p);
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
      const int p = rnd(j) * NT8 + t, row = p >> 3;
      off[j] = (unsigned)row_off(row) + (((p & 7) ^ direct_swz(row)) << 4);
    }
  }
  int turn = 0;            // (see DirectOp)
  __device__ __forceinline__ int rnd(int j) const { const int r = j + turn; return r >= R ? r - R : r; }
  __device__ __forceinline__ void issue_one(unsigned tile, int kt, int j) const {
    buffer_to_lds16(rsrc, off[j], (unsigned)kt * 128u, tile + wave_uniform_id() * 1024 + rnd(j) * NT8 * 16);
  }
};

// The rows in 8 bits are whole slices long here (zeros behind the last value); sx: this thread's (t < 128) dwords of its row's scales;
// s_scale: [2][128] dwords of LDS, four slices each.  What is loaded ahead behind the last slice is not looked at.
template <class TL, int SC>
__device__ __forceinline__ void mainloop_8bit(const Rows8<TL>& A, const Cols8& B, const WeightScales<SC>& W, const uint8_t* sx, int K, char* lds,
                                              unsigned* s_scale, Block (&acc)[TL::FM][TL::FN]) {
  typedef typename WeightScales<SC>::V V;
  constexpr int COLS = 2 * TL::FN, LOADS = Rows8<TL>::R + Cols8::R, PER_STEP = TL::FM == 4 ? LOADS / 3 : LOADS;
  static_assert(TL::FM != 4 || LOADS % 3 == 0, "the loads of the next slice go with three quarters of a slice's products, or the first half");
  const int l = lane_id(), t = threadIdx.x, wave = t >> 6;
  const int nk = (K + 127) / 128;
  const unsigned lds_u = lds_address(lds);
  unsigned fetched = 0;
  V ws[2];
  W.load(0, ws);
  if (t < TL::BM) s_scale[t] = *(const unsigned*)sx;
#pragma unroll
  for (int j = 0; j < Rows8<TL>::R; ++j) A.issue_one(lds_u, 0, j);
#pragma unroll
  for (int j = 0; j < Cols8::R; ++j) B.issue_one(lds_u + LDS8_B<TL>, 0, j);
  auto slice = [&](int kt) {
    const char* ta = lds + (kt & 1) * Rows8<TL>::LDS_BYTES;
    const unsigned na = lds_u + ((kt & 1) ^ 1) * Rows8<TL>::LDS_BYTES;
    // this thread's pieces of slice kt have landed, everyone's have, and everyone is done with slice kt - 1
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // (taken here, where nothing is on its way: a wait for them further down would be one for the next slice's pieces)
    asm volatile("" : "+v"(ws[0]), "+v"(ws[1]), "+v"(fetched));
    __builtin_amdgcn_sched_barrier(0);
    i32x8 fb[COLS];
#pragma unroll
    for (int j = 0; j < COLS; ++j) fb[j] = fragment8<Stage8>(lds + LDS8_B<TL>, wave * TL::WTN + j * 16);
    // (the dword of a fragment's rows is read again for each of its four slices: eight registers less)
    const unsigned* sc = s_scale + ((kt >> 2) & 1) * TL::BM + (l & 15);
    i32x8 fa[2][2];
    unsigned xs[2][2];
    auto rows = [&](int s, int i) {
      fa[s & 1][i] = fragment8<Rows8<TL>>(ta, (2 * s + i) * 16);
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
        if (q < Cols8::R) B.issue_one(lds_u + LDS8_B<TL>, kt + 1, q);
        else A.issue_one(na, (kt + 1) * 64, q - Cols8::R);
      }
      __builtin_amdgcn_sched_barrier(0);
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
  template <typename V>
  static __device__ __forceinline__ void put(char* lds, int row, int col, V q) { *(V*)(lds + row * ROW + col) = q; }
  // ROWS rows to `out`, `ld` bytes apart, `rows` and `cols` (a multiple of 16) of them there
  template <int ROWS>
  static __device__ __forceinline__ void store(const char* lds, uint8_t* out, int64_t ld, int rows, int cols) {
    const int t = late_thread<Tile8<128>>();
#pragma unroll
    for (int p = 0; p < ROWS * (WIDTH / 16) / NT8; ++p) {
      const int piece = p * NT8 + t, r = piece / (WIDTH / 16), c = piece % (WIDTH / 16) * 16;
      const i32x4 v = *(const i32x4*)(lds + r * ROW + c);
      if (r < rows && c < cols) *(i32x4*)(out + r * ld + c) = v;
    }
  }
};

// The gated unit behind a product.  A tile holds 128 columns of the hidden rows, one block: a wave 32 of each half (accumulators [.][0],
// [.][1]: the linear half and the gate's, by which rows of the weights the wave takes), so that a lane has both halves of its
// values, and a row's largest magnitude is that of four lanes and four waves.  It is bound by its own arithmetic: with a choice of the
// gate's half and of columns that are not there for each value, and the scale multiplied in before a conversion without one,
// 4150 instructions instead of 2660, 1054 instead of 1015 us (4099 tokens, 8 experts, 4096 / 14336; 8192 tokens to 8 of 128
// experts, 2048 / 768, with the checkpoint: 319, 303).  As a pass over the product's float32 rows: 1065 + 191 us (229 + 90).
template <class TL>
__device__ __forceinline__ void epilogue_unit(Block (&acc)[TL::FM][TL::FN], const Product8Args& a, int row0, int rows, int n_tile,
                                              const float* s_bias, char* lds) {
  typedef ByteTile<QB> Bytes;
  constexpr int ROWS = TL::BM == 64 ? 32 : 64, PARTS = TL::BM / ROWS, FR = ROWS / 16, SIDE = ROWS * Bytes::ROW;
  const int t = late_thread<TL>(), wave = t >> 6, l = t & 63, F = a.N / 2, fb = (int)scale_blocks(F);
  const bool mine = n_tile * QB + wave * 32 < F;          // (F is a multiple of 32)
  const int64_t ld = scale_blocks(F) * QB;                         // (hidden rows are whole slices long, zeros behind the last value)
  float* top = (float*)(lds + 3 * SIDE);                           // [the unit, its halves][wave][row]
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    float unit[FR][2][4];
    if (part) __syncthreads();
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int ai = (part * FR + i) >> 1, aq = 2 * ((part * FR + i) & 1);
      float m[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float* b = s_bias + wave * TL::WTN + 8 * (l >> 4) + 4 * g;
        f32x4 &lin = acc[ai][0].q[aq + g], &gate = acc[ai][1].q[aq + g];
        lin += *(const f32x4*)b, gate += *(const f32x4*)(b + 32);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          unit[i][g][c] = glu_h(a.act, gate[c], lin[c]);
          m[0] = fmaxf(m[0], fabsf(unit[i][g][c])), m[1] = fmaxf(m[1], fabsf(lin[c])), m[2] = fmaxf(m[2], fabsf(gate[c]));
        }
      }
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        m[s] = row_max(mine ? m[s] : 0.0f);
        if (l < 16) top[(s * 4 + wave) * ROWS + i * 16 + l] = m[s];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int ai = (part * FR + i) >> 1, aq = 2 * ((part * FR + i) & 1), r = i * 16 + (l & 15);
      const int64_t row = row0 + part * ROWS + r;
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        if (s && !a.P8) break;
        const float* most = top + s * 4 * ROWS + r;
        const int byte = scale_byte(fmaxf(fmaxf(most[0], most[ROWS]), fmaxf(most[2 * ROWS], most[3 * ROWS])));
        const float scale = scale_of(byte);
        i32x2 both;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const f32x4 &lin = acc[ai][0].q[aq + g], &gate = acc[ai][1].q[aq + g];
          const int q = s == 0   ? to_e4m3x4(unit[i][g][0], unit[i][g][1], unit[i][g][2], unit[i][g][3], scale)
                        : s == 1 ? to_e4m3x4(lin[0], lin[1], lin[2], lin[3], scale)
                                 : to_e4m3x4(gate[0], gate[1], gate[2], gate[3], scale);
          both[g] = mine ? q : 0;
        }
        Bytes::put(lds + s * SIDE, r, wave * 32 + 8 * (l >> 4), both);
        if (wave == 0 && l < 16 && part * ROWS + r < rows) {
          uint8_t* out = s == 0 ? a.HS + row * scale_row(F) : a.PS + (2 * row + s - 1) * fb;
          out[n_tile] = (uint8_t)byte;
        }
      }
    }
    __syncthreads();
    const int64_t first = row0 + part * ROWS;
    Bytes::template store<ROWS>(lds, a.H8 + first * ld + n_tile * QB, ld, rows - part * ROWS, QB);
    if (a.P8) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        Bytes::template store<ROWS>(lds + (1 + h) * SIDE, a.P8 + (first * 2 + h) * F + n_tile * QB, 2 * F, rows - part * ROWS, min(QB, F - n_tile * QB));
    }
  }
}

// The gated unit's gradient behind a product that is dh.  F is a multiple of 128, so that the blocks of both halves of d(pre) lie in a tile: 256
// columns of dh, two blocks of each half.  32 rows at a time: the linear half's gradients take dh's registers, the gate's 32 more.
// 8192 tokens to 8 of 128 experts, 2048 / 768: 222 us, as a pass over the product's float32 rows 229 + 112.
template <class TL>
__device__ __forceinline__ void epilogue_unit_grad(Block (&acc)[TL::FM][TL::FN], const Product8Args& a, int row0, int rows, int n0, char* lds) {
  typedef ByteTile<TL::BN> Bytes;
  constexpr int ROWS = 32, PARTS = TL::BM / ROWS, FR = ROWS / 16;
  const int t = late_thread<TL>(), wave = t >> 6, l = t & 63, F = a.N;
  float* top = (float*)(lds + 2 * ROWS * Bytes::ROW);             // [half][wave][row]
  const int swapped = a.act & 1, lin_at = swapped * F, gate_at = F - lin_at;            // the gate's half is the first one
  const bool mine = n0 + wave * TL::WTN < F;
  const int n = mine ? n0 + wave * TL::WTN : 0, fb = F / QB;
  const int64_t Ds = scale_row(2 * F);
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    float dgate[FR][2 * TL::FN][4];
    if (part) __syncthreads();
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int r = part * ROWS + i * 16 + (l & 15), row = row0 + min(r, rows - 1);
      const uint8_t* p8 = a.P8 + (int64_t)row * 2 * F + n;
      const uint8_t* ps = a.PS + (int64_t)row * 2 * fb + n / QB;
      const float s1 = scale_of(ps[0]), s2 = scale_of(ps[fb]);
      float m1 = 0.0f, m2 = 0.0f;
      const i32x4 lin8 = *(const i32x4*)(p8 + 16 * (l >> 4)), gate8 = *(const i32x4*)(p8 + F + 16 * (l >> 4));
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j) {
        float lin[4], gate[4];
        from_e4m3x4_exact(lin8[j], s1, lin);
        from_e4m3x4_exact(gate8[j], s2, gate);
        f32x4& d = acc[(part * FR + i) >> 1][j >> 1].q[2 * ((part * FR + i) & 1) + (j & 1)];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float dl;
          glu_grad(a.act, d[c], gate[c], lin[c], dl, dgate[i][j][c]);
          d[c] = dl;
          m1 = fmaxf(m1, fabsf(d[c])), m2 = fmaxf(m2, fabsf(dgate[i][j][c]));
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
      const float f1 = scale_of(b1), f2 = scale_of(b2);
      i32x4 dl8, dg8;
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j) {
        const f32x4& d = acc[(part * FR + i) >> 1][j >> 1].q[2 * ((part * FR + i) & 1) + (j & 1)];
        dl8[j] = to_e4m3x4(d[0], d[1], d[2], d[3], f1);
        dg8[j] = to_e4m3x4(dgate[i][j][0], dgate[i][j][1], dgate[i][j][2], dgate[i][j][3], f2);
      }
      Bytes::put(lds, r, wave * TL::WTN + 16 * (l >> 4), dl8);
      Bytes::put(lds + ROWS * Bytes::ROW, r, wave * TL::WTN + 16 * (l >> 4), dg8);
      if ((wave & 1) == 0 && l < 16 && part * ROWS + r < rows && mine) {
        uint8_t* s = a.HS + (int64_t)(row0 + part * ROWS + r) * Ds + n / QB;
        s[swapped * fb] = (uint8_t)b1, s[(1 - swapped) * fb] = (uint8_t)b2;
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      Bytes::template store<ROWS>(lds + h * ROWS * Bytes::ROW, a.H8 + (int64_t)(row0 + part * ROWS) * 2 * F + (h ? gate_at : lin_at) + n0, 2 * F, rows - part * ROWS,
                                  min(TL::BN, F - n0));      // (whole slices: 2 F is a multiple of them)
  }
}

// ---- who takes what --------------------------------------------------------------------------------------
// Tiles in one line: expert by expert, inside an expert bands of eight tile rows, inside a band column by column.  A round is what the card
// runs side by side, two workgroups per CU; XCD x (a workgroup's index modulo 8) takes the x-th eighth of a round, 64 neighbours in
// line, which share eight row panels and eight column panels in its L2.  A product of few rounds that ends in a round of at
// most half the card's tiles cuts their contraction into parts, one workgroup each, which leave their sums in `partial`;
// product_8bit_join_kernel adds the parts up in their order.  8 experts x 1025 rows on average, 14336 -> 4096, 2.3 rounds: 554 us,
// in parts 461 + 16 for the sums.  At 4096 values to contract the parts save less than the sums cost (12 tile rows x 16 columns: 78 us, in parts 78 + 15).
// Bands of 4 and 16 tile rows: 1.00 and 1.01 times the time.
static constexpr int BAND8 = 8, PARTS8 = 8, PART_SLICES = 16, SPLIT_SLICES = 64, SPLIT_ROUNDS = 8;
template <class TL> static constexpr int64_t TILE8_FLOATS = TL::BM * TL::BN;
template <int SC, int BM> static constexpr int round_tiles = SC == SCALES_EXACT ? 256 : BM == 64 ? 768 : 512;
struct Share8 {
  int e, row0, rows, row, column;
  int part, parts, slice0, slices;      // the contraction's part, of `parts`; its slices
  int slot;                             // of this part's sums
};
// Share number b of a product (JOIN: tile number b of those whose contraction is cut).  The same answer in every wave.
template <int BM, int ROUND, bool JOIN>
__device__ __forceinline__ bool find_share(const Product8Args& a, int b, int n_tiles, Share8& s) {
  const int nk = (a.K + QB - 1) / QB;
  const int total = count_tile_rows<BM>(a.off, a.E) * n_tiles;
  int rest = 0;
  s.part = 0, s.parts = 1, s.slice0 = 0, s.slices = nk, s.slot = 0;
  if (a.partial) {
    rest = total % ROUND;
    int parts = rest ? min(min(ROUND / rest, PARTS8), nk / PART_SLICES) : 1;
    if (parts < 2) {
      rest = 0;
    } else {
      s.slices = ((nk + parts - 1) / parts + 3) & ~3;               // (four slices' scales are one dword)
      s.parts = (nk + s.slices - 1) / s.slices;
    }
  }
  const int whole = total - rest;                                  // tiles that are multiplied in one piece
  int l;
  if (JOIN) {
    if (b >= rest) return false;
    l = whole + b;
    s.slot = b * s.parts;
  } else {
    const int first = b / ROUND * ROUND;                           // of this workgroup's round
    const int x = b & 7, j = (b - first) >> 3;
    if (first < whole) {
      const int there = min(ROUND, whole - first), len = (there + 7) >> 3;
      if (j >= len || x * len + j >= there) return false;
      l = first + x * len + j;
      s.parts = 1, s.slices = nk;
    } else {
      const int start = (whole + ROUND - 1) / ROUND * ROUND, there = rest * s.parts, len = (there + 7) >> 3;
      if (first != start || j >= len || x * len + j >= there) return false;
      const int u = x * len + j;
      s.part = u / rest;
      const int tile = u - s.part * rest;
      l = whole + tile;
      s.slot = tile * s.parts + s.part;
      s.slice0 = s.part * s.slices;
      s.slices = min(s.slices, nk - s.slice0);
    }
  }
  int before = 0;                                                  // tile rows of the experts before this group of 64
  for (int e0 = 0; e0 < a.E; e0 += 64) {
    int lo, hi;
    load_expert_rows(a.off, a.E, e0, lo, hi);
    const int nt = (hi - lo + BM - 1) / BM, incl = wave_scan(nt), cum = before + incl;
    const unsigned long long hit = __ballot((int64_t)cum * n_tiles > l);
    if (hit) {
      const int src = __ffsll((long long)hit) - 1;
      const int lo_s = __builtin_amdgcn_readlane(lo, src), hi_s = __builtin_amdgcn_readlane(hi, src);
      const int rows_e = __builtin_amdgcn_readlane(nt, src);
      int in = l - (__builtin_amdgcn_readlane(cum, src) - rows_e) * n_tiles;
      const int bands = max(1, (rows_e + BAND8 / 2 - 1) / BAND8), step = (rows_e + bands - 1) / bands;      // 1 to 12 tile rows each
      const int band = in / (step * n_tiles), high = min(step, rows_e - band * step);
      in -= band * (step * n_tiles);
      const int column = in / high, row = band * step + in - column * high;
      s.e = __builtin_amdgcn_readfirstlane(e0 + src);
      s.column = __builtin_amdgcn_readfirstlane(column);
      s.row = __builtin_amdgcn_readfirstlane(row);
      s.row0 = lo_s + s.row * BM;
      s.rows = min(BM, hi_s - s.row0);
      s.part = __builtin_amdgcn_readfirstlane(s.part), s.parts = __builtin_amdgcn_readfirstlane(s.parts);
      s.slice0 = __builtin_amdgcn_readfirstlane(s.slice0), s.slices = __builtin_amdgcn_readfirstlane(s.slices);
      s.slot = __builtin_amdgcn_readfirstlane(s.slot);
      return true;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// A tile's sums, rounded, through LDS to its rows: 16-byte pieces, a wave whole 128-byte lines, or value by value where rows do not
// start at multiples of 16 bytes.  Float32 goes in two halves of 128 columns, the 64 KB of a 16-bit tile.
template <class TL, typename TO>
__device__ __forceinline__ void store_rows(const Block (&acc)[TL::FM][TL::FN], const Product8Args& a, int n0, const int64_t* s_dst,
                                           const float* s_bias, char* lds) {
  constexpr int PER = 16 / (int)sizeof(TO), HALVES = (int)sizeof(TO) / 2, COLS = TL::BN / HALVES, CPR = COLS / PER;      // 32 pieces a row
  const int t = late_thread<TL>(), wave = t >> 6, l = t & 63;
  TO* Y = (TO*)a.Y;
  const bool whole = ((uintptr_t)Y & 15) == 0 && ((a.sym | a.N) & (PER - 1)) == 0;
  auto place = [](int row, int col) { return row * (COLS * (int)sizeof(TO)) + (((col / PER) ^ (row & (CPR - 1))) << 4) + (col % PER) * (int)sizeof(TO); };
#pragma unroll
  for (int half = 0; half < HALVES; ++half) {
    if (half) __syncthreads();
    if (HALVES == 1 || (wave >> 1) == half) {
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; j += PER / 4) {
        const int tc = wave * TL::WTN + 16 * (l >> 4) + 4 * j;
#pragma unroll
        for (int i = 0; i < 2 * TL::FM; ++i) {
          TO v[PER];
#pragma unroll
          for (int c = 0; c < PER; ++c)
            v[c] = from_f32<TO>(acc[i >> 1][(j + c / 4) >> 1].q[2 * (i & 1) + ((j + c / 4) & 1)][c & 3] + s_bias[tc + c]);
          i32x4 p;
          __builtin_memcpy(&p, v, 16);
          *(i32x4*)(lds + place(i * 16 + (l & 15), tc % COLS)) = p;
        }
      }
    }
    __syncthreads();
    constexpr int PIECES = TL::BM * CPR / TL::NT, GRP = 8;
#pragma unroll
    for (int g0 = 0; g0 < PIECES; g0 += GRP) {
      i32x4 v[GRP];
      int64_t d[GRP];
#pragma unroll
      for (int g = 0; g < GRP; ++g) {
        const int p = (g0 + g) * TL::NT + t, r = p / CPR;
        d[g] = s_dst[r];
        v[g] = *(const i32x4*)(lds + place(r, p % CPR * PER));
      }
#pragma unroll
      for (int g = 0; g < GRP; ++g) {
        const int n = n0 + half * COLS + ((g0 + g) * TL::NT + t) % CPR * PER;
        if (d[g] < 0 || n >= a.N) continue;
        if (whole) {
          stream_store(v[g], (i32x4*)(Y + d[g] + n));
        } else {
          TO e[PER];
          __builtin_memcpy(e, &v[g], 16);
#pragma unroll
          for (int c = 0; c < PER; ++c)
            if (n + c < a.N) Y[d[g] + n + c] = e[c];
        }
      }
    }
  }
}

// What follows a tile's sums: the bias, and the rows or the unit or its gradient
template <class TL, typename TO, int EPI>
__device__ __forceinline__ void finish(Block (&acc)[TL::FM][TL::FN], const Product8Args& a, int bias_dtype, int e, int row0, int rows, int n_tile,
                                       const int64_t* s_dst, float* s_bias, char* lds) {
  const int t = late_thread<TL>(), F = a.N / 2, n0 = n_tile * (EPI == EPI_UNIT ? QB : TL::BN);
  if constexpr (EPI == EPI_UNIT_GRAD) {
    epilogue_unit_grad<TL>(acc, a, row0, rows, n0, lds);
  } else {
    // the tile's 256 columns' biases through LDS, zeros without one
    int n = n0 + t;
    bool there = n < a.N;
    if constexpr (EPI == EPI_UNIT) {
      n = n0 + (t >> 6) * 32 + (t & 31);
      there = n < F;
      n += (t & 32 ? 1 - (a.act & 1) : a.act & 1) * F;
    }
    s_bias[t] = a.b && there ? bias_value(a.b, e * a.sbe + n * a.sbn, bias_dtype) : 0.0f;
    __syncthreads();
    if constexpr (EPI == EPI_UNIT) epilogue_unit<TL>(acc, a, row0, rows, n_tile, s_bias, lds);
    else store_rows<TL, TO>(acc, a, n0, s_dst, s_bias, lds);
  }
}

// (float32 rows: the operands as bfloat16 take the registers of a second workgroup)
template <typename TO, int SC, int EPI, int BM>
__global__ __launch_bounds__(NT8, SC == SCALES_EXACT ? 1 : BM == 64 ? 3 : 2) void product_8bit_kernel(Product8Args a, int bias_dtype, int n_tiles) {
  typedef Tile8<BM> TL;
  __shared__ __attribute__((aligned(16))) char lds[LDS8<TL>];
  __shared__ unsigned s_scale[2 * TL::BM];
  __shared__ int64_t s_dst[EPI == EPI_ROWS ? TL::BM : 1];
  __shared__ __attribute__((aligned(16))) float s_bias[TL::BN];
  __shared__ int s_src[TL::BM];
  Share8 share;
  if (!find_share<BM, round_tiles<SC, BM>, false>(a, blockIdx.x, n_tiles, share)) return;
  const int e = share.e, row0 = share.row0, rows = share.rows, n_tile = share.column, k0 = share.slice0;
  const int t = threadIdx.x, F = a.N / 2;
  const int n0 = n_tile * (EPI == EPI_UNIT ? QB : TL::BN);         // first output column of the tile (of either half)
  const uint8_t* sx = nullptr;
  if (t < TL::BM) {
    const int row = row0 + (t < rows ? t : rows - 1);                  // rows behind the last one repeat it
    int slot = 0;
    if (!a.x_grouped || (EPI == EPI_ROWS && !a.y_grouped)) slot = (int)a.idx[row];
    const int src = a.x_grouped ? row : (int)((unsigned)slot / (unsigned)a.fan);
    s_src[t] = src;
    if constexpr (EPI == EPI_ROWS) s_dst[t] = t < rows ? (int64_t)(a.y_grouped ? row : slot) * a.sym : -1;
    sx = a.XS + src * scale_row(a.K) + k0;
  }
  __syncthreads();
  Rows8<TL> A;
  A.rot = (n_tile % BAND8 * Rows8<TL>::R / BAND8) % Rows8<TL>::R;
  const int src0 = a.x_grouped ? row0 : 0;
  const int64_t ld = (a.K + QB - 1) / QB * QB;                         // the rows are whole slices long
  A.init((const char*)a.X + src0 * ld + k0 * QB, [&](int row) { return (int64_t)(s_src[row] - src0) * ld; });
  // (which column a weight row in LDS belongs to is ours to choose: a lane's four fragments' columns lie side by side, 16 of them, in the unit 8 of
  // either half, so that it writes and reads whole pieces of rows)
  Cols8 B;
  const int turn = (share.row % BAND8 * Cols8::R / BAND8) % Cols8::R;
  const int64_t swn = a.swn;
  const int wave_u = (int)wave_uniform_id();
  int nb[2];
  if constexpr (EPI == EPI_UNIT) {
    // tile column -> weight row: first 32 of a wave's 64 from the linear half of the rows, the others from the gate's
    const int lin_at = (a.act & 1) * F, gate_at = F - lin_at;
    B.init((const char*)a.W + e * a.swe + k0 * QB, (int64_t)a.N * swn - k0 * QB, turn, [&](int tc) {
      const int of_wave = ((tc & 12) << 1) + ((tc & 16) >> 2) + (tc & 3);
      return (int64_t)(min(n0 + (tc >> 6) * 32 + of_wave, F - 1) + (tc & 32 ? gate_at : lin_at)) * swn;
    });
    const int hc = min(n0 + wave_u * 32, F - 1);
    nb[0] = (lin_at + hc) / QB, nb[1] = (gate_at + hc) / QB;
  } else {
    const int last = a.N - 1 - n0;
    B.init((const char*)a.W + e * a.swe + n0 * swn + k0 * QB, (a.N - n0) * swn - k0 * QB, turn, [&](int tc) {
      const int of_wave = ((tc & 12) << 2) + ((tc & 48) >> 2) + (tc & 3);
      return (int64_t)min((tc & ~63) + of_wave, last) * swn;
    });
    nb[0] = nb[1] = min(n0 + wave_u * TL::WTN, a.N - 1) / QB;
  }
  WeightScales<SC> W;
  const int WSB = SC == SCALES_BYTES ? 1 : SC == SCALES_FLOAT || a.ws_f32 ? 4 : 1;
#pragma unroll
  for (int h = 0; h < 2; ++h) W.at[h] = (const char*)a.WS + (e * a.sse + nb[h] * a.ssn + k0 * a.ssk) * WSB;
  W.step = a.ssk * WSB;
  W.f32 = a.ws_f32 != 0;
  Block acc[TL::FM][TL::FN];
#pragma unroll
  for (int i = 0; i < TL::FM; ++i)
#pragma unroll
    for (int j = 0; j < TL::FN; ++j) acc[i][j].clear();
  mainloop_8bit<TL, SC>(A, B, W, sx, min(a.K - k0 * QB, share.slices * QB), lds, s_scale, acc);
  if (share.parts > 1) {
    // this part's sums as they lie in the registers (scalar offsets: addresses in registers would have to be held beside them)
    const __amdgpu_buffer_rsrc_t P =
        __builtin_amdgcn_make_buffer_rsrc((void*)make_uniform((const char*)(a.partial + share.slot * TILE8_FLOATS<TL>)), 0, TILE8_FLOATS<TL> * 4, 0x00020000);
    typedef unsigned u32x4_8b __attribute__((ext_vector_type(4)));
    const int at = late_thread<TL>() * 16;
#pragma unroll
    for (int i = 0; i < TL::FM; ++i)
#pragma unroll
      for (int j = 0; j < TL::FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_8b, acc[i][j].q[g]), P, at, ((i * TL::FN + j) * 4 + g) * TL::NT * 16, 0);
    return;
  }
  __syncthreads();
  finish<TL, TO, EPI>(acc, a, bias_dtype, e, row0, rows, n_tile, s_dst, s_bias, lds);
}

// The tiles whose contraction was cut: the parts' sums in their order, and what follows a product
template <typename TO, int SC, int EPI, int BM>
__global__ __launch_bounds__(NT8, 2) void product_8bit_join_kernel(Product8Args a, int bias_dtype, int n_tiles) {
  typedef Tile8<BM> TL;
  __shared__ __attribute__((aligned(16))) char lds[LDS8<TL>];
  __shared__ int64_t s_dst[EPI == EPI_ROWS ? TL::BM : 1];
  __shared__ __attribute__((aligned(16))) float s_bias[TL::BN];
  Share8 share;
  if (!find_share<BM, round_tiles<SC, BM>, true>(a, blockIdx.x, n_tiles, share)) return;
  const int t = threadIdx.x;
  if (EPI == EPI_ROWS && t < TL::BM)
    s_dst[t] = t < share.rows ? (a.y_grouped ? (int64_t)(share.row0 + t) : a.idx[share.row0 + t]) * a.sym : -1;
  Block acc[TL::FM][TL::FN];
#pragma unroll
  for (int i = 0; i < TL::FM; ++i)
#pragma unroll
    for (int j = 0; j < TL::FN; ++j) acc[i][j].clear();
  for (int p = 0; p < share.parts; ++p) {
    const f32x4* P = (const f32x4*)(a.partial + (share.slot + p) * TILE8_FLOATS<TL>) + t;
#pragma unroll
    for (int i = 0; i < TL::FM; ++i)
#pragma unroll
      for (int j = 0; j < TL::FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[i][j].q[g] += P[((i * TL::FN + j) * 4 + g) * TL::NT];
  }
  __syncthreads();
  finish<TL, TO, EPI>(acc, a, bias_dtype, share.e, share.row0, share.rows, share.column, s_dst, s_bias, lds);
}

template <typename TO, int SC, int EPI, int BM>
static int launch_product(const Product8Args& a, int bias_dtype, int n_tiles, hipStream_t st) {
  constexpr int ROUND = round_tiles<SC, BM>;
  // every share of the most tiles that the rows can make, and a round of parts
  const int64_t tiles = max_tiles(a.L, a.E, BM) * n_tiles;
  const int64_t grid = (tiles + ROUND - 1) / ROUND * ROUND + (a.partial ? ROUND : 0);
  if (grid > 0x7fffff00LL) { set_error("product_8bit: grid too large"); return SMOE_ERR_RANGE; }
  product_8bit_kernel<TO, SC, EPI, BM><<<(unsigned)grid, NT8, 0, st>>>(a, bias_dtype, n_tiles);
  if (a.partial) product_8bit_join_kernel<TO, SC, EPI, BM><<<ROUND / 2, NT8, 0, st>>>(a, bias_dtype, n_tiles);
  return launch_status("product_8bit");
}
// Tiles of 64 rows instead of 128: a third workgroup per CU waits for its weights beside two others.  us in tiles of 128 -> 64 at 16, 32, 64, 128
// rows per expert, even and as 1 / rank^0.5: 8 experts, 4096 -> 28672 214 -> 185, 215 -> 187, 220 -> 190, 230 -> 237 and 213 -> 184, 214 -> 184, 219 ->
// 223, 217 -> 248; 128 experts, 2048 -> 1536 80 -> 67, 87 -> 76, 95 -> 86, 106 -> 111 and 79 -> 85, 85 -> 89, 93 -> 104, 119 -> 123; 32 experts,
// 2880 -> 5760 115 -> 104, 120 -> 107, 133 -> 118, 148 -> 162 and 117 -> 106, 117 -> 132, 131 -> 161, 170 -> 180.  What decides is the tile rows that the
// loads make, which the host does not know; by the average, 24 rows lie between the even loads, which gain up to 32 (wide experts up to 64), and
// the uneven ones, of which many small experts lose 6 % at 16.
static bool low_tiles(int64_t L, int E) { return L <= 24 * (int64_t)E; }
template <typename TO, bool EXACT, int EPI>
static int launch_product(const Product8Args& a, int bias_dtype, hipStream_t st) {
  const int n_tiles = EPI == EPI_UNIT ? (a.N / 2 + QB - 1) / QB : (a.N + BN8 - 1) / BN8;
  if constexpr (EXACT) return launch_product<TO, SCALES_EXACT, EPI, 128>(a, bias_dtype, n_tiles, st);
  else if (low_tiles(a.L, a.E)) return a.ws_f32 ? launch_product<TO, SCALES_FLOAT, EPI, 64>(a, bias_dtype, n_tiles, st) : launch_product<TO, SCALES_BYTES, EPI, 64>(a, bias_dtype, n_tiles, st);
  else return a.ws_f32 ? launch_product<TO, SCALES_FLOAT, EPI, 128>(a, bias_dtype, n_tiles, st) : launch_product<TO, SCALES_BYTES, EPI, 128>(a, bias_dtype, n_tiles, st);
}

int64_t product_8bit_floats(int64_t L, int64_t K, int64_t columns, int E, bool exact) {
  const bool low = !exact && low_tiles(L, E);
  const int64_t round = exact ? round_tiles<SCALES_EXACT, 128> : low ? round_tiles<SCALES_BYTES, 64> : round_tiles<SCALES_BYTES, 128>;
  const int64_t tiles = max_tiles(L, E, low ? 64 : 128) * ((columns + BN8 - 1) / BN8);
  if ((K + QB - 1) / QB < SPLIT_SLICES || tiles > SPLIT_ROUNDS * round) return 0;
  const int64_t slots = tiles * PARTS8 < round ? tiles * PARTS8 : round;
  return slots * (low ? TILE8_FLOATS<Tile8<64>> : TILE8_FLOATS<Tile8<128>>);
}

// The unit's blocks are 128 hidden columns, and a wave's 32 of either half have one scale of the weights; its weight rows are
// 32-bit offsets from the expert's first.  Else the product's float32 rows go through a pass of their own.
bool unit_rides(int64_t d, int64_t F) { return F % 32 == 0 && 2 * F * padded_row(d) < (1LL << 31); }
// The gradient's blocks run along both halves: they lie within one half where F is whole blocks.
bool unit_grad_rides(int64_t F) { return F % QB == 0; }

int launch_product_8bit(const Product8Args& a, bool exact, int row_dtype, int out_dtype, hipStream_t st, int epilogue) {
  if (epilogue == EPI_UNIT) return exact ? launch_product<float, true, EPI_UNIT>(a, row_dtype, st) : launch_product<float, false, EPI_UNIT>(a, row_dtype, st);
  if (epilogue == EPI_UNIT_GRAD)
    return exact ? launch_product<float, true, EPI_UNIT_GRAD>(a, row_dtype, st) : launch_product<float, false, EPI_UNIT_GRAD>(a, row_dtype, st);
  if (exact) return launch_product<float, true, EPI_ROWS>(a, row_dtype, st);
  if (out_dtype == SMOE_F32) return launch_product<float, false, EPI_ROWS>(a, row_dtype, st);
  if (out_dtype == SMOE_BF16) return launch_product<bf16_t, false, EPI_ROWS>(a, row_dtype, st);
  return launch_product<f16_t, false, EPI_ROWS>(a, row_dtype, st);
}

}  // namespace smoe
