// The projection beside low-rank adapters for many rows, bf16 / fp16: Y = X W^T (+ bias) + U B[a]^T in tiles of the matrix-core
// kernels (main loops, operands and epilogues of gemm_mfma.hpp).
//
// The rows are taken in the order of their adapters, each adapter's padded to a whole number of 16: a fragment of 16 rows then has
// one adapter, so its U B^T is a product of whole fragments, and what another request's adapter holds, infinities included, never meets
// its rows.  A tile spans as many adapters as it has fragments: the shared product does not care, and no tile is cut short
// where an adapter ends.  The accumulators start with U B^T and the main loop adds X W^T to them: one rounding.  U comes in two
// parts of 16 bits (2^-18 of its value; one part would cost as much as the output's own rounding; float16 parts times a power of
// two of their row where float16 would not hold them, PLANES_TOP, 81 us of a product instead of 80), operands straight from
// global memory: for rank 16, 80 loads of 1 KB and 128 products per wave and 256 x 256 tile, against 64 slices of 128
// products for K = 4096.
//
// Bound by the matrix cores where rounds are full: 8192 rows, 4096 -> 4096, rank 16 231 us forward and 236 on the transposed weight
// (1.19 PFLOP/s; a large library product reaches 1.40).  4099 rows, 2880 -> 2880 78 us (0.88): 204 tiles leave a fifth of the CUs
// idle.  1777 rows, 2048 -> 4096, rank 64 40.5 us (0.74): 128 x 128 tiles read their operands from the L2s more often, and U B^T
// takes a tenth of the time (tiles of 256 x 128 with one wave per SIMD, one round: slower at 15 of 16 sizes, up to 45 %, and 2 % faster
// at the other).
#include "gemm_mfma.hpp"

namespace smoe {

struct AdapterTiles {
  AdapterProjectArgs p;
  Raster rast;
  int64_t fragments, first;                          // all, the launch's first
};

// Tile classes: 0 one wave per SIMD (long contractions of whole slices), 1 eight waves, 2 tiles of 128 x 128 and 3 of 64 x 128, two
// workgroups per CU
template <int CLASS> struct AdapterTile;
template <> struct AdapterTile<0> { typedef Tile<256, 256, 2, 2, 2, true> type; };
template <> struct AdapterTile<1> { typedef Tile<256, 256, 2, 4> type; };
template <> struct AdapterTile<3> { typedef Tile<64, 128, 2, 2, 3, false, 2> type; };
template <> struct AdapterTile<2> { typedef Tile<128, 128, 2, 2, 2, false, 2> type; };

// Eight values of a float16 plane from their block's power of two to the row's, 2^down <= 1 of it (what that leaves below float16 is
// at most 2^-22 of the row's largest).  In two halves: the values begin at 2^15, so that 2^down itself may lie below float16's smallest.
template <typename T>
__device__ __forceinline__ i32x4 planes_times(i32x4 u, int down) {
  typedef T v8 __attribute__((ext_vector_type(8)));
  const int all = max(down, -48), half = all / 2;
  return __builtin_bit_cast(i32x4, __builtin_bit_cast(v8, u) * (T)ldexpf(1.0f, half) * (T)ldexpf(1.0f, all - half));
}

template <typename T, int CLASS, bool W_TR>
__global__ __launch_bounds__(AdapterTile<CLASS>::type::NT, AdapterTile<CLASS>::type::WAVES_PER_SIMD) void adapter_tiles_kernel(AdapterTiles args) {
  typedef typename AdapterTile<CLASS>::type TL;
  typedef DirectOp<TL::BM, TL::NT> AOp;
  typedef typename std::conditional<W_TR, TransOp<TL::BN, TL::NT, false, false, TL::RS>, DirectOp<TL::BN, TL::NT>>::type BOp;
  constexpr int STAGE = (TL::BM + TL::BN) * 128, FRAGS = TL::BM / 16;
  static_assert(TL::BM * TL::BN * 2 <= TL::NS * STAGE, "staged tile must fit the operand buffers");
  __shared__ __attribute__((aligned(16))) char lds[TL::NS * STAGE];
  __shared__ int64_t sDst[TL::BM];
  constexpr bool SCALED = std::is_same<T, f16_t>::value;      // planes of powers of two (PLANES_TOP)
  __shared__ int sSrc[TL::BM], sAdapter[FRAGS], sExponent[SCALED ? TL::BM : 1];
  __shared__ __attribute__((aligned(16))) float sBias[TL::RS ? TL::BN : 4];
  const AdapterProjectArgs& a = args.p;
  int m_tile, n_tile, m_loc, n_loc;
  if (!args.rast.map(blockIdx.x, m_tile, n_tile, m_loc, n_loc)) return;
  const int n0 = n_tile * TL::BN, lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // rows of the tile's fragments; one behind the last row repeats the fragment's first, or any
  const int64_t fragments = args.fragments, f0 = args.first + (int64_t)m_tile * FRAGS;
  bool any = false, scaled = false;                          // some row of the tile, some plane not as it is
  for (int m = threadIdx.x; m < TL::BM; m += TL::NT) {
    const int64_t f = f0 + (m >> 4);
    const int* s = a.slots + f * 17;
    const int t = f < fragments ? s[m & 15] : -1, first = f < fragments ? s[0] : -1;
    any |= first >= 0;
    sSrc[m] = t >= 0 ? t : max(first, 0);
    sDst[m] = t >= 0 ? (int64_t)t * a.sym : -1;
    if ((m & 15) == 0) sAdapter[m >> 4] = f < fragments ? s[16] : -1;
    if constexpr (SCALED) {                                  // the row's: the largest of its blocks'
      int e = PLANES_NONE;
      const int* of = a.exponents + (f * 16 + (m & 15)) * (a.rp / 16);
      for (int b = 0; b < a.rp / 16 && f < fragments; ++b) {
        const int block = of[b];
        e = max(e, block);
        scaled |= block != 0 && block != PLANES_NONE;
      }
      sExponent[m] = e == PLANES_NONE ? 0 : e;
    }
  }
  if (!__syncthreads_or(any)) return;
  if constexpr (SCALED) scaled = __syncthreads_or(scaled);

  const int wm = wave / TL::WN, wn = wave % TL::WN, lr = lane & 15, lq = lane >> 4;
  Block acc[TL::FM][TL::FN];
  float rs[2 * TL::FM];
#pragma unroll
  for (int i = 0; i < TL::FM; ++i)
#pragma unroll
    for (int j = 0; j < TL::FN; ++j) acc[i][j].clear();
  for (int k0 = 0; k0 < a.rp; k0 += 32) {
    const int k = k0 + 8 * lq;
    const bool inside = k < a.r;                             // (rows of B end with a whole piece, those of U with a whole step, in zeros)
    // (a fragment's operands are on their way while the one before is multiplied; B of an adapter that goes on from there stays:
    // us of a call, rank 64, eight adapters, 1777 rows 2048 -> 4096 59.7 -> 55.5, 4096 rows 4096 -> 4096 186 -> 178)
    auto same = [&](int i) {
      const int f = (wm * TL::WTM >> 4) + i;
      return i > 0 && __builtin_amdgcn_readfirstlane(sAdapter[f]) == __builtin_amdgcn_readfirstlane(sAdapter[max(f - 1, 0)]);
    };
    i32x4 u[2][2], bv[2][2 * TL::FN];
    int down[2];
    auto load = [&](int i, int p) {
      const int row = wm * TL::WTM + 16 * i;
      const int id = __builtin_amdgcn_readfirstlane(sAdapter[row >> 4]);
      int src = sSrc[row + lr];
      if constexpr (SCALED && TL::RS) asm volatile("" : "+v"(src));      // (addresses of all fragments, kept, would be spilled)
      const T* x = (const T*)a.planes + (int64_t)src * 2 * a.rp + k;
      u[p][0] = *(const i32x4*)x;
      u[p][1] = *(const i32x4*)(x + a.rp);
      if (SCALED && scaled)
        down[p] = a.exponents[(min(f0 + (row >> 4), fragments - 1) * 16 + lr) * (a.rp / 16) + (k >> 4)] - sExponent[row + lr];
      if (same(i)) return;
      const T* b = (const T*)a.B + (int64_t)max(id, 0) * a.sbr + (inside ? k : 0);
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j) bv[p][j] = *(const i32x4*)(b + (int64_t)min(n0 + wn * TL::WTN + 16 * j + lr, a.N - 1) * a.sbn);
    };
    load(0, 0);
#pragma unroll
    for (int i = 0; i < 2 * TL::FM; ++i) {
      if (same(i)) {
#pragma unroll
        for (int j = 0; j < 2 * TL::FN; ++j) bv[i & 1][j] = bv[(i & 1) ^ 1][j];
      }
      if (i + 1 < 2 * TL::FM) load(i + 1, (i + 1) & 1);
      __builtin_amdgcn_sched_barrier(0);
      const bool none = !inside || sAdapter[(wm * TL::WTM >> 4) + i] < 0;
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j)
        if (none) bv[i & 1][j] = i32x4{0, 0, 0, 0};
      if (SCALED && scaled) {
#pragma unroll
        for (int h = 0; h < 2; ++h) u[i & 1][h] = planes_times<T>(u[i & 1][h], down[i & 1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2 * TL::FN; ++j) {
          f32x4& c = acc[i >> 1][j >> 1].q[2 * (i & 1) + (j & 1)];
          c = Mfma<T>::run(bv[i & 1][j], u[i & 1][h], c);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (SCALED && scaled) {                                    // (a lane's accumulators of a fragment are of one row)
#pragma unroll
    for (int i = 0; i < 2 * TL::FM; ++i) {
      const float back = ldexpf(1.0f, sExponent[wm * TL::WTM + 16 * i + lr]);
#pragma unroll
      for (int j = 0; j < 2 * TL::FN; ++j) {
        f32x4& c = acc[i >> 1][j >> 1].q[2 * (i & 1) + (j & 1)];
        if constexpr (TL::RS) asm volatile("" : "+a"(c));
        c *= back;
        // (back to the matrix unit's own registers at once: all of them together would not fit the vector unit's)
        if constexpr (TL::RS) asm volatile("" : "+a"(c));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  AOp A;
  A.rot = TL::RS ? 0 : (n_loc * AOp::R / Raster::SN) % AOp::R;
  A.init((const char*)a.X, [&](int row) { return (int64_t)sSrc[row] * a.sxm * 2; });
  BOp B;
  B.rot = TL::RS ? 0 : (m_loc * BOp::R / Raster::SM) % BOp::R;
  if constexpr (W_TR) B.init((const char*)a.W + (int64_t)n0 * 2, a.swk * 2, a.N - n0);
  else B.init((const char*)a.W, [&](int row) { return (int64_t)min(n0 + row, a.N - 1) * a.swn * 2; });
  if constexpr (TL::RS) mainloop_rs<T, TL, AOp, BOp>(A, B, a.K, lds, acc);
  else if constexpr (TL::NS > 2) mainloop_ring<T, TL, AOp, BOp>(A, B, a.K, lds, acc);
  else mainloop<T, TL, AOp, BOp, false>(A, B, a.K, lds, false, acc, rs);

  __syncthreads();
  const T* bias = (const T*)a.bias;
  if constexpr (TL::RS) {
    stage_accumulators<T, TL>(acc, lds, [&](int tc) { return plain_bias<T>(bias, a.sb, a.N, n0 + tc); }, sBias);
    epilogue_staged<T, TL>(acc, (T*)a.Y, sDst, n0, a.N, bias, a.sb, lds);
  } else {
    if (((uintptr_t)a.Y & 15) == 0 && ((a.sym | a.N) & 7) == 0) epilogue_staged<T, TL>(acc, (T*)a.Y, sDst, n0, a.N, bias, a.sb, lds);
    else epilogue<T, TL>(acc, (T*)a.Y, sDst, n0, a.N, bias, a.sb);
  }
}

// Super tiles share operands best; but an XCD takes whole ones, and where one is left over it runs a round of its own: column
// stripes then, if they make fewer rounds of `wgs` workgroups per CU (4099 rows, 24 adapters, 2880 -> 2880, nine super tiles: 139 -> 78
// us).
static Raster tile_order(int64_t m_tiles, int n_tiles, int wgs) {
  const Raster supers = make_raster(m_tiles, n_tiles, GM_S2S);
  const int64_t round = NUM_CU / 8 * wgs, super = Raster::SM * Raster::SN;
  const int64_t by_supers = cdiv64(cdiv64(supers.supers, 8) * super, round);
  const int64_t by_stripes = cdiv64(cdiv64(m_tiles / GM_RING * n_tiles, 8) * GM_RING + cdiv64(n_tiles, 8) * (m_tiles % GM_RING), round);
  return by_stripes < by_supers ? make_striped(m_tiles, n_tiles, GM_RING) : supers;
}

// Fragments [first, last) in tiles of a class
template <typename T, int CLASS>
static int launch_tiles(const AdapterProjectArgs& a, bool w_tr, int64_t first, int64_t last, hipStream_t st) {
  typedef typename AdapterTile<CLASS>::type TL;
  const int64_t m_tiles = cdiv64(last - first, TL::BM / 16);
  const int n_tiles = (a.N + TL::BN - 1) / TL::BN;
  AdapterTiles args{a, tile_order(m_tiles, n_tiles, TL::WG), last, first};
  const int64_t grid = args.rast.grid();
  if (grid > 0x7fffffffLL) { set_error("adapters: grid too large"); return SMOE_ERR_RANGE; }
  if (w_tr) hipLaunchKernelGGL((adapter_tiles_kernel<T, CLASS, true>), dim3((unsigned)grid), dim3(TL::NT), 0, st, args);
  else hipLaunchKernelGGL((adapter_tiles_kernel<T, CLASS, false>), dim3((unsigned)grid), dim3(TL::NT), 0, st, args);
  return launch_status("adapter_tiles_kernel");
}

// Below two thirds of a round of 256 x 256 tiles: smaller ones, 64 x 128 while 128 x 128 ones would leave CUs without a tile.  us of
// a whole call, 128 x 128 / 64 x 128, T rows K -> N: 256, 4096 -> 4096 56 / 43; 512, 4096 -> 4096 58 / 52; 777, 2880 -> 2880 47 / 42;
// 1000, 4096 -> 1024 58 / 45; 1024, 4096 -> 4096 69 / 83; 1777, 2048 -> 4096 49 / 64 (256 x 128 tiles 56).
static constexpr int SMALL_MIN_TILES = 200;
template <typename T>
static int launch_small(const AdapterProjectArgs& a, bool w_tr, int64_t first, int64_t last, hipStream_t st) {
  return cdiv64(last - first, 8) * cdiv64(a.N, 128) < SMALL_MIN_TILES ? launch_tiles<T, 3>(a, w_tr, first, last, st)
                                                                      : launch_tiles<T, 2>(a, w_tr, first, last, st);
}

template <typename T>
static int dispatch_tiles(const AdapterProjectArgs& a, bool w_tr, hipStream_t st) {
  const int64_t fragments = adapter_fragments(a.T, a.R), rows = cdiv64(fragments, 16), columns = cdiv64(a.N, 256), tiles = rows * columns;
  if (cdiv64(a.T, 256) * columns < MAIN_MIN_TILES) return launch_small<T>(a, w_tr, 0, fragments, st);
  // Whole rounds of 256 x 256 tiles; what is left, up to half a round, would take as long as a round (4096 rows and eight adapters'
  // padding, 4096 -> 4096, a call: 204 -> 158 us): tile rows of a launch of their own, in smaller tiles.  A tile row of more than a
  // round stays as it is (100 rows, 4096 -> 151936, 594 tiles: 370 us, all in smaller ones 424; 66 rows 365 and 331).
  const int64_t whole = tiles / NUM_CU * NUM_CU;
  const int64_t main = whole >= columns && tiles - whole <= NUM_CU / 2 ? std::min(fragments, whole / columns * 16) : fragments;
  const bool slices = a.K % BK == 0 && ((uintptr_t)a.Y & 15) == 0 && ((a.sym | a.N) & 7) == 0;
  // (the descriptors of a strided operand end with its last row: rows must not overlap)
  const int rc = a.K >= RS_MIN_K && slices && (!w_tr || a.swk >= a.N) ? launch_tiles<T, 0>(a, w_tr, 0, main, st)
                                                                      : launch_tiles<T, 1>(a, w_tr, 0, main, st);
  return rc || main == fragments ? rc : launch_small<T>(a, w_tr, main, fragments, st);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// Whole pieces of 16 bytes in all operands (rows of B padded with zeros to them), and lane offsets of 32 bits into X and W
bool try_adapter_tiles(const AdapterProjectArgs& a, int dtype, hipStream_t st, int& rc) {
  if ((dtype != SMOE_BF16 && dtype != SMOE_F16) || a.planes == nullptr || a.slots == nullptr) return false;
  if (a.K < 8 || a.K % 8 != 0 || a.sxm % 8 != 0 || !aligned16(a.X) || !aligned16(a.W)) return false;
  if (a.sbn < (a.r + 7) / 8 * 8 || a.sbj != 1 || a.sbn % 8 != 0 || a.sbr % 8 != 0 || !aligned16(a.B) || a.rp % 32 != 0 || !aligned16(a.planes)) return false;
  bool w_tr;
  if (a.swk == 1 && a.swn % 8 == 0) w_tr = false;
  else if (a.swn == 1 && a.swk % 8 == 0 && a.N % 8 == 0) w_tr = true;
  else return false;
  const int64_t most = 0xffffffffLL;
  if ((a.T - 1) * a.sxm * 2 + (int64_t)a.K * 2 > most) return false;
  if (w_tr ? BK * a.swk * 2 + (int64_t)a.N * 2 > most : (a.N - 1) * a.swn * 2 + (int64_t)a.K * 2 > most) return false;
  rc = dtype == SMOE_BF16 ? dispatch_tiles<bf16_t>(a, w_tr, st) : dispatch_tiles<f16_t>(a, w_tr, st);
  return true;
}

}  // namespace smoe
