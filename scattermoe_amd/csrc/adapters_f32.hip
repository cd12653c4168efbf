// The projection beside low-rank adapters for many rows, float32: Y = X W^T (+ bias) + U B[a]^T in tiles on the float32 matrix
// instructions (16 x 16 x 4), operands through LDS.
//
// A workgroup of four waves has BM x BN outputs, each wave a quarter.  Operands whose contraction is contiguous lie in LDS as [row][k]: the order
// in which a contraction's elements meet is free as long as both operands share it, so a lane's 16 bytes are its operand
// of four instructions.  A weight that is taken transposed (DX) lies as [k][column], as in memory: a lane's 16
// bytes are its operand of one element and four blocks of columns, lane l's next to each other.
// The rows are taken in the order of their adapters: in the epilogue a lane has one column and walks its rows, B[a] of
// its column in registers while the adapter lasts.
//
// Bound by the matrix unit: a slice of 32 takes a 128 x 128 tile 4400 clocks, 4096 of them products; what kept it at 5300 was memory instructions
// in a row (LDS takes 8 clocks for each of a wave's and the products stand behind them), not their latency.  us of a call with u and the
// ordering of the rows (about 20): 1024 rows, 4096 -> 4096 273 (the product at 140 TFLOP/s; a large library one reaches 151), 4096 rows 992,
// 1024 rows, 1024 -> 4096 91, 256 rows, 4096 -> 4096 95 (one round of 64 x 64 tiles, a third more than the chain of their products).
#include "few_rows.hpp"
#include <algorithm>

namespace smoe {

typedef float f32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));

static constexpr int TF_K = 32, TF_NT = 256, TF_LDK = TF_K + 4, TF_RANKS = 16, TF_LDU = TF_RANKS + 4;

// What a thread carries of an operand's slice from memory to LDS: ROWS rows of TF_K elements in pieces of 16 bytes
template <int ROWS>
struct SliceRows {
  static constexpr int N = ROWS * TF_K / 4 / TF_NT;
  const float* p[N];
  f32x4 v[2][N];
  template <class Row>
  __device__ __forceinline__ void init(Row row) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = row(i * (TF_NT / 8) + (threadIdx.x >> 3)) + (threadIdx.x & 7) * 4;
  }
  __device__ __forceinline__ void load(int k0, f32x4 (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = *(const f32x4_by4*)(p[i] + k0);
  }
  __device__ __forceinline__ void load_rest(int k0, int K, f32x4 (&v)[N]) const {
    const int k = k0 + (threadIdx.x & 7) * 4;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][e] = 0.0f;
        if (k + e < K) v[i][e] = p[i][k0 + e];
      }
  }
  __device__ __forceinline__ void store(float* s, const f32x4 (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) *(f32x4*)(s + (i * (TF_NT / 8) + (threadIdx.x >> 3)) * TF_LDK + (threadIdx.x & 7) * 4) = v[i];
  }
};
// ... TF_K rows of COLS elements, the contraction from row to row
template <int COLS>
struct SliceColumns {
  static constexpr int N = COLS * TF_K / 4 / TF_NT, PER_ROW = COLS / 4, LD = COLS + 4;
  const float* p;
  int64_t ld;
  f32x4 v[2][N];
  int shift;
  // `columns` from the first one to the last; there are four and more in all.  A piece over the last column, or beyond it, is the one
  // that ends with it, and `shift` elements in front of its own.
  __device__ __forceinline__ void init(const float* first, int64_t ld_, int columns) {
    const int c = (threadIdx.x % PER_ROW) * 4;
    ld = ld_;
    shift = max(c - (columns - 4), 0);
    p = first + (c - shift);
  }
  static __device__ __forceinline__ int row(int i) { return i * (TF_NT / PER_ROW) + threadIdx.x / PER_ROW; }
  __device__ __forceinline__ void load(int k0, f32x4 (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = *(const f32x4_by4*)(p + (k0 + row(i)) * ld);
  }
  __device__ __forceinline__ void load_rest(int k0, int K, f32x4 (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (k0 + row(i) < K) v[i] = *(const f32x4_by4*)(p + (k0 + row(i)) * ld);
    }
  }
  __device__ __forceinline__ void store(float* s, const f32x4 (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f32x4 u = v[i];
      if (shift > 0) u = f32x4{shift == 1 ? u[1] : shift == 2 ? u[2] : u[3], shift == 1 ? u[2] : u[3], u[3], u[3]};
      *(f32x4*)(s + row(i) * LD + (threadIdx.x % PER_ROW) * 4) = u;
    }
  }
};

template <int BM, int BN, bool W_TR>
__global__ __launch_bounds__(TF_NT, 2) void adapter_tiles_f32_kernel(AdapterProjectArgs a, int m_tiles, int n_tiles) {
  constexpr int FM = BM / 32, FN = BN / 32;                  // blocks of 16 x 16 of a wave
  typedef SliceRows<BM> SliceA;
  typedef typename std::conditional<W_TR, SliceColumns<BN>, SliceRows<BN>>::type SliceB;
  constexpr int SIZE_A = BM * TF_LDK, SIZE_B = W_TR ? TF_K * SliceColumns<BN>::LD : BN * TF_LDK;
  static_assert(BM * TF_LDU <= 2 * (SIZE_A + SIZE_B), "U fits the operands' buffers");
  __shared__ __attribute__((aligned(16))) float lds[2 * (SIZE_A + SIZE_B)];
  __shared__ int64_t sRow[BM];
  __shared__ int sAdapter[BM];

  // an XCD takes a run of tiles, rows fastest: its columns of W are read from memory once
  const int64_t all = (int64_t)m_tiles * n_tiles, per = (all + 7) / 8;
  const int64_t tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || tile >= all) return;
  const int64_t m0 = tile % m_tiles * BM;
  const int n0 = (int)(tile / m_tiles) * BN;
  for (int m = threadIdx.x; m < BM; m += TF_NT) {
    const int64_t i = m0 + m, t = a.idx[std::min(i, a.T - 1)], id = a.ids[t];
    sRow[m] = i < a.T ? t : -1 - t;
    sAdapter[m] = i < a.T && (uint64_t)id < (uint64_t)a.R ? (int)id : -1;
  }
  __syncthreads();

  const int lane = lane_id(), quad = lane >> 4, lr = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  SliceA A;
  SliceB B;
  A.init([&](int m) { const int64_t t = sRow[m]; return (const float*)a.X + (t < 0 ? -1 - t : t) * a.sxm; });
  if constexpr (W_TR) B.init((const float*)a.W + n0, a.swk, a.N - n0);
  else B.init([&](int n) { return (const float*)a.W + std::min(n0 + n, a.N - 1) * a.swn; });
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // Whole slices through two buffers of LDS, each in two blocks of 16, which are read a block ahead of their products.  Once the second
  // one is read no wave needs this buffer any more and the other is whole: the one barrier, with the second block's products still to
  // come.  Slices on their way from memory have two register sets, so that each has the time of two slices' products.  (No conditions
  // inside: a load that may not have been made costs the waits their precision.  What is loaded behind the last slice is that one
  // again, unread.)
  typedef float Columns __attribute__((ext_vector_type(FN)));
  f32x4 x[2][FM], w[2][FN];
  auto fetch = [&](const float* buf, int c) {
    const float* sa = buf + (wm * (BM / 2) + lr) * TF_LDK + 16 * c + 4 * quad;
#pragma unroll
    for (int i = 0; i < FM; ++i) x[c][i] = *(const f32x4*)(sa + i * 16 * TF_LDK);
    if constexpr (W_TR) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Columns n = *(const Columns*)(buf + SIZE_A + (16 * c + 4 * quad + e) * SliceColumns<BN>::LD + wn * (BN / 2) + lr * FN);
#pragma unroll
        for (int j = 0; j < FN; ++j) w[c][j][e] = n[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < FN; ++j) w[c][j] = *(const f32x4*)(buf + SIZE_A + (wn * (BN / 2) + j * 16 + lr) * TF_LDK + 16 * c + 4 * quad);
    }
  };
  auto products = [&](int c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[c][i][e], w[c][j][e], acc[i][j], 0, 0, 0);
  };
  auto store = [&](float* buf, auto set) { A.store(buf, A.v[set]), B.store(buf + SIZE_A, B.v[set]); };
  const int whole = a.K / TF_K;
  auto load = [&](int s, auto set) { A.load(min(s, whole - 1) * TF_K, A.v[set]), B.load(min(s, whole - 1) * TF_K, B.v[set]); };
  auto slice = [&](int s, auto odd) {
    constexpr int ODD = decltype(odd)::value;
    constexpr std::integral_constant<int, 1 - ODD> set{};
    float* cur = lds + ODD * (SIZE_A + SIZE_B);
    float* other = lds + (1 - ODD) * (SIZE_A + SIZE_B);
    // (a memory instruction behind every few products: a row of them would hold the products up, as LDS takes 8 clocks for each)
    constexpr int PRODUCTS = 4 * FM * FN, READS = FM + (W_TR ? 4 : FN), LOADS = SliceA::N + SliceB::N, WRITES = LOADS;
    constexpr int EACH0 = std::max(1, PRODUCTS / (READS + WRITES + LOADS)), EACH1 = std::max(1, PRODUCTS / READS);
    __builtin_amdgcn_sched_barrier(0);
    fetch(cur, 1);
    store(other, set);
    load(s + 3, set);
    products(0);
#pragma unroll
    for (int n = 0; n < READS; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, EACH0, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int n = 0; n < WRITES; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, EACH0, 0);
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
    }
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, EACH0, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    fetch(other, 0);
    products(1);
#pragma unroll
    for (int n = 0; n < READS; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x008, EACH1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  if (whole > 0) {
    load(0, even);
    store(lds, even);
    load(1, odd);
    load(2, even);
    __syncthreads();
    fetch(lds, 0);
#pragma unroll 1
    for (int s = 0;; s += 2) {
      slice(s, even);
      if (s + 1 >= whole) break;
      slice(s + 1, odd);
      if (s + 2 >= whole) break;
    }
    __syncthreads();
  }
  if (whole * TF_K < a.K) {                                  // the rest, with zeros behind it
    A.load_rest(whole * TF_K, a.K, A.v[0]);
    B.load_rest(whole * TF_K, a.K, B.v[0]);
    store(lds, even);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < TF_K / 16; ++c) {
      fetch(lds, c);
      products(c);
    }
    __syncthreads();
  }

  // register e of a lane: row 4 (lane / 16) + e and, of block j, column 16 j + lane % 16 (W_TR: FN (lane % 16) + j) of the wave's
  auto row_of = [&](int i, int e) { return wm * (BM / 2) + i * 16 + quad * 4 + e; };
  int column[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) column[j] = n0 + wn * (BN / 2) + (W_TR ? lr * FN + j : j * 16 + lr);
  for (int q0 = 0; q0 < a.r; q0 += TF_RANKS) {
    if (q0) __syncthreads();
    for (int p = threadIdx.x; p < BM * TF_RANKS; p += TF_NT) {
      const int m = p / TF_RANKS, q = q0 + p % TF_RANKS;
      lds[m * TF_LDU + p % TF_RANKS] = q < a.r && sAdapter[m] >= 0 ? a.U[sRow[m] * a.r + q] : 0.0f;
    }
    __syncthreads();
    float b[FN][TF_RANKS];
    int at = -1;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = row_of(i, e), id = sAdapter[m];
        if (id >= 0 && id != at) {
          at = id;
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const float* from = (const float*)a.B + (int64_t)id * a.sbr + std::min(column[j], a.N - 1) * a.sbn + q0 * a.sbj;
            if (a.sbj == 1 && q0 + TF_RANKS <= a.r) {
#pragma unroll
              for (int q = 0; q < TF_RANKS; q += 4) *(f32x4*)&b[j][q] = *(const f32x4_by4*)(from + q);
            } else {
#pragma unroll
              for (int q = 0; q < TF_RANKS; ++q) {
                b[j][q] = 0.0f;
                if (q0 + q < a.r) b[j][q] = from[q * a.sbj];
              }
            }
          }
        }
        if (id >= 0) {
          float u[TF_RANKS];
#pragma unroll
          for (int q = 0; q < TF_RANKS; q += 4) *(f32x4*)&u[q] = *(const f32x4*)(lds + m * TF_LDU + q);
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            float v = acc[i][j][e];
#pragma unroll
            for (int q = 0; q < TF_RANKS; ++q) v = fmaf(u[q], b[j][q], v);
            acc[i][j][e] = v;
          }
        }
      }
  }
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    if (column[j] >= a.N) continue;
    const float bias = a.bias ? ((const float*)a.bias)[column[j] * a.sb] : 0.0f;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = sRow[row_of(i, e)];
        if (t >= 0) ((float*)a.Y)[t * a.sym + column[j]] = acc[i][j][e] + bias;
      }
  }
}

template <int SIDE>
static int launch_tiles_f32(const AdapterProjectArgs& a, hipStream_t st) {
  const int64_t m_tiles = cdiv64(a.T, SIDE), n_tiles = cdiv64(a.N, SIDE), grid = cdiv64(m_tiles * n_tiles, 8) * 8;
  if (grid > 0x7fffffffLL) { set_error("adapters: too many rows and columns for one launch"); return SMOE_ERR_RANGE; }
  if (a.swk == 1) hipLaunchKernelGGL((adapter_tiles_f32_kernel<SIDE, SIDE, false>), dim3((unsigned)grid), dim3(TF_NT), 0, st, a, (int)m_tiles, (int)n_tiles);
  else hipLaunchKernelGGL((adapter_tiles_f32_kernel<SIDE, SIDE, true>), dim3((unsigned)grid), dim3(TF_NT), 0, st, a, (int)m_tiles, (int)n_tiles);
  return launch_status("adapter_tiles_f32_kernel");
}

static int64_t tiles_f32(int64_t T, int64_t N, int64_t side) { return cdiv64(T, side) * cdiv64(N, side); }
static constexpr int TF_CUS = 256;
// Whether a product goes in these tiles, `strided` a weight whose contraction is.  Each of them is a chain of K products, TF_CUS of them side by
// side; the rows' kernel (project_t in adapters.hip) has work for the whole chip from few rows on, at 66 TFLOP/s, and a weight to copy
// first where its contraction is strided.  us of a call, rows' kernel / tiles, forward and gradient of the input: 65 rows, 4096 -> 4096
// 81 / 90 and 108 / 101; 128 86 / 93 and 113 / 101; 256 147 / 95 and 179 / 103; 256, 2048 -> 2048 51 / 56 and 62 / 63; 512 83 / 58 and 96 / 65; 1024,
// 512 -> 512 23 / 27 and 25 / 29; 1024, 1003 -> 1517 69 / 56 and 77 / 57; 203 30 / 36 and 34 / 50; 1024, 4096 -> 4096 513 / 273 and 572 / 295.
bool adapter_takes_tiles_f32(int64_t T, int64_t K, int64_t N, bool strided) {
  if (T <= ADAPTER_FEW_ROWS || N < 4) return false;
  return (double)(T + (strided ? 53 : 0)) * N * K > 617e3 * cdiv64(tiles_f32(T, N, 64), TF_CUS) * (K + 160);
}
// 128 x 128 where they fill their rounds of workgroups: their operands go twice as far (us of a call, 128 x 128 / 64 x 64: 1024 rows, 4096 ->
// 4096, 256 tiles 273 / 280; 4096 rows 992 / 1073; 128 tiles, 1024 rows, 2048 -> 2048 151 / 88; 64 x 128 and 128 x 64 between the two).
int launch_adapter_tiles_f32(const AdapterProjectArgs& a, hipStream_t st) {
  return cdiv64(tiles_f32(a.T, a.N, 128), TF_CUS) * 4 * 15 <= cdiv64(tiles_f32(a.T, a.N, 64), TF_CUS) * 16 ? launch_tiles_f32<128>(a, st) : launch_tiles_f32<64>(a, st);
}

}  // namespace smoe
