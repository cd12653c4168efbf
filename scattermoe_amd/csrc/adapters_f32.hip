// The projection beside low-rank adapters for many rows, float32: Y = X W^T (+ bias) + U B[a]^T in tiles on the float32 matrix
// instructions (16 x 16 x 4), operands through LDS.
//
// A workgroup of four waves has BM x BN outputs, each wave a quarter.  Operands whose contraction is contiguous lie in LDS as [row][k]: the order
// in which a contraction's elements meet is free as long as both operands share it, so a lane's 16 bytes are its operand
// of four instructions.  A weight that is taken transposed (DX) lies as [k][column], as in memory: a lane's 16
// bytes are its operand of one element and four blocks of columns, lane l's next to each other.
// The rows are taken in the order of their adapters; U B[a]^T is products of 16 x 16 blocks like the others.
//
// Bound by the matrix unit: a slice of 32 takes a 128 x 128 tile 4400 clocks, 4096 of them products; what kept it at 5300 was memory instructions
// in a row (LDS takes 8 clocks for each of a wave's and the products stand behind them), not their latency.  us of a call with u and the
// ordering of the rows (about 13): 1024 rows, 4096 -> 4096 269 (the product at 140 TFLOP/s; a large library one reaches 151), 4096 rows 990,
// 1024 rows, 1024 -> 4096 89, 256 rows, 4096 -> 4096 90, 65 rows 57.
#include "few_rows.hpp"
#include <algorithm>

namespace smoe {

typedef float f32x4_by4 __attribute__((ext_vector_type(4), aligned(4)));

static constexpr int TF_CUS = 256, TF_K = 32, TF_NT = 256, TF_LDK = TF_K + 4;

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

// A tile of SIDE x SIDE outputs by four waves, each a quarter in blocks of 16 x 16
template <int SIDE, bool W_TR>
struct TileF32 {
  static constexpr int F = SIDE / 32;
  typedef SliceRows<SIDE> SliceA;
  typedef typename std::conditional<W_TR, SliceColumns<SIDE>, SliceRows<SIDE>>::type SliceB;
  static constexpr int SIZE_A = SIDE * TF_LDK, SIZE_B = W_TR ? TF_K * SliceColumns<SIDE>::LD : SIDE * TF_LDK;
  struct Shared {
    float lds[2 * (SIZE_A + SIZE_B)];
    int64_t row[SIDE];                               // the row's place, -1 less it behind the last row
    int adapter[SIDE];                               // or -1
  };
  typedef float Columns __attribute__((ext_vector_type(F)));
  typedef float ColumnsBy4 __attribute__((ext_vector_type(F), aligned(4)));
  f32x4 acc[F][F];
  int quad, lr, wm, wn, n0;

  // rows m0 and up, in the order of their adapters
  __device__ __forceinline__ void start(const AdapterProjectArgs& a, Shared& s, int64_t m0, int n0_) {
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    quad = lane >> 4, lr = lane & 15, wm = wave >> 1, wn = wave & 1, n0 = n0_;
    static_assert(SIDE <= TF_NT, "a thread per row");
    if (threadIdx.x < SIDE) {
      const int m = threadIdx.x;
      const int64_t i = m0 + m, t = a.idx[std::min(i, a.T - 1)], id = a.ids[t];
      s.row[m] = i < a.T ? t : -1 - t;
      s.adapter[m] = i < a.T && (uint64_t)id < (uint64_t)a.R ? (int)id : -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // acc += X W^T over slices [first, last) of TF_K of the contraction, of which the last one may be a part
  __device__ __forceinline__ void multiply(const AdapterProjectArgs& a, Shared& sh, int first, int last) {
    float* lds = sh.lds;
    SliceA A;
    SliceB B;
    A.init([&](int m) { const int64_t t = sh.row[m]; return (const float*)a.X + (t < 0 ? -1 - t : t) * a.sxm; });
    if constexpr (W_TR) B.init((const float*)a.W + n0, a.swk, a.N - n0);
    else B.init([&](int n) { return (const float*)a.W + std::min(n0 + n, a.N - 1) * a.swn; });
    // Whole slices through two buffers of LDS, each in two blocks of 16, which are read a block ahead of their products.  Once the second
    // one is read no wave needs this buffer any more and the other is whole: the one barrier, with the second block's products still to
    // come.  Slices on their way from memory have two register sets, so that each has the time of two slices' products.  (No conditions
    // inside: a load that may not have been made costs the waits their precision.  What is loaded behind the last slice is that one
    // again, unread.)
    f32x4 x[2][F], w[2][F];
    auto fetch = [&](const float* buf, int c) {
      const float* sa = buf + (wm * (SIDE / 2) + lr) * TF_LDK + 16 * c + 4 * quad;
#pragma unroll
      for (int i = 0; i < F; ++i) x[c][i] = *(const f32x4*)(sa + i * 16 * TF_LDK);
      if constexpr (W_TR) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Columns n = *(const Columns*)(buf + SIZE_A + (16 * c + 4 * quad + e) * SliceColumns<SIDE>::LD + wn * (SIDE / 2) + lr * F);
#pragma unroll
          for (int j = 0; j < F; ++j) w[c][j][e] = n[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < F; ++j) w[c][j] = *(const f32x4*)(buf + SIZE_A + (wn * (SIDE / 2) + j * 16 + lr) * TF_LDK + 16 * c + 4 * quad);
      }
    };
    auto products = [&](int c) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
          for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[c][i][e], w[c][j][e], acc[i][j], 0, 0, 0);
    };
    auto store = [&](float* buf, auto set) { A.store(buf, A.v[set]), B.store(buf + SIZE_A, B.v[set]); };
    const int whole = min(last, a.K / TF_K);
    auto load = [&](int s, auto set) { A.load(min(s, whole - 1) * TF_K, A.v[set]), B.load(min(s, whole - 1) * TF_K, B.v[set]); };
    auto slice = [&](int s, auto odd) {
      constexpr int ODD = decltype(odd)::value;
      constexpr std::integral_constant<int, 1 - ODD> set{};
      float* cur = lds + ODD * (SIZE_A + SIZE_B);
      float* other = lds + (1 - ODD) * (SIZE_A + SIZE_B);
      // (a memory instruction behind every few products: a row of them would hold the products up, as LDS takes 8 clocks for each)
      constexpr int PRODUCTS = 4 * F * F, READS = F + (W_TR ? 4 : F), LOADS = SliceA::N + SliceB::N, WRITES = LOADS;
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
    if (first < whole) {
      load(first, even);
      store(lds, even);
      load(first + 1, odd);
      load(first + 2, even);
      __syncthreads();
      fetch(lds, 0);
#pragma unroll 1
      for (int s = first;; s += 2) {
        slice(s, even);
        if (s + 1 >= whole) break;
        slice(s + 1, odd);
        if (s + 2 >= whole) break;
      }
      __syncthreads();
    }
    if (last > whole) {                                      // a part of a slice, with zeros behind it
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
  }

  // Elements [q, q + 4) of U's row t, zeros behind the rank
  static __device__ __forceinline__ f32x4 ranks(const AdapterProjectArgs& a, int64_t t, int q) {
    const float* u = a.U + t * a.r + q;
    if (q + 4 <= a.r) return *(const f32x4_by4*)u;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q + e < a.r ? u[e] : 0.0f;
    return v;
  }
  // B of adapter `id` for this lane's columns, ranks [q, q + 4), zeros behind the rank
  __device__ __forceinline__ void factors(const AdapterProjectArgs& a, int id, int q, const int (&column)[F], f32x4 (&b)[F]) const {
    const float* from = (const float*)a.B + (int64_t)id * a.sbr + q * a.sbj;
    if (W_TR && a.sbn == 1 && column[F - 1] < a.N) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Columns c = q + e < a.r ? (Columns)*(const ColumnsBy4*)(from + e * a.sbj + column[0]) : Columns{};
#pragma unroll
        for (int j = 0; j < F; ++j) b[j][e] = c[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < F; ++j) {
        const float* of = from + std::min(column[j], a.N - 1) * a.sbn;
        if (a.sbj == 1 && q + 4 <= a.r) b[j] = *(const f32x4_by4*)of;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) b[j][e] = q + e < a.r ? of[e * a.sbj] : 0.0f;
      }
    }
  }

  // Y = acc + U B[a]^T (+ bias): of a block of 16 rows one adapter's part after the other, as products of the whole block of which
  // the adapter's rows keep theirs: no row meets what another's adapter holds, nor depends on its neighbours.
  __device__ __forceinline__ void finish(const AdapterProjectArgs& a, Shared& sh) {
    // register e of a lane: row 4 (lane / 16) + e and, of block j, column 16 j + lane % 16 (W_TR: F (lane % 16) + j) of the wave's
    auto row_of = [&](int i, int e) { return wm * (SIDE / 2) + i * 16 + quad * 4 + e; };
    int column[F];
#pragma unroll
    for (int j = 0; j < F; ++j) column[j] = n0 + wn * (SIDE / 2) + (W_TR ? lr * F + j : j * 16 + lr);
#pragma unroll 1
    for (int q0 = 0; q0 < a.r; q0 += 16) {
      f32x4 b[F];
      int at = -1;                                           // whose B that is
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int64_t t = sh.row[wm * (SIDE / 2) + i * 16 + lr];
        const int mine = sh.adapter[wm * (SIDE / 2) + i * 16 + lr];
        unsigned left = (unsigned)__ballot(mine >= 0) & 0xffff;
        if (left == 0) continue;
        const f32x4 u = ranks(a, t < 0 ? -1 - t : t, q0 + 4 * quad);
        while (left) {
          const int id = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
          const unsigned rows = (unsigned)__ballot(mine == id) & 0xffff;
          left &= ~rows;
          if (id != at) factors(a, at = id, q0 + 4 * quad, column, b);
          f32x4 v[F];
#pragma unroll
          for (int j = 0; j < F; ++j) v[j] = acc[i][j];
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < F; ++j) v[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[e], b[j][e], v[j], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool keep = rows >> (quad * 4 + e) & 1;
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j][e] = keep ? v[j][e] : acc[i][j][e];
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < F; ++j) {
      if (column[j] >= a.N) continue;
      const float bias = a.bias ? ((const float*)a.bias)[column[j] * a.sb] : 0.0f;
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t t = sh.row[row_of(i, e)];
          if (t >= 0) ((float*)a.Y)[t * a.sym + column[j]] = acc[i][j][e] + bias;
        }
    }
  }

  // what a workgroup has of a tile that it does not finish
  __device__ __forceinline__ void leave(float* to) const {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) *(f32x4*)(to + ((i * F + j) * TF_NT + threadIdx.x) * 4) = acc[i][j];
  }
  __device__ __forceinline__ void take(const float* from) {
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int j = 0; j < F; ++j) acc[i][j] += *(const f32x4*)(from + ((i * F + j) * TF_NT + threadIdx.x) * 4);
  }
};

// Tiles one after another, rows fastest; an XCD takes a run of them: its columns of W are read from memory once.
static __device__ __forceinline__ int64_t xcd_run(int64_t all) {
  const int64_t per = (all + 7) / 8, at = blockIdx.x >> 3;
  return at < per ? (blockIdx.x & 7) * per + at : all;
}

template <int SIDE, bool W_TR>
__global__ __launch_bounds__(TF_NT, 2) void adapter_tiles_f32_kernel(AdapterProjectArgs a, int m_tiles, int n_tiles) {
  typedef TileF32<SIDE, W_TR> Tile;
  __shared__ __attribute__((aligned(16))) typename Tile::Shared s;
  const int64_t all = (int64_t)m_tiles * n_tiles, tile = xcd_run(all);
  if (tile >= all) return;
  Tile t;
  t.start(a, s, tile % m_tiles * SIDE, (int)(tile / m_tiles) * SIDE);
  t.multiply(a, s, 0, (a.K + TF_K - 1) / TF_K);
  t.finish(a, s);
}

// Slices of all tiles in one row, dealt to TF_WGS workgroups in equal runs: a tile that a run's end cuts is left in parts, at most two by a
// workgroup (of the tile that it begins in, and of the one it ends in), and joined in the order of its slices.
static constexpr int TF_WGS = 512, TF_SIDE = 64, TF_MOST_TILES = 1 << 16;
struct TileRuns {
  int64_t slices, all;                               // of a tile, of all tiles
  __host__ __device__ int64_t first(int64_t w) const { return all * w / TF_WGS; }
};
template <bool W_TR>
__global__ __launch_bounds__(TF_NT, 2) void adapter_runs_f32_kernel(AdapterProjectArgs a, int m_tiles, TileRuns runs, float* parts) {
  typedef TileF32<TF_SIDE, W_TR> Tile;
  __shared__ __attribute__((aligned(16))) typename Tile::Shared s;
  const int64_t w = xcd_run(TF_WGS), last = runs.first(w + 1);
#pragma unroll 1
  for (int64_t u = runs.first(w); u < last;) {
    const int64_t tile = u / runs.slices;
    const int from = (int)(u - tile * runs.slices), to = (int)std::min(runs.slices, from + last - u);
    Tile t;
    t.start(a, s, tile % m_tiles * TF_SIDE, (int)(tile / m_tiles) * TF_SIDE);
    t.multiply(a, s, from, to);
    if (from == 0 && to == runs.slices) t.finish(a, s);
    else t.leave(parts + (2 * w + (from == 0)) * TF_SIDE * TF_SIDE);
    u += to - from;
    __syncthreads();
  }
}
template <bool W_TR>
__global__ __launch_bounds__(TF_NT, 2) void adapter_runs_join_f32_kernel(AdapterProjectArgs a, int m_tiles, TileRuns runs, const float* parts) {
  typedef TileF32<TF_SIDE, W_TR> Tile;
  __shared__ __attribute__((aligned(16))) typename Tile::Shared s;
  const int64_t tile = blockIdx.x, begin = tile * runs.slices, end = begin + runs.slices;
  int64_t w = begin * TF_WGS / runs.all;                     // the run that the tile begins in
  while (runs.first(w + 1) <= begin) ++w;
  if (runs.first(w + 1) >= end) return;                      // ... and ends in
  Tile t;
  t.start(a, s, tile % m_tiles * TF_SIDE, (int)(tile / m_tiles) * TF_SIDE);
  for (; runs.first(w) < end; ++w)
    if (runs.first(w) < runs.first(w + 1)) t.take(parts + (2 * w + (runs.first(w) <= begin)) * TF_SIDE * TF_SIDE);
  t.finish(a, s);
}

template <int SIDE>
static int launch_tiles_f32(const AdapterProjectArgs& a, hipStream_t st) {
  const int64_t m_tiles = cdiv64(a.T, SIDE), n_tiles = cdiv64(a.N, SIDE), grid = cdiv64(m_tiles * n_tiles, 8) * 8;
  if (grid > 0x7fffffffLL) { set_error("adapters: too many rows and columns for one launch"); return SMOE_ERR_RANGE; }
  if (a.swk == 1) hipLaunchKernelGGL((adapter_tiles_f32_kernel<SIDE, false>), dim3((unsigned)grid), dim3(TF_NT), 0, st, a, (int)m_tiles, (int)n_tiles);
  else hipLaunchKernelGGL((adapter_tiles_f32_kernel<SIDE, true>), dim3((unsigned)grid), dim3(TF_NT), 0, st, a, (int)m_tiles, (int)n_tiles);
  return launch_status("adapter_tiles_f32_kernel");
}
static int launch_runs_f32(const AdapterProjectArgs& a, float* parts, hipStream_t st) {
  const int64_t m_tiles = cdiv64(a.T, TF_SIDE), tiles = m_tiles * cdiv64(a.N, TF_SIDE), slices = cdiv64(a.K, TF_K);
  const TileRuns runs{slices, tiles * slices};
  if (a.swk == 1) hipLaunchKernelGGL(adapter_runs_f32_kernel<false>, dim3(TF_WGS), dim3(TF_NT), 0, st, a, (int)m_tiles, runs, parts);
  else hipLaunchKernelGGL(adapter_runs_f32_kernel<true>, dim3(TF_WGS), dim3(TF_NT), 0, st, a, (int)m_tiles, runs, parts);
  if (int rc = launch_status("adapter_runs_f32_kernel")) return rc;
  if (a.swk == 1) hipLaunchKernelGGL(adapter_runs_join_f32_kernel<false>, dim3((unsigned)tiles), dim3(TF_NT), 0, st, a, (int)m_tiles, runs, parts);
  else hipLaunchKernelGGL(adapter_runs_join_f32_kernel<true>, dim3((unsigned)tiles), dim3(TF_NT), 0, st, a, (int)m_tiles, runs, parts);
  return launch_status("adapter_runs_join_f32_kernel");
}

int64_t adapter_f32_parts() { return (int64_t)2 * TF_WGS * TF_SIDE * TF_SIDE; }
static int64_t tiles_f32(int64_t T, int64_t N, int64_t side) { return cdiv64(T, side) * cdiv64(N, side); }
// A round of whole tiles, one per CU, is a chain of K products, and a tile more than whole rounds is a round more; runs of slices have no rounds,
// but parts to leave and a launch to join them; the rows' kernel (project_t in adapters.hip) has work for the whole chip from few rows on, at
// 66 TFLOP/s, and a weight whose contraction is strided to copy first.  The times below in us; measured, us of a call (u and the order of
// the rows in it), rows' kernel / 128 x 128 / 64 x 64 / runs: 65 rows, 4096 -> 4096 72 / 255 / 81 / 57; 256 rows 142 / 257 / 90 / 92; 320 rows 173 /
// 259 / 148 / 107; 520 rows 286 / 260 / 208 / 174; 1024 rows 509 / 269 / 277 / 277; 4096 rows 1984 / 990 / 1038 / 1060; 128 rows, 2048 -> 2048
// 28 / 137 / 47 / 33; 256 rows 47 / 139 / 50 / 40; 1024 rows 141 / 142 / 86 / 84; 203 rows, 1003 -> 1517 28 / 81 / 32 / 33; 1024 rows 66 / 86 / 53 /
// 53, 512 -> 512 22 / 52 / 24 / 28, 1472 -> 2064 (528 tiles of 64 x 64) 125 / 109 / 91 / 79; an elementary product and its small ones, for 320, 520
// and 1024 rows of 4096 113, 183 and 281.
AdapterF32 adapter_f32_class(int64_t T, int64_t K, int64_t N, bool strided) {
  if (T <= ADAPTER_FEW_ROWS || N < 4) return ADAPTER_F32_ROWS;
  const double k = (double)K, small = (double)tiles_f32(T, N, 64) / TF_CUS;
  const int64_t rounds = cdiv64(tiles_f32(T, N, 64), TF_CUS), large = cdiv64(tiles_f32(T, N, 128), TF_CUS);
  double least = std::max(2e-6 / 66 * (32 * cdiv64(T, 32)) * N * k, 3.0) + (strided ? 4.0 + 1.6e-6 * N * k : 0.0);
  AdapterF32 best = ADAPTER_F32_ROWS;
  auto take = [&](AdapterF32 how, double time) { if (time < least) least = time, best = how; };
  take(ADAPTER_F32_128, large * (0.0598 * k + 5.0));
  take(ADAPTER_F32_64, rounds == 1 ? 0.0187 * k + 3.0 : rounds * (0.0163 * k + 2.0));
  if (tiles_f32(T, N, 64) <= TF_MOST_TILES) take(ADAPTER_F32_RUNS, small * 0.0166 * k + 14.0);
  return best;
}
int launch_adapter_f32(const AdapterProjectArgs& a, AdapterF32 how, float* parts, hipStream_t st) {
  if (how == ADAPTER_F32_RUNS) return launch_runs_f32(a, parts, st);
  return how == ADAPTER_F32_128 ? launch_tiles_f32<128>(a, st) : launch_tiles_f32<64>(a, st);
}

}  // namespace smoe
