// Low-rank adapters of many requests beside a shared projection.  Row t carries the adapter a = ids[t]; a row whose id
// lies outside [0, R) carries none:
//   U[t] = s[a] A[a] X[t]                 (r values, float32)
//   Y[t] = W X[t] + bias + B[a] U[t]
// The backward pass is made of the same two products with the factors exchanged (V[t] = s[a] B[a]^T DY[t],
// DX[t] = W^T DY[t] + A[a]^T V[t]) and of the adapters' own gradients, sums over the rows that carry them:
//   DA[a] = sum_t V[t] X[t]^T,   DB[a] = sum_t DY[t] U[t]^T.
//
// The reference has no counterpart; the rows pick their weights by id as in scattermoe/parallel_experts.py:148-182.
#include "few_rows.hpp"
#include <algorithm>

namespace smoe {

// U in float32: it is a factor of the second product and of a gradient, and is r values per row.
template <typename T>
__global__ __launch_bounds__(256) void adapter_low_any_kernel(AdapterLowArgs a) {
  const int64_t t = blockIdx.x;
  const int64_t id = a.ids[t];
  const bool has = (uint64_t)id < (uint64_t)a.R;
  const float scale = has ? (a.scales ? a.scales[id] : 1.0f) : 0.0f;
  for (int j = threadIdx.x >> 6; j < a.r; j += 4) {
    float v = 0.0f;
    if (has) {
      const T* x = (const T*)a.X + t * a.sxm;
      const T* w = (const T*)a.A + id * a.sar + j * a.saj;
      for (int i = lane_id(); i < a.K; i += 64) v = fmaf(to_f32(x[i]), to_f32(w[i * a.sak]), v);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    }
    if (lane_id() == 0) a.U[t * a.r + j] = has ? v * scale : 0.0f;
  }
}

// Any layout: 64 x 64 output tiles, fp32 multiply-adds through LDS.
static constexpr int PBM = 64, PBN = 64, PBK = 16, PT = 256;
template <typename T>
__global__ __launch_bounds__(PT) void adapter_project_any_kernel(AdapterProjectArgs a) {
  __shared__ float sA[PBK][PBM + 4];
  __shared__ float sB[PBK][PBN + 4];
  const int across = (a.N + PBN - 1) / PBN, n0 = (int)(blockIdx.x % across) * PBN, tid = threadIdx.x;
  const int64_t t0 = (int64_t)(blockIdx.x / across) * PBM;
  const int ty = tid / 16, tx = tid % 16;
  const T* X = (const T*)a.X;
  const T* W = (const T*)a.W;
  const bool n_fast = a.swn == 1;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += PBK) {
#pragma unroll
    for (int i = 0; i < PBM * PBK / PT; ++i) {
      const int lin = tid + i * PT, kk = lin % PBK, mm = lin / PBK;
      sA[kk][mm] = t0 + mm < a.T && k0 + kk < a.K ? to_f32(X[(t0 + mm) * a.sxm + k0 + kk]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < PBN * PBK / PT; ++i) {
      const int lin = tid + i * PT;
      const int kk = n_fast ? lin / PBN : lin % PBK, nn = n_fast ? lin % PBN : lin / PBK;
      sB[kk][nn] = k0 + kk < a.K && n0 + nn < a.N ? to_f32(W[(k0 + kk) * a.swk + (n0 + nn) * a.swn]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < PBK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sA[kk][ty * 4 + i], sB[kk][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty * 4 + i;
    if (t >= a.T) continue;
    const int64_t id = a.ids[t];
    const bool has = (uint64_t)id < (uint64_t)a.R;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= a.N) continue;
      float v = acc[i][j];
      if (a.bias) v += to_f32(((const T*)a.bias)[n * a.sb]);
      if (has) {
        const T* b = (const T*)a.B + id * a.sbr + n * a.sbn;
        for (int q = 0; q < a.r; ++q) v = fmaf(a.U[t * a.r + q], to_f32(b[q * a.sbj]), v);
      }
      ((T*)a.Y)[t * a.sym + n] = from_f32<T>(v);
    }
  }
}

// Gradient of one factor of every adapter: OUT[a][j][c] = sum over the adapter's rows t of P[t][j] M[t][c].
// A workgroup has 64 columns of one adapter; its four waves take the rows in turn and are added up in a fixed order.
static constexpr int GRAD_RANKS = 8;
template <typename T>
__global__ __launch_bounds__(256) void adapter_grad_any_kernel(AdapterGradArgs a) {
  __shared__ float part[4][GRAD_RANKS][64];
  const int id = blockIdx.y, lane = lane_id(), wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  const int64_t lo = id ? a.off[id - 1] : 0, hi = a.off ? a.off[id] : a.T;
  for (int j0 = 0; j0 < a.r; j0 += GRAD_RANKS) {
    float acc[GRAD_RANKS] = {};
    for (int64_t i = lo + wave; i < hi; i += 4) {
      const int64_t t = a.idx ? a.idx[i] : i;
      const float m = c < a.C ? to_f32(((const T*)a.M)[t * a.smm + c]) : 0.0f;
#pragma unroll
      for (int j = 0; j < GRAD_RANKS; ++j)
        if (j0 + j < a.r) acc[j] = fmaf(a.P ? a.P[t * a.r + j0 + j] : 1.0f, m, acc[j]);
    }
#pragma unroll
    for (int j = 0; j < GRAD_RANKS; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < GRAD_RANKS / 4; ++q) {
      const int j = wave + 4 * q;
      if (j0 + j < a.r && c < a.C)
        ((T*)a.OUT)[id * a.soa + (j0 + j) * a.soj + c * a.soc] =
            from_f32<T>(((part[0][j][lane] + part[1][j][lane]) + part[2][j][lane]) + part[3][j][lane]);
    }
    __syncthreads();
  }
}

// ---- U, contiguous rows ------------------------------------------------------------------------------------------------
// Few rows: DOT_ROWS values of one row by a workgroup.  Bound by latency (1 row of 4096, rank 16 4.4 us; 48 rows of 2880, rank 32, 64
// adapters 5.5 us for 12 MB of factors).
template <typename T>
__global__ __launch_bounds__(DOT_NW * 64) void adapter_low_dots_kernel(AdapterLowArgs a) {
  __shared__ float part[DOT_NW * DOT_ROWS];
  const int64_t t = blockIdx.x, id = a.ids[t];
  const int j = blockIdx.y * DOT_ROWS + threadIdx.x;
  const bool mine = threadIdx.x < DOT_ROWS && j < a.r;
  if ((uint64_t)id >= (uint64_t)a.R) {
    if (mine) a.U[t * a.r + j] = 0.0f;
    return;
  }
  const T* w[DOT_ROWS];
#pragma unroll
  for (int i = 0; i < DOT_ROWS; ++i) w[i] = (const T*)a.A + id * a.sar + std::min<int>(blockIdx.y * DOT_ROWS + i, a.r - 1) * a.saj;
  const float v = dot_rows<T>((const T*)a.X + t * a.sxm, w, a.K, part);
  if (mine) a.U[t * a.r + j] = v * (a.scales ? a.scales[id] : 1.0f);
}

// Many rows, ordered by adapter: 16 rows of one adapter and LOW_RANKS of the rank by a workgroup.  (The rows' elements come
// from memory once, the factor's from the caches: rows of one adapter follow one another.)  8192 rows of 4096, rank 16 17.3 us: 67 MB
// of rows at 3.9 TB/s; 1777 rows of 2048, rank 64 9.3 us, four workgroups reading a row.
static constexpr int LOW_NW = 8, LOW_RANKS = 16;
static_assert(LOW_RANKS == 16, "exponents of the planes: one for the 16 ranks of a workgroup");
template <typename T>
__global__ __launch_bounds__(LOW_NW * 64, 4) void adapter_low_rows_kernel(AdapterLowArgs a) {
  __shared__ float part[FEW_PART<LOW_NW, LOW_RANKS, 16>];
  int id, row0, rows;
  const bool has = find_tile<16>(a.off, a.R + 1, blockIdx.x, id, row0, rows);
  if (a.slots && blockIdx.y == 0 && threadIdx.x < 17) {
    int* s = a.slots + (int64_t)blockIdx.x * 17;
    if (threadIdx.x < 16) s[threadIdx.x] = has && (int)threadIdx.x < rows ? (int)a.idx[row0 + threadIdx.x] : -1;
    else s[16] = has && id < a.R ? id : -1;
  }
  const int m_ = threadIdx.x / LOW_RANKS, n_ = threadIdx.x % LOW_RANKS;
  // where this row of the fragment has its power of two
  int* exponent = nullptr;
  if constexpr (std::is_same<T, f16_t>::value) {
    if (a.planes && n_ == 0 && m_ < 16) exponent = a.exponents + ((int64_t)blockIdx.x * 16 + m_) * (a.rp / LOW_RANKS) + blockIdx.y;
    if (exponent && (!has || m_ >= rows)) *exponent = PLANES_NONE;
  }
  if (!has) return;
  const int j0 = blockIdx.y * LOW_RANKS, j = j0 + n_;
  const bool some = id < a.R && j0 < a.r;
  if (some) {
    few_tile<T, 2, 2, 1, LOW_NW, LOW_RANKS, false>([&](int n) { return (const T*)a.A + id * a.sar + min(j0 + n, a.r - 1) * a.saj; },
                                                   [&](int m) { return (const T*)a.X + a.idx[row0 + min(m, rows - 1)] * a.sxm; }, 0, a.K, part);
    __syncthreads();
  }
  if (m_ >= rows) return;
  float v = 0.0f;
  if (some && j < a.r) v = few_sum<LOW_NW, LOW_RANKS, 16>(part, n_, m_) * (a.scales ? a.scales[id] : 1.0f);
  const int64_t t = a.idx[row0 + m_];
  if (j < a.r) a.U[t * a.r + j] = v;
  if (a.planes && j < a.rp) {
    float w = v;
    if constexpr (std::is_same<T, f16_t>::value) {
      // (the 16 lanes of a row; beside a value that is not finite the finite ones are nothing)
      float most = v == v ? fabsf(v) : INFINITY;
#pragma unroll
      for (int o = LOW_RANKS / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
      const int log = most > 0.0f ? ilogbf(most) : PLANES_NONE + PLANES_TOP;
      const int e = log >= PLANES_LEAST && log <= PLANES_TOP ? 0 : min(max(log - PLANES_TOP, PLANES_NONE), PLANES_MOST);
      w = ldexpf(v, -e);
      if (exponent) *exponent = e;
    }
    T* p = (T*)a.planes + t * 2 * a.rp + j;
    split<T>(w, p[0], p[a.rp]);
  }
}

// ... float32, where such workgroups would be few: 16 / P rows and ranks each, so that a CU fetches less.  us, 16 x 16 / 8 x 8 / 4 x 4, rows of
// 4096: 320 rows, rank 8 13.0 / 6.5 / 4.6, eight adapters of rank 16 13.8 / 7.2 / 8.5; 1024 rows, rank 8 13.2 / 6.7 / 7.6, eight adapters of rank 16 14.6
// / 14.0 / 15.6; 2048 rows 16.1 / 17.6 / 26.0; 1024 rows, 64 adapters of rank 32 16.4 / 24.6 / 41.8, one of rank 64 28.0 / 22.5 / 40.6.
static constexpr int64_t LOW_PARTS4 = 4096, LOW_PARTS2 = 16384;          // rows times rank
template <int P>
__global__ __launch_bounds__(LOW_NW * 64, 4) void adapter_low_parts_kernel(AdapterLowArgs a) {
  constexpr int SIDE = 16 / P;
  __shared__ float part[FEW_PART<LOW_NW, SIDE, SIDE>];
  int id, row0, rows;
  if (!find_tile<SIDE>(a.off, a.R + 1, blockIdx.x, id, row0, rows)) return;
  const int m = threadIdx.x / SIDE, n = threadIdx.x % SIDE, j0 = blockIdx.y * SIDE, j = j0 + n;
  if (id < a.R) {
    few_tile<float, P, 1, 1, LOW_NW, SIDE, false>([&](int n) { return (const float*)a.A + id * a.sar + min(j0 + n, a.r - 1) * a.saj; },
                                                  [&](int m) { return (const float*)a.X + a.idx[row0 + min(m, rows - 1)] * a.sxm; }, 0, a.K, part);
    __syncthreads();
  }
  if (m >= rows || j >= a.r) return;
  a.U[a.idx[row0 + m] * a.r + j] = id < a.R ? few_sum<LOW_NW, SIDE, SIDE>(part, n, m) * (a.scales ? a.scales[id] : 1.0f) : 0.0f;
}

// ---- Y, few rows or little work: tiles of COLS columns and 16 G / P rows, both operands from the caches or from memory ------------
// Few rows are a stream over the weights: 1 row, 4096 -> 4096 8.0 us (4.2 TB/s; the launch's ends are a third of it), 48 rows,
// 2880 -> 4096 13.3 us (the weights come once from memory and once more from the caches).  float32 is bound by the operands' way from
// the caches (66 TFLOP/s): 203 rows, 1003 -> 1517 21.2 us (0.62 GFLOP); beyond a measured line its products go in adapters_f32.hip's tiles.
template <typename T, int P, int G, int NW, int COLS>
__global__ __launch_bounds__(NW * 64, G > 4 ? 2 : 4) void adapter_project_rows_kernel(AdapterProjectArgs a) {
  constexpr int INPUTS = 16 * G / P;
  __shared__ float part[FEW_PART<NW, COLS, INPUTS>];
  const int across = (a.N + COLS - 1) / COLS, n0 = (int)(blockIdx.x % across) * COLS;
  const int64_t t0 = (int64_t)(blockIdx.x / across) * INPUTS;
  few_tile<T, P, G, 1, NW, COLS, false, P == 4 ? 4 : 0>([&](int n) { return (const T*)a.W + std::min(n0 + n, a.N - 1) * a.swn; },
                                        [&](int m) { return (const T*)a.X + std::min<int64_t>(t0 + m, a.T - 1) * a.sxm; }, 0, a.K, part);
  __syncthreads();
  for (int p = threadIdx.x; p < COLS * INPUTS; p += NW * 64) {
    const int m = p / COLS, c = p % COLS, n = n0 + c;
    const int64_t t = t0 + m;
    if (t >= a.T || n >= a.N) continue;
    float v = few_sum<NW, COLS, INPUTS>(part, c, m);
    if (a.bias) v += to_f32(((const T*)a.bias)[n * a.sb]);
    const int64_t id = a.ids[t];
    if ((uint64_t)id < (uint64_t)a.R) {
      const T* b = (const T*)a.B + id * a.sbr + n * a.sbn;
      const float* u = a.U + t * a.r;
      int q = 0;
      if (a.sbj == 1) {
        constexpr int PER = Few<T>::PER;
        typedef T V __attribute__((ext_vector_type(PER)));
        for (; q + PER <= a.r; q += PER) {
          const V bv = __builtin_bit_cast(V, load_piece<T, false>(b + q));
#pragma unroll
          for (int i = 0; i < PER; ++i) v = fmaf(u[q + i], to_f32(bv[i]), v);
        }
      }
      for (; q < a.r; ++q) v = fmaf(u[q], to_f32(b[q * a.sbj]), v);
    }
    ((T*)a.Y)[t * a.sym + n] = from_f32<T>(v);
  }
}

// ---- the adapters' gradients, contiguous rows ------------------------------------------------------------------------
// OUT[a][j][c] on float32 matrix instructions (16 x 16 x 4): P stays the float32 it is, and its rows, the contraction, need no
// transposition, as a lane of the instruction holds one element of one row.  A lane loads 16 bytes of a row of M, and element i of
// them is its column of product i: columns PER l + i.  A workgroup has 16 PER columns, JT x 16 of the rank and a slice of the
// adapter's rows, which its waves take in turn, four at a time.
// The gradients of both factors in one launch: the one's workgroups fill what the other's leave idle (8192 rows, 4096 and 4096 columns,
// rank 16: two launches 22 us each, one 37.7: 134 MB of rows at 3.6 TB/s).  Bound by the rows there; 24 adapters of 170 mixed rows each,
// 2880 columns, rank 24 take 31 us for 47 MB: three rounds of a wave, each waiting for its rows (one round more in flight took
// registers that waves needed: 37; bounds for four waves per SIMD, or one tile of ranks per workgroup: no difference).
static constexpr int GRAD_NW = 4, GRAD_MAX_SLICES = 16;
struct GradLaunch {
  AdapterGradArgs a;
  int slices, columns, ranks;                        // of the rows; tiles of columns, of ranks
  float* partial;                                    // the slices' sums, (slices, R, r, C)
  __host__ __device__ int64_t all_blocks() const { return (int64_t)columns * ranks * a.R * slices; }
  __host__ __device__ int64_t all_joins() const { return slices > 1 ? (int64_t)((a.C + 255) / 256) * a.r * a.R : 0; }
  __host__ __device__ int blocks() const { return (int)all_blocks(); }
  __host__ __device__ int joins() const { return (int)all_joins(); }
};
struct GradPair { GradLaunch of[2]; };
template <typename T, int JT>
__global__ __launch_bounds__(GRAD_NW * 64) void adapter_grad_kernel(GradPair pair) {
  const bool second = (int)blockIdx.x >= pair.of[0].blocks();
  const GradLaunch& g = pair.of[second];
  const AdapterGradArgs& a = g.a;
  const int slices = g.slices;
  float* partial = g.partial;
  int at = blockIdx.x - (second ? pair.of[0].blocks() : 0);
  const int column = at % g.columns;
  at /= g.columns;
  const int rank = at % g.ranks;
  at /= g.ranks;
  constexpr int PER = Few<T>::PER, COLS = 16 * PER;
  typedef T V __attribute__((ext_vector_type(PER)));
  __shared__ __attribute__((aligned(16))) float part[GRAD_NW][16][COLS];
  const int id = at / slices, slice = at % slices, lane = lane_id(), wave = threadIdx.x >> 6;
  const int l = lane & 15, q = lane >> 4, j0 = rank * JT * 16;
  const int c0 = column * COLS + l * PER, c = min(c0, a.C - PER);        // (the last columns: once more, by the lane before them)
  const int64_t first = id ? a.off[id - 1] : 0, count = (a.off ? a.off[id] : a.T) - first;
  const int64_t lo = first + count * slice / slices, hi = first + count * (slice + 1) / slices;
  f32x4 acc[JT][PER];
#pragma unroll
  for (int j = 0; j < JT; ++j)
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int SIDE = 4;                                    // steps of four rows whose loads are issued side by side
  // (the rows' indices one round ahead of their elements)
  int64_t next[SIDE];
  auto fetch = [&](int64_t s) {
#pragma unroll
    for (int u = 0; u < SIDE; ++u) {
      const int64_t i = std::min(s + 4 * u + q, hi - 1);
      next[u] = a.idx ? a.idx[i] : i;
    }
  };
  if (lo + wave * 4 * SIDE < hi) fetch(lo + wave * 4 * SIDE);
#pragma unroll 1
  for (int64_t s = lo + wave * 4 * SIDE; s < hi; s += GRAD_NW * 4 * SIDE) {
    V m[SIDE];
    float p[SIDE][JT];
#pragma unroll
    for (int u = 0; u < SIDE; ++u) {
      m[u] = __builtin_bit_cast(V, load_piece<T, false>((const T*)a.M + next[u] * a.smm + c));
#pragma unroll
      for (int j = 0; j < JT; ++j) p[u][j] = a.P ? a.P[next[u] * a.r + min(j0 + 16 * j + l, a.r - 1)] : 1.0f;
    }
    if (s + GRAD_NW * 4 * SIDE < hi) fetch(s + GRAD_NW * 4 * SIDE);
    __builtin_amdgcn_sched_barrier(0);
    if (s + 4 * SIDE > hi) {
#pragma unroll
      for (int u = 0; u < SIDE; ++u)
        if (s + 4 * u + q >= hi) {
          m[u] = __builtin_bit_cast(V, i32x4{0, 0, 0, 0});
#pragma unroll
          for (int j = 0; j < JT; ++j) p[u][j] = 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < SIDE; ++u)
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[u][j], to_f32(m[u][i]), acc[j][i], 0, 0, 0);
  }
  // a lane holds ranks j0 + 16 j + 4 q + e of columns c + i: the waves' sums in LDS as rows of columns, then a piece of a row per thread
  const int row = threadIdx.x >> 4, piece = threadIdx.x & 15;
  const int from = column * COLS + piece * PER, to = min(from, a.C - PER);
  static_assert(GRAD_NW * 64 == 256, "a piece per thread");
#pragma unroll
  for (int j = 0; j < JT; ++j) {
    if (j > 0) __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < PER; i += 4)
        *(f32x4*)(part[wave][4 * q + e] + l * PER + i) = f32x4{acc[j][i][e], acc[j][i + 1][e], acc[j][i + 2][e], acc[j][i + 3][e]};
    __syncthreads();
    const int r = j0 + 16 * j + row;
    if (r >= a.r || from >= a.C) continue;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      f32x4 s = *(const f32x4*)(part[0][row] + piece * PER + i);
#pragma unroll
      for (int w = 1; w < GRAD_NW; ++w) s += *(const f32x4*)(part[w][row] + piece * PER + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i + k] = s[k];
    }
    if (slices > 1) {
      float* p = partial + (((int64_t)slice * a.R + id) * a.r + r) * a.C + to;
#pragma unroll
      for (int i = 0; i < PER; ++i) p[i] = v[i];
    } else {
      T* out = (T*)a.OUT + id * a.soa + r * a.soj + to * a.soc;
#pragma unroll
      for (int i = 0; i < PER; ++i) out[i * a.soc] = from_f32<T>(v[i]);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void adapter_grad_join_kernel(GradPair pair) {
  const bool second = (int)blockIdx.x >= pair.of[0].joins();
  const GradLaunch& g = pair.of[second];
  const AdapterGradArgs& a = g.a;
  const int slices = g.slices, across = (a.C + 255) / 256;
  const float* partial = g.partial;
  const int at = blockIdx.x - (second ? pair.of[0].joins() : 0);
  const int c = at % across * 256 + threadIdx.x, j = at / across % a.r, id = at / across / a.r;
  if (c >= a.C) return;
  const float* p = partial + ((int64_t)id * a.r + j) * a.C + c;
  const int64_t apart = (int64_t)a.R * a.r * a.C;
  float v[GRAD_MAX_SLICES];
#pragma unroll
  for (int s = 0; s < GRAD_MAX_SLICES; ++s) v[s] = s < slices ? p[s * apart] : 0.0f;
#pragma unroll
  for (int s = 1; s < GRAD_MAX_SLICES; ++s) v[0] += v[s];
  ((T*)a.OUT)[id * a.soa + j * a.soj + c * a.soc] = from_f32<T>(v[0]);
}

// ---- factors in another order ---------------------------------------------------------------------------------------
// DST[a][i][0 .. ld) = SRC[a, i, 0 .. n2), zeros behind: for the products that want the contraction contiguous, whole pieces of 16 bytes
// or rows that start at them.  With `off`, adapters without rows are left out (nobody reads them).
// Two copies in one launch: every launch costs about as much as the copy (factors of 24 adapters, 2880 x 24 12.8 us, 4096 x 16 of one
// 8.3; a 4096 x 4096 weight 26 us, 2.6 TB/s).
struct AdapterPacks { AdapterPackArgs of[2]; };
template <typename T>
__global__ __launch_bounds__(256) void adapter_pack_kernel(AdapterPacks packs) {
  __shared__ T tile[64][64 + 4 / sizeof(T)];
  const int first = packs.of[0].tiles();
  const AdapterPackArgs& a = packs.of[(int)blockIdx.x < first ? 0 : 1];
  int at = (int)blockIdx.x < first ? blockIdx.x : blockIdx.x - first;
  const int across = (a.ld + 63) / 64, down = (a.n1 + 63) / 64, id = at / (across * down);
  at -= id * across * down;
  if (a.off && a.off[id] == (id ? a.off[id - 1] : 0)) return;
  const int i0 = at / across * 64, k0 = at % across * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const T* src = (const T*)a.SRC + id * a.s0;
  T* dst = (T*)a.DST + (int64_t)id * a.n1 * a.ld;
  if (a.s2 == 1) {
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int i = i0 + y + 4 * u;
      if (i < a.n1 && k0 + x < a.ld) dst[(int64_t)i * a.ld + k0 + x] = k0 + x < a.n2 ? src[i * a.s1 + k0 + x] : from_f32<T>(0.0f);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int k = y + 4 * u;
    if (i0 + x < a.n1) tile[k][x] = k0 + k < a.n2 ? src[(i0 + x) * a.s1 + (k0 + k) * a.s2] : from_f32<T>(0.0f);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int i = y + 4 * u;
    if (i0 + i < a.n1 && k0 + x < a.ld) dst[(int64_t)(i0 + i) * a.ld + k0 + x] = tile[x][i];
  }
}

template <typename T>
static int low_t(const AdapterLowArgs& a, hipStream_t st) {
  const bool pieces = a.sak == 1 && a.K >= Few<T>::PER;
  if (pieces && a.idx != nullptr) {
    if constexpr (sizeof(T) == 4) {
      const int P = a.T * a.r <= LOW_PARTS4 ? 4 : a.T * a.r <= LOW_PARTS2 ? 2 : 1;
      const dim3 grid((unsigned)max_tiles(a.T, a.R + 1, 16 / P), (unsigned)cdiv64(a.r, 16 / P)), block(LOW_NW * 64);
      if (P == 4) hipLaunchKernelGGL(adapter_low_parts_kernel<4>, grid, block, 0, st, a);
      else if (P == 2) hipLaunchKernelGGL(adapter_low_parts_kernel<2>, grid, block, 0, st, a);
      if (P > 1) return launch_status("adapter_low_parts_kernel");
    }
    hipLaunchKernelGGL(adapter_low_rows_kernel<T>, dim3((unsigned)adapter_fragments(a.T, a.R), ((a.planes ? a.rp : a.r) + LOW_RANKS - 1) / LOW_RANKS), dim3(LOW_NW * 64), 0, st, a);
    return launch_status("adapter_low_rows_kernel");
  }
  if (pieces) {
    hipLaunchKernelGGL(adapter_low_dots_kernel<T>, dim3((unsigned)a.T, (a.r + DOT_ROWS - 1) / DOT_ROWS), dim3(DOT_NW * 64), 0, st, a);
    return launch_status("adapter_low_dots_kernel");
  }
  hipLaunchKernelGGL(adapter_low_any_kernel<T>, dim3((unsigned)a.T), dim3(256), 0, st, a);
  return launch_status("adapter_low_any_kernel");
}

template <typename T, int P, int G, int NW, int COLS>
static int project_rows(const AdapterProjectArgs& a, hipStream_t st) {
  const int64_t grid = cdiv64(a.T, 16 * G / P) * cdiv64(a.N, COLS);
  if (grid > 0x7fffffffLL) { set_error("adapters: too many rows and columns for one launch"); return SMOE_ERR_RANGE; }
  hipLaunchKernelGGL((adapter_project_rows_kernel<T, P, G, NW, COLS>), dim3((unsigned)grid), dim3(NW * 64), 0, st, a);
  return launch_status("adapter_project_rows_kernel");
}
template <typename T>
static int project_t(const AdapterProjectArgs& a, hipStream_t st) {
  if (a.swk == 1 && a.K >= Few<T>::PER) {
    // Beyond 32 rows: 16-bit types in chunks of 32 (48 rows, 2880 -> 4096 20 -> 12 us, 64 rows, 4096 -> 4096 29 -> 18, against tiles of
    // 64 x 32: twice the workgroups count for more than half the weights' traffic from the caches); float32, whose products are what
    // takes the time, without parts (64 rows, 2048 -> 2048 16 -> 15 us), in wider tiles from 65 rows on (1024 rows, 4096 -> 4096 695 -> 501).
    if (a.T <= 4) return project_rows<T, 4, 1, 8, 16>(a, st);
    if (a.T <= 8) return project_rows<T, 2, 1, 8, 16>(a, st);
    if (a.T <= 16) return project_rows<T, 2, 2, 8, 16>(a, st);
    if (a.T <= 32 || sizeof(T) == 2) return project_rows<T, 2, 4, 8, 16>(a, st);
    if constexpr (sizeof(T) == 4) return a.T <= 64 ? project_rows<T, 1, 2, 8, 16>(a, st) : project_rows<T, 1, 2, 8, 32>(a, st);
  }
  const int64_t grid = cdiv64(a.T, PBM) * cdiv64(a.N, PBN);
  if (grid > 0x7fffffffLL) { set_error("adapters: too many rows and columns for one launch"); return SMOE_ERR_RANGE; }
  hipLaunchKernelGGL(adapter_project_any_kernel<T>, dim3((unsigned)grid), dim3(PT), 0, st, a);
  return launch_status("adapter_project_any_kernel");
}

static int pieces(int dtype) { return dtype == SMOE_F32 ? 4 : 8; }           // elements of 16 bytes
// Slices of an adapter's rows: enough workgroups for the chip, at least GRAD_MIN_ROWS rows each at even loads
static constexpr int GRAD_WGS = 1024, GRAD_MIN_ROWS = 128;
static int grad_tiles(int64_t C, int dtype) { return (int)cdiv64(C, dtype == SMOE_F32 ? 64 : 128); }
static int grad_ranks(int64_t r) { return r <= 16 ? 1 : 2; }
static int grad_slices(int64_t T, int64_t C, int64_t r, int64_t R, int dtype) {
  if (C < pieces(dtype)) return 1;
  const int64_t wgs = grad_tiles(C, dtype) * R * cdiv64(r, 16 * grad_ranks(r));
  return (int)std::max<int64_t>(1, std::min<int64_t>({GRAD_WGS / wgs, T / R / GRAD_MIN_ROWS, GRAD_MAX_SLICES}));
}
static size_t grad_bytes(int64_t T, int64_t C, int64_t r, int64_t R, int dtype) {
  const int slices = grad_slices(T, C, r, R, dtype);
  return slices > 1 ? (size_t)slices * R * r * C * sizeof(float) : 0;
}
template <typename T>
static int grad_t(const GradPair& p, int r, hipStream_t st) {
  const int64_t blocks = p.of[0].all_blocks() + p.of[1].all_blocks(), joins = p.of[0].all_joins() + p.of[1].all_joins();
  if (blocks > 0x7fffffffLL || joins > 0x7fffffffLL) { set_error("adapters: too many adapters and columns for one launch"); return SMOE_ERR_RANGE; }
  if (blocks > 0) {
    if (grad_ranks(r) == 1) hipLaunchKernelGGL((adapter_grad_kernel<T, 1>), dim3((unsigned)blocks), dim3(GRAD_NW * 64), 0, st, p);
    else hipLaunchKernelGGL((adapter_grad_kernel<T, 2>), dim3((unsigned)blocks), dim3(GRAD_NW * 64), 0, st, p);
    if (int rc = launch_status("adapter_grad_kernel")) return rc;
  }
  if (joins == 0) return 0;
  hipLaunchKernelGGL(adapter_grad_join_kernel<T>, dim3((unsigned)joins), dim3(256), 0, st, p);
  return launch_status("adapter_grad_join_kernel");
}
template <typename T>
static int grad_any_t(const AdapterGradArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(adapter_grad_any_kernel<T>, dim3((a.C + 63) / 64, a.R), dim3(256), 0, st, a);
  return launch_status("adapter_grad_any_kernel");
}

// ---- the launches of a call, over one workspace ------------------------------------------------------------------------
static int low(const AdapterLowArgs& a, int dtype, hipStream_t st) {
  return dtype == SMOE_F32 ? low_t<float>(a, st) : dtype == SMOE_BF16 ? low_t<bf16_t>(a, st) : low_t<f16_t>(a, st);
}
static int project(const AdapterProjectArgs& a, int dtype, hipStream_t st) {
  int rc = 0;
  if (try_adapter_tiles(a, dtype, st, rc)) return rc;
  return dtype == SMOE_F32 ? project_t<float>(a, st) : dtype == SMOE_BF16 ? project_t<bf16_t>(a, st) : project_t<f16_t>(a, st);
}
// Gradients that go into the launch together; one narrower than a piece goes by itself
static int grads(const AdapterGradArgs* of, void* const* workspace, int n, int dtype, hipStream_t st) {
  GradPair pair = {};
  int rank = 1;
  for (int i = 0; i < n; ++i) {
    const AdapterGradArgs& a = of[i];
    if (a.C < pieces(dtype)) {
      const int rc = dtype == SMOE_F32 ? grad_any_t<float>(a, st) : dtype == SMOE_BF16 ? grad_any_t<bf16_t>(a, st) : grad_any_t<f16_t>(a, st);
      if (rc) return rc;
      continue;
    }
    rank = a.r;
    pair.of[i] = GradLaunch{a, grad_slices(a.T, a.C, a.r, a.R, dtype), grad_tiles(a.C, dtype), (int)cdiv64(a.r, 16 * grad_ranks(a.r)), (float*)workspace[i]};
  }
  return dtype == SMOE_F32 ? grad_t<float>(pair, rank, st) : dtype == SMOE_BF16 ? grad_t<bf16_t>(pair, rank, st) : grad_t<f16_t>(pair, rank, st);
}
static int pack(const AdapterPackArgs& a, const AdapterPackArgs& b, int dtype, hipStream_t st) {
  const int64_t tiles = a.all_tiles() + b.all_tiles();
  if (tiles > 0x7fffffffLL) { set_error("adapters: factors too large to copy"); return SMOE_ERR_RANGE; }
  if (tiles == 0) return 0;
  const dim3 grid((unsigned)tiles), block(256);
  const AdapterPacks p{{a, b}};
  if (dtype == SMOE_F32) hipLaunchKernelGGL(adapter_pack_kernel<float>, grid, block, 0, st, p);
  else if (dtype == SMOE_BF16) hipLaunchKernelGGL(adapter_pack_kernel<bf16_t>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(adapter_pack_kernel<f16_t>, grid, block, 0, st, p);
  return launch_status("adapter_pack_kernel");
}

// Pieces of the workspace, each at a multiple of 256 bytes.  Without one (a dry run) it only counts, and nothing is launched.
struct Space {
  char* base;
  size_t used = 0;
  bool dry() const { return base == nullptr; }
  template <typename T> T* take(int64_t n) {
    T* p = dry() ? nullptr : (T*)(base + used);
    used += ((size_t)n * sizeof(T) + 255) / 256 * 256;
    return p;
  }
  char* bytes(int64_t n) { return take<char>(n); }
};
static int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
static int64_t width(int dtype) { return dtype == SMOE_F32 ? 4 : 2; }

static int order_rows(const int64_t* ids, int64_t T, int R, int64_t* idx, int64_t* off, Space& s, hipStream_t st) {
  int64_t* eid = s.take<int64_t>(T);
  char* ws = s.bytes((int64_t)route_workspace_bytes(T, R + 1));
  if (s.dry()) return 0;
  return launch_route_adapters(ids, T, R, eid, idx, off, ws, st);
}

// Y = X W^T (+ bias) + U B[a]^T with U = s A[a] X, for factors in any order: the product both ways.  `off` (with the rows in order):
// factors whose contraction is not contiguous, or not whole pieces, are copied, those of adapters that have rows.
struct Product {
  const void* X; int64_t sxm;
  const void* W; int64_t swn, swk;
  const void* bias;
  const void* A; int64_t sar, saj, sak;
  const void* B; int64_t sbr, sbn, sbj;
  void* Y;                                           // NULL: U alone
  float* U;
  int64_t K, N;
};
// Rows from which 16-bit products go in tiles, fewer where there is more to do: the rows' own kernel reads the weights once per 32
// rows, but has a workgroup per 16 columns (us of a call, row by row / tiles: 80 rows, 4096 -> 4096 33 / 42; 128 rows 40 / 42; 256
// rows 63 / 43; 100 rows, 2048 -> 2048 18 / 28; 300 rows, 512 -> 512 13 / 17; 777 rows, 2880 -> 2880 93 / 42)
static constexpr int64_t TILES_MIN_ROWS = 320, TILES_MIN_WORK = 2000000000;
// ... and a shared weight whose contraction is strided (dx) would be copied for the rows' kernel: tiles earlier, where the copy is
// long and there are tiles enough (us of a backward call, row by row / tiles: 65 rows, 4096 -> 4096 65 / 51; 120, 2880 -> 2880 69 / 55;
// 300, 2048 -> 2048 47 / 37; 128, 768 -> 8192 101 / 40; but 300, 512 -> 512 19 / 22; 65, 8192 -> 768 63 / 85)
static constexpr int64_t COPY_MIN = 1 << 22, COPY_MIN_TILES = 32;
static int product(const AdapterCall& c, Product p, const int64_t* idx, const int64_t* off, Space& s, hipStream_t st) {
  const bool many = c.T > ADAPTER_FEW_ROWS;
  const bool long_copy = p.swk != 1 && p.N * p.K >= COPY_MIN && cdiv64(c.T, 64) * cdiv64(p.N, 128) >= COPY_MIN_TILES;
  const bool tiles = c.dtype != SMOE_F32 && p.K >= 8 && (c.T > TILES_MIN_ROWS || (many && (long_copy || c.T * p.N * p.K > TILES_MIN_WORK)));
  const AdapterF32 f32 = c.dtype == SMOE_F32 ? adapter_f32_class(c.T, p.K, p.N, p.swk != 1) : ADAPTER_F32_ROWS;
  const int64_t w = width(c.dtype);
  // The copies, at most the factors' and those of the shared product, in pairs
  AdapterPackArgs copies[4] = {};
  int n = 0;
  auto copy = [&](const void*& src, int64_t& s0, int64_t& s1, int64_t& s2, int64_t n0, int64_t n1, int64_t n2, int64_t ld) {
    char* dst = s.bytes(n0 * n1 * ld * w);
    copies[n++] = AdapterPackArgs{src, s0, s1, s2, dst, (int)ld, n0 == 1 ? nullptr : off, (int)n0, (int)n1, (int)n2};
    src = dst;
    s0 = n1 * ld, s1 = ld, s2 = 1;
  };
  int64_t zero = 0, one = 1;
  // (also where the rows are few; us of a backward call, bf16, elements looked up where they lie / copied first: 1 row 4096 -> 4096,
  // rank 16 87 / 50; 64 rows 1024 -> 1024 31 / 24; 16 rows 2048 -> 2048, rank 64 159 / 85)
  if (p.sak != 1 && p.K >= pieces(c.dtype)) copy(p.A, p.sar, p.saj, p.sak, c.R, c.r, p.K, p.K);
  const void* X = p.X;
  int64_t sxm = p.sxm, K = p.K;
  if (p.Y != nullptr && tiles) {
    K = up8(p.K);
    if (p.sbj != 1 || c.r % 8) copy(p.B, p.sbr, p.sbn, p.sbj, c.R, p.N, c.r, up8(c.r));
    const bool w_tr = p.swn == 1 && p.swk != 1;
    if (p.K % 8 || (w_tr && p.N % 8)) copy(p.W, zero, p.swn, p.swk, 1, p.N, p.K, K);
    if (p.K % 8) copy(X, zero, sxm, one, 1, c.T, p.K, K);
  } else if (p.Y != nullptr && f32 == ADAPTER_F32_ROWS && p.swk != 1 && p.K >= pieces(c.dtype)) {
    copy(p.W, zero, p.swn, p.swk, 1, p.N, p.K, p.K);
  }
  for (int i = 0; i < n && !s.dry(); i += 2)
    if (int rc = pack(copies[i], copies[i + 1], c.dtype, st)) return rc;
  const int rp = (c.r + 31) / 32 * 32;
  char* planes = tiles ? s.bytes(c.T * 2 * rp * w) : nullptr;
  int* slots = tiles ? s.take<int>(adapter_fragments(c.T, c.R) * 17) : nullptr;
  float* parts = f32 == ADAPTER_F32_RUNS ? s.take<float>(adapter_f32_parts()) : nullptr;
  int* exponents = tiles && c.dtype == SMOE_F16 ? s.take<int>(adapter_fragments(c.T, c.R) * rp) : nullptr;
  if (!s.dry()) {
    const AdapterLowArgs a{p.X, p.sxm, p.A, p.sar, p.saj, p.sak, c.ids, c.scales, many ? idx : nullptr, many ? off : nullptr, p.U, planes, rp, slots, exponents,
                           c.T, (int)p.K, c.r, c.R};
    if (int rc = low(a, c.dtype, st)) return rc;
  }
  if (p.Y == nullptr) return 0;
  if (s.dry()) return 0;
  const AdapterProjectArgs a{X, sxm, p.W, p.swn, p.swk, p.bias, 1, p.U, planes, rp, slots, exponents, p.B, p.sbr, p.sbn, p.sbj, c.ids,
                             many ? idx : nullptr, p.Y, p.N, c.T, (int)K, (int)p.N, c.r, c.R};
  return f32 != ADAPTER_F32_ROWS ? launch_adapter_f32(a, f32, parts, st) : project(a, c.dtype, st);
}

static int forward(const AdapterCall& c, Space& s, hipStream_t st) {
  if (c.T > ADAPTER_FEW_ROWS)
    if (int rc = order_rows(c.ids, c.T, c.R, c.idx, c.off, s, st)) return rc;
  // (a dry run asks for all that the call may want)
  return product(c, Product{c.X, c.sxm, c.W, c.K, 1, c.bias, c.A, c.r * c.K, c.K, 1, c.B, c.N * c.r, c.r, 1, s.dry() ? &s : c.Y, c.U, c.K, c.N},
                 c.idx, c.off, s, st);
}

static int backward(const AdapterCall& c, Space& s, hipStream_t st) {
  const bool dry = s.dry(), any = dry || c.DA || c.DB;
  const int64_t *idx = c.idx, *off = c.off;
  if (c.T <= ADAPTER_FEW_ROWS && any) {
    int64_t* own = s.take<int64_t>(c.T + c.R + 1);
    if (int rc = order_rows(c.ids, c.T, c.R, own, own + c.T, s, st)) return rc;
    idx = own, off = own + c.T;
  }
  AdapterGradArgs of[2];
  void* ws[2];
  int n = 0;
  if (dry || c.DX || c.DA) {
    float* V = s.take<float>(c.T * c.r);
    const Product p{c.DY, c.N, c.W, 1, c.K, nullptr, c.B, c.N * c.r, 1, c.r, c.A, c.r * c.K, 1, c.K, dry ? &s : c.DX, V, c.N, c.K};
    if (int rc = product(c, p, idx, off, s, st)) return rc;
    if (dry || c.DA) {
      ws[n] = s.bytes((int64_t)grad_bytes(c.T, c.K, c.r, c.R, c.dtype));
      of[n++] = AdapterGradArgs{V, c.X, c.sxm, idx, off, c.DA, c.r * c.K, c.K, 1, c.T, (int)c.K, c.r, c.R};
    }
  }
  if (dry || c.DB) {
    ws[n] = s.bytes((int64_t)grad_bytes(c.T, c.N, c.r, c.R, c.dtype));
    of[n++] = AdapterGradArgs{c.U, c.DY, c.N, idx, off, c.DB, c.N * c.r, 1, c.r, c.T, (int)c.N, c.r, c.R};
  }
  if (n > 0 && !dry)
    if (int rc = grads(of, ws, n, c.dtype, st)) return rc;
  if (dry || c.DBIAS) {
    ws[0] = s.bytes((int64_t)grad_bytes(c.T, c.N, 1, 1, c.dtype));
    of[0] = AdapterGradArgs{nullptr, c.DY, c.N, nullptr, nullptr, c.DBIAS, 0, 0, 1, c.T, (int)c.N, 1, 1};
    if (!dry) return grads(of, ws, 1, c.dtype, st);
  }
  return 0;
}

size_t adapter_workspace_bytes(const AdapterCall& call, bool back) {
  AdapterCall c{};                                           // (its sizes alone)
  c.T = call.T, c.K = call.K, c.N = call.N, c.r = call.r, c.R = call.R, c.dtype = call.dtype;
  Space s{nullptr};
  if (back) backward(c, s, nullptr);
  else forward(c, s, nullptr);
  return s.used;
}
int launch_adapter_call(const AdapterCall& c, bool back, void* workspace, hipStream_t st) {
  static char none;
  Space s{workspace ? (char*)workspace : &none};
  return back ? backward(c, s, st) : forward(c, s, st);
}

}  // namespace smoe
