// A whole gated mixture-of-experts layer for a few tokens, from the tokens to the layer's output:
//   l[t, e] = sum_c X[t, c] WR[e, c]                        (float32; returned)
//   S[t, :] = the k largest of l[t, :],  g[t, j] = softmax(l[t, :])[S[t, j]]  (divided by their sum when renormalised)
//   h[t, j] = a * silu(b),  (a, b) the halves of W1[e] X[t] + b1[e],  e = S[t, j]
//   OUT[t]  = sum_j g[t, j] (W2[e] h[t, j] + b2[e])
// in three launches up to 4 tokens (logits; hidden rows, selection inside; output) and five beyond (logits, selection, hidden rows,
// output rows, their sum).  Every sum and gate stays in float32; hidden values are the sum of two of the operand's type (few_rows.hpp,
// split): bfloat16 2^-18 of the value off, float16 2^-24 or 2^-25 in all, infinite where float16 is, as in the general path.  So
// whatever the weights' layout: what a token gets does not depend on it.
//
// What bounds it: the weights of the experts that were hit, read from memory once (counted: 471 + 236 MB for 1 token, 2 of 8 experts,
// 4096 / 14336, 942 + 477 for 17 tokens, 4 of 32, 2880 / 2880); a kernel that only reads reaches 6.3 to 6.75 TB/s here.
// us, all launches (weights at TB/s): 1 token, 8 of 128 experts, 2048 / 768 24.2 (3.1; launches that depend on each other);
// 1 token, 2 of 8, 4096 / 14336 118 (6.0); 17 tokens, 4 of 32, 2880 / 2880 222 (6.4); 64 tokens, 8 of 128, 2048 / 768 220 (5.4).
//
// Counterpart in the reference: the router, softmax and top-k of its Hugging Face injection (scattermoe/utils/replace_moe.py:60-95)
// and GLUMLP.forward (scattermoe/mlp.py:74-95) behind them.
#include "few_rows.hpp"
#include "router_select.hpp"
#include <algorithm>

namespace smoe {

// This lane's share of the dot product of two strided vectors
template <typename A, typename B>
__device__ __forceinline__ float lane_dot(const A* __restrict__ a, int64_t sa, const B* __restrict__ b, int64_t sb, int n) {
  float v = 0.0f;
  for (int i = lane_id(); i < n; i += 64) v = fmaf(to_f32(a[i * sa]), to_f32(b[i * sb]), v);
  return v;
}

// ---- routing --------------------------------------------------------------------------------------------------------
// The logits of DOT_ROWS experts and one token by a workgroup.  Bound by latency: 1 token, 128 experts of 2048 4.1 us, 64 tokens 7.8 us
// (33 MB read from the caches).
template <typename T>
__global__ __launch_bounds__(DOT_NW * 64) void layer_logits_kernel(RoutedLayerArgs a) {
  __shared__ float part[DOT_NW * DOT_ROWS];
  const int t = blockIdx.y, e0 = blockIdx.x * DOT_ROWS;
  const T* x = (const T*)a.X + t * a.sxm;
  const T* w[DOT_ROWS];
#pragma unroll
  for (int j = 0; j < DOT_ROWS; ++j) w[j] = (const T*)a.WR + min(e0 + j, a.E - 1) * a.sre;
  if (a.sxk == 1 && a.srk == 1 && a.d >= Few<T>::PER) {
    const float v = dot_rows<T>(x, w, a.d, part);
    if (threadIdx.x < DOT_ROWS && e0 + (int)threadIdx.x < a.E) a.LOGITS[(int64_t)t * a.E + e0 + threadIdx.x] = v;
  } else {
    const int j = threadIdx.x >> 6;                          // a wave per expert
    const float v = wave_sum(lane_dot(x, a.sxk, (const T*)a.WR + min(e0 + j, a.E - 1) * a.sre, a.srk, a.d));
    if (lane_id() == 0 && e0 + j < a.E) a.LOGITS[(int64_t)t * a.E + e0 + j] = v;
  }
}

// Selection of token t by one wave (64 tokens, 8 of 128 experts 5.5 us, k rounds of a maximum across the wave); `expert(j, e)` and the returned gates as select_experts
template <class Expert>
__device__ __forceinline__ float layer_select(const RoutedLayerArgs& a, int t, Expert expert) {
  const float* l = a.LOGITS + (int64_t)t * a.E;
  return select_experts(a.E, a.k, a.renorm != 0, [&](int e) { return l[e]; }, [](float v) { return expf(v); }, expert);
}
__global__ __launch_bounds__(64) void layer_select_kernel(RoutedLayerArgs a) {
  const int t = blockIdx.x;
  const float g = layer_select(a, t, [&](int j, int e) { a.experts[t * a.k + j] = e; });
  if (lane_id() < a.k) a.gates[t * a.k + lane_id()] = g;
}

static_assert(DOT_NW == DOT_ROWS, "any layout: a wave per expert");

// Hidden values are held as two parts of the operand's type (float32: one)
template <typename T> static constexpr int HIDDEN_PARTS = sizeof(T) == 4 ? 1 : 2;

// ---- any layout: one wave per hidden value, one wave per output value ----------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void layer_hidden_any_kernel(RoutedLayerArgs a) {
  const int f = blockIdx.x * 4 + (threadIdx.x >> 6), row = blockIdx.y;
  if (f >= a.F) return;
  const int e = a.experts[row];
  const T* x = (const T*)a.X + row / a.k * a.sxm;
  const T* w = (const T*)a.W1 + e * a.sw1e;
  float first = wave_sum(lane_dot(x, a.sxk, w + f * a.sw1n, a.sw1k, a.d));
  float second = wave_sum(lane_dot(x, a.sxk, w + (f + a.F) * a.sw1n, a.sw1k, a.d));
  if (a.b1) {
    const T* b = (const T*)a.b1 + e * a.sb1e;
    first += to_f32(b[f * a.sb1n]);
    second += to_f32(b[(f + a.F) * a.sb1n]);
  }
  if (lane_id() == 0) {
    float v = (a.act & 1) ? glu_h(a.act, first, second) : glu_h(a.act, second, first);
    if constexpr (HIDDEN_PARTS<T> == 2) {
      T part, rest;
      split<T>(v, part, rest);
      v = to_f32(part) + to_f32(rest);
    }
    a.hidden[(int64_t)row * a.F + f] = v;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void layer_out_any_kernel(RoutedLayerArgs a) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), t = blockIdx.y;
  if (n >= a.d) return;
  float sum = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    const int row = t * a.k + j, e = a.experts[row];
    float v = wave_sum(lane_dot((const T*)a.W2 + e * a.sw2e + n * a.sw2n, a.sw2k, a.hidden + (int64_t)row * a.F, 1, a.F));
    if (a.b2) v += to_f32(((const T*)a.b2)[e * a.sb2e + n * a.sb2n]);
    sum = fmaf(a.gates[row], v, sum);
  }
  if (lane_id() == 0) ((T*)a.OUT)[t * a.som + n] = from_f32<T>(sum);
}

// ---- contiguous rows: streams over the weights of the experts that were hit ----------------------------------------
// The rows (token, slot) by expert, put together by every workgroup for itself (at most 512 ids; a launch for it would cost
// more than the workgroups wait).  The order of an expert's rows among themselves is whatever the LDS atomics make it: a row's
// values do not depend on its place, since all passes over an expert's rows have one form.
struct RowLists {
  int count[512], first[513], rows[SMOE_FEW_ROWS], hit[512], hits;
};
template <int NT>
__device__ __forceinline__ void list_rows(const int* __restrict__ experts, int L, int E, RowLists& s) {
  for (int e = threadIdx.x; e < E; e += NT) s.count[e] = 0;
  __syncthreads();
  int e[(SMOE_FEW_ROWS + NT - 1) / NT], rank[(SMOE_FEW_ROWS + NT - 1) / NT];
#pragma unroll
  for (int u = 0; u < (SMOE_FEW_ROWS + NT - 1) / NT; ++u) {
    const int i = u * NT + threadIdx.x;
    if (i < L) {
      e[u] = experts[i];
      rank[u] = atomicAdd(&s.count[e[u]], 1);
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    int before = 0, hits = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int x = e0 + (int)threadIdx.x, n = x < E ? s.count[x] : 0;
      const int incl = wave_scan(n);
      if (x < E) s.first[x] = before + incl - n;
      const unsigned long long some = __ballot(n > 0);
      if (n > 0) s.hit[hits + __popcll(some & ((1ull << threadIdx.x) - 1))] = x;
      hits += __popcll(some);
      before += __builtin_amdgcn_readlane(incl, 63);
    }
    if (threadIdx.x == 0) s.hits = hits;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < (SMOE_FEW_ROWS + NT - 1) / NT; ++u) {
    const int i = u * NT + threadIdx.x;
    if (i < L) s.rows[s.first[e[u]] + rank[u]] = i;
  }
  __syncthreads();
}

// Hidden rows, `ldh` elements of every part: a workgroup of four waves has ROWS weight rows (each hidden value's two next to each other) of one expert's
// rows; the waves take the contraction's blocks in turn and are added up in LDS.  Two weight rows of each hidden value meet in one
// workgroup, so its halves need no trip through memory.  us (weights at TB/s): 1 token, 2048 -> 2 x 768, 8 experts 14.0 (3.6); 1 token,
// 4096 -> 2 x 14336, 2 experts 75.9 (6.2); 17 tokens, 2880 -> 2 x 2880, 29 experts 139 (6.8); 64 tokens, 126 experts 132 (6.1).
static constexpr int HID_NW = 4, FEWEST = 4;
static_assert(FEWEST <= HID_NW, "a wave per token");
template <typename T, int P, int G, int ROWS>
__device__ __forceinline__ void hidden_tile(const RoutedLayerArgs& a, int e, int f0, const int* rows, int M, float* part) {
  constexpr int INPUTS = G * 16 / P;
  const T* W = (const T*)a.W1 + e * a.sw1e;
  few_tile<T, P, G, 1, HID_NW, ROWS, true, P == 4 && ROWS == 16 ? 4 : G == 4 ? 2 : 0>([&](int n) { return W + (min(f0 + (n >> 1), a.F - 1) + (n & 1 ? a.F : 0)) * a.sw1n; },
                                         [&](int m) { return (const T*)a.X + rows[min(m, M - 1)] / a.k * a.sxm; }, 0, a.d, part);
  __syncthreads();
  const T* b1 = a.b1 ? (const T*)a.b1 + e * a.sb1e : nullptr;
  for (int p = threadIdx.x; p < ROWS / 2 * INPUTS; p += HID_NW * 64) {
    const int m = p / (ROWS / 2), c = p % (ROWS / 2), f = f0 + c;
    if (m >= M || f >= a.F) continue;
    float first = few_sum<HID_NW, ROWS, INPUTS>(part, 2 * c, m), second = few_sum<HID_NW, ROWS, INPUTS>(part, 2 * c + 1, m);
    T* out = (T*)a.hidden + (int64_t)rows[m] * HIDDEN_PARTS<T> * a.ldh + f;
    if (b1) {
      first += to_f32(b1[f * a.sb1n]);
      second += to_f32(b1[(f + a.F) * a.sb1n]);
    }
    const float v = (a.act & 1) ? glu_h(a.act, first, second) : glu_h(a.act, second, first);
    if constexpr (HIDDEN_PARTS<T> == 2) split<T>(v, out[0], out[a.ldh]);
    else out[0] = v;
  }
}

// GROUPS: 0 for up to 4 tokens, else the groups of 8 rows that a pass over an expert's weights takes (row_groups).  Up to 4 tokens
// every workgroup makes their selections for itself, a wave each, out of the logits (the first one leaves them to the
// output's launch): a launch for that would cost more.
template <typename T, int GROUPS, int ROWS>
__global__ __launch_bounds__(HID_NW * 64, GROUPS > 2 ? 2 : GROUPS == 2 ? 3 : 4) void layer_hidden_kernel(RoutedLayerArgs a) {
  constexpr bool MANY = GROUPS > 0;
  __shared__ float part[FEW_PART<HID_NW, ROWS, MANY ? GROUPS * 8 : 4>];
  __shared__ RowLists s;
  __shared__ int mine[MANY ? 1 : FEWEST * 64];
  if constexpr (!MANY) {
    const int t = threadIdx.x >> 6;
    if (t < a.T) {
      const float g = layer_select(a, t, [&](int j, int e) { mine[t * a.k + j] = e; });
      if (blockIdx.x == 0 && blockIdx.y == 0 && lane_id() < a.k) {
        a.gates[t * a.k + lane_id()] = g;
        a.experts[t * a.k + lane_id()] = mine[t * a.k + lane_id()];
      }
    }
    __syncthreads();
  }
  if constexpr (!MANY) {
    if (a.T == 1) {                                          // (a token's experts are all different)
      const int row = blockIdx.y;
      hidden_tile<T, 4, 1, ROWS>(a, mine[row], blockIdx.x * (ROWS / 2), &row, 1, part);
      return;
    }
  }
  list_rows<HID_NW * 64>(MANY ? a.experts : mine, a.T * a.k, a.E, s);
  if ((int)blockIdx.y >= s.hits) return;
  const int e = s.hit[blockIdx.y], f0 = blockIdx.x * (ROWS / 2);
  const int* rows = s.rows + s.first[e];
  if constexpr (MANY) {
    // (the form goes by all of the expert's rows, not by those that are left: forms sum in orders of their own)
    const int count = s.count[e];
    for (int M = count;;) {
      if (GROUPS == 1 || count <= 8) hidden_tile<T, 2, 1, ROWS>(a, e, f0, rows, min(M, 8), part);
      else if (GROUPS == 2 || count <= 16) hidden_tile<T, 2, GROUPS == 1 ? 1 : 2, ROWS>(a, e, f0, rows, min(M, 16), part);
      else hidden_tile<T, 2, GROUPS, ROWS>(a, e, f0, rows, min(M, 8 * GROUPS), part);
      if ((M -= 8 * GROUPS) <= 0) break;
      rows += 8 * GROUPS;
      __syncthreads();
    }
  } else {
    hidden_tile<T, 4, 1, ROWS>(a, e, f0, rows, s.count[e], part);
  }
}

// Output, more than 4 tokens: tiles as the hidden rows', TILE_COLS output columns of one expert's rows each, left times their gates in
// float32; the join adds up a token's rows in the order of their slots, so that no atomics decide it.  (Rows of T * k * d sums written
// and read are a few percent of the weights.)  us (weights at TB/s): 17 tokens, 2880 -> 2880, 29 experts 73.2 (6.6); 64 tokens,
// 768 -> 2048, 126 experts 76.0 (5.2: one or two blocks of the contraction per wave) and 4.9 for the join.
static constexpr int TILE_NW = 4;
template <typename T, int P, int G, int TILE_COLS>
__device__ __forceinline__ void out_tile(const RoutedLayerArgs& a, int e, int n0, const int* rows, int M, float* part) {
  constexpr int INPUTS = G * 16 / P, H = HIDDEN_PARTS<T>;
  const T* W = (const T*)a.W2 + e * a.sw2e;
  few_tile<T, P, G, H, TILE_NW, TILE_COLS, true, G == 4 ? 2 : 0>([&](int n) { return W + min(n0 + n, a.d - 1) * a.sw2n; },
                                           [&](int m) { return (const T*)a.hidden + (int64_t)rows[min(m, M - 1)] * H * a.ldh; }, a.ldh,
                                           a.F, part);
  __syncthreads();
  for (int p = threadIdx.x; p < TILE_COLS * INPUTS; p += TILE_NW * 64) {
    const int m = p / TILE_COLS, c = p % TILE_COLS, n = n0 + c;
    if (m >= M || n >= a.d) continue;
    float v = few_sum<TILE_NW, TILE_COLS, INPUTS>(part, c, m);
    if (a.b2) v += to_f32(((const T*)a.b2)[e * a.sb2e + n * a.sb2n]);
    a.out_rows[(int64_t)rows[m] * a.d + n] = a.gates[rows[m]] * v;
  }
}
template <typename T, int GROUPS, int TILE_COLS>
__global__ __launch_bounds__(TILE_NW * 64, GROUPS > 2 ? 2 : GROUPS == 2 ? 3 : 4) void layer_out_tiles_kernel(RoutedLayerArgs a) {
  __shared__ float part[FEW_PART<TILE_NW, TILE_COLS, GROUPS * 8>];
  __shared__ RowLists s;
  list_rows<TILE_NW * 64>(a.experts, a.T * a.k, a.E, s);
  if ((int)blockIdx.y >= s.hits) return;
  const int e = s.hit[blockIdx.y], n0 = blockIdx.x * TILE_COLS;
  const int* rows = s.rows + s.first[e];
  const int count = s.count[e];
  for (int M = count;;) {
    if (GROUPS == 1 || count <= 8) out_tile<T, 2, 1, TILE_COLS>(a, e, n0, rows, min(M, 8), part);
    else if (GROUPS == 2 || count <= 16) out_tile<T, 2, GROUPS == 1 ? 1 : 2, TILE_COLS>(a, e, n0, rows, min(M, 16), part);
    else out_tile<T, 2, GROUPS, TILE_COLS>(a, e, n0, rows, min(M, 8 * GROUPS), part);
    if ((M -= 8 * GROUPS) <= 0) break;
    rows += 8 * GROUPS;
    __syncthreads();
  }
}
template <typename T>
__global__ __launch_bounds__(256) void layer_join_kernel(RoutedLayerArgs a) {
  const int t = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  if (n >= a.d) return;
  float v = 0.0f;
  for (int j = 0; j < a.k; ++j) v += a.out_rows[(int64_t)(t * a.k + j) * a.d + n];
  ((T*)a.OUT)[t * a.som + n] = from_f32<T>(v);
}

// Output, up to 4 tokens: a workgroup has COLS output columns of all tokens.  The blocks of the contraction over all hit
// experts are dealt to its waves in pieces of equal length; a wave adds what its share of an expert gives, times the gates, to
// sums of its own per token in LDS, and the waves' sums are added up at the end in their order.  us (weights at TB/s): 1 token,
// 768 -> 2048, 8 experts 7.3 (3.4); 14336 -> 4096, 2 experts 37.8 (6.2).
static constexpr int OUT_NW = 8;
template <int COLS> static constexpr int OUT_LD = COLS + 4;
template <typename T, int COLS> static constexpr int OUT_BLOCK = 8192 / COLS / (int)sizeof(T);          // eight loads of a wave
template <typename T, int COLS>
__device__ __forceinline__ void out_share(const RoutedLayerArgs& a, int e, const int* rows, int M, int n0, int b0, int b1, float* sums) {
  typedef FewLane<T, 4> Lane;
  constexpr int H = HIDDEN_PARTS<T>, NT = COLS / Lane::ROWS, STEP = Lane::STEP, BLOCK = OUT_BLOCK<T, COLS>, SIDE = BLOCK / STEP;
  const Lane l;
  const T* w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) w[j] = (const T*)a.W2 + e * a.sw2e + min(n0 + j * Lane::ROWS + l.sub, a.d - 1) * a.sw2n + l.at;
  const T* x = (const T*)a.hidden + (int64_t)rows[min(l.sub, M - 1)] * H * a.ldh + l.at;
  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto block = [&](int k0, auto load) {
    i32x4 wv[NT][SIDE], xv[H][SIDE];
#pragma unroll
    for (int s = 0; s < SIDE; ++s) {
#pragma unroll
      for (int j = 0; j < NT; ++j) wv[j][s] = load(w[j], k0 + s * STEP, std::true_type());
#pragma unroll
      for (int p = 0; p < H; ++p) xv[p][s] = load(x + p * a.ldh, k0 + s * STEP, std::false_type());
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < SIDE; ++s)
#pragma unroll
      for (int p = 0; p < H; ++p)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = Few<T>::mma(wv[j][s], xv[p][s], acc[j]);
  };
  const int whole = min(b1, a.F / BLOCK);
#pragma unroll 1
  for (int b = b0; b < whole; ++b) block(b * BLOCK, [&](const T* p, int k, auto once) { return load_piece<T, decltype(once)::value>(p + k); });
  if (whole < b1) block(whole * BLOCK, [&](const T* p, int k, auto) { return load_piece_of<T>(p + k, a.F - k - l.at); });
  const int row = rows[min(l.sub, M - 1)];
  const float g = a.gates[row];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float v[1];
    FewSums<4>::take(acc[j], l.part, v);
    const int n = j * Lane::ROWS + l.q;
    if (l.part != 0 || l.sub >= M) continue;
    if (a.b2 && b0 == 0 && n0 + n < a.d) v[0] += to_f32(((const T*)a.b2)[e * a.sb2e + (n0 + n) * a.sb2n]);
    float* to = sums + row / a.k * OUT_LD<COLS> + n;
    *to = fmaf(g, v[0], *to);
  }
}

template <typename T, int COLS>
__global__ __launch_bounds__(OUT_NW * 64) void layer_out_kernel(RoutedLayerArgs a) {
  __shared__ float sums[OUT_NW][FEWEST * OUT_LD<COLS>];
  __shared__ RowLists s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * COLS;
  for (int i = lane_id(); i < a.T * OUT_LD<COLS>; i += 64) sums[wave][i] = 0.0f;
  if (a.T == 1) {                                            // (a token's experts are all different)
    const int i = threadIdx.x;
    if (i < a.k) {
      const int e = a.experts[i];
      s.hit[i] = e, s.rows[i] = i, s.first[e] = i, s.count[e] = 1;
    }
    if (i == 0) s.hits = a.k;
    __syncthreads();
  } else {
    list_rows<OUT_NW * 64>(a.experts, a.T * a.k, a.E, s);
  }
  constexpr int BLOCK = OUT_BLOCK<T, COLS>;
  const int nb = (a.F + BLOCK - 1) / BLOCK, total = s.hits * nb;
  const int last = (int)((int64_t)total * (wave + 1) / OUT_NW);
  for (int u = (int)((int64_t)total * wave / OUT_NW); u < last;) {
    const int h = u / nb, b0 = u - h * nb, b1 = min(nb, b0 + last - u);
    const int e = s.hit[h];
    out_share<T, COLS>(a, e, s.rows + s.first[e], s.count[e], n0, b0, b1, sums[wave]);
    u += b1 - b0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * COLS; i += OUT_NW * 64) {
    const int t = i / COLS, n = n0 + i % COLS;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < OUT_NW; ++w) v += sums[w][t * OUT_LD<COLS> + i % COLS];
    if (n < a.d) ((T*)a.OUT)[t * a.som + n] = from_f32<T>(v);
  }
}

// The workspace: experts and gates of the T * k rows, then their hidden values, in two parts of two bytes or one of four.
static size_t rows_bytes(int64_t L) { return (size_t)(L * 4 + 255) / 256 * 256; }
static int64_t hidden_ld(int64_t F) { return (F + 7) / 8 * 8; }
static int64_t hidden_bytes(int64_t L, int64_t F) { return (L * hidden_ld(F) * (int64_t)sizeof(float) + 255) / 256 * 256; }
static bool has_out_rows(int64_t T) { return T > FEWEST; }
size_t routed_layer_workspace_bytes(int64_t T, int k, int64_t d, int64_t F) {
  const int64_t L = T * k;
  return 2 * rows_bytes(L) + hidden_bytes(L, F) + (has_out_rows(T) ? (size_t)L * d * sizeof(float) : 0);
}

static int hit_experts(const RoutedLayerArgs& a) { return std::min(a.E, a.T * a.k); }          // at most
template <typename T, int GROUPS, int ROWS>
static int launch_hidden(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((layer_hidden_kernel<T, GROUPS, ROWS>), dim3((2 * a.F + ROWS - 1) / ROWS, hit_experts(a)), dim3(HID_NW * 64), 0, st, a);
  return launch_status("layer_hidden_kernel");
}
template <typename T, int GROUPS, int COLS>
static int launch_out_tiles(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((layer_out_tiles_kernel<T, GROUPS, COLS>), dim3((a.d + COLS - 1) / COLS, hit_experts(a)), dim3(TILE_NW * 64), 0, st, a);
  return launch_status("layer_out_tiles_kernel");
}
template <typename T, int COLS>
static int launch_out(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((layer_out_kernel<T, COLS>), dim3((a.d + COLS - 1) / COLS), dim3(OUT_NW * 64), 0, st, a);
  return launch_status("layer_out_kernel");
}
// Up to 4 tokens.  Half as much per workgroup where there would be few of them.  us, whole / half, 1 token: hidden, by workgroups of whole
// ones: 128 10.6 / 8.3 (float32, 1024 / 1024), 256 11.0 / 10.6 (2048 / 1024), 384 14.9 / 14.0 (2048 / 768), 448 19.2 / 20.8 (3584 / 1792), 512 16.4 /
// 17.2 (2560 / 2048) and 16.7 / 15.0 (2048 / 2048), 528 19.2 / 20.0 (2048 / 1408), 720 23.8 / 27.1 (2880 / 2880), 1792 75.5 / 71.7 (4096 /
// 14336); output, by workgroups of 16 columns: 64 6.2 / 4.7, 128 8.6 / 7.0, 10.2 / 8.1 and 11.0 / 8.4, 160 10.7 / 11.8, 10.2 / 11.6 and, float32, 7.8 /
// 7.5, 180 15.1 / 16.2, 224 10.9 / 11.0, 256 36.8 / 37.6 and 8.2 / 7.4.
static constexpr int FEWEST_WGS = 512;
template <typename T>
static int launch_fewest(const RoutedLayerArgs& a, hipStream_t st) {
  const int64_t tiles = (int64_t)(2 * a.F + 31) / 32 * hit_experts(a);
  if (int rc = tiles < FEWEST_WGS ? launch_hidden<T, 0, 16>(a, st) : launch_hidden<T, 0, 32>(a, st)) return rc;
  return a.d / 16 < 160 ? launch_out<T, 8>(a, st) : launch_out<T, 16>(a, st);
}
// More than 4 tokens, eight rows of an expert per pass: 16 weight rows per workgroup instead of 32, so that a wave has more of each on
// its way, where weight rows are long and, 16 bits, few rows of an expert meet them; for each product by its own rows.  us, 32 / 16,
// bytes of a weight row in brackets.  bf16, hidden: 2 of 16 experts, 1024 / 4096, 5 tokens (2048) 27.0 / 30.2; 4 of 64, 512 / 3584, 20 tokens (1024)
// 61.7 / 80.8; 4 of 64, 1792 / 1792, 20 tokens (3584) 90.3 / 89.0; 4 of 32, 2048 / 1024, 16 tokens (4096) 42.8 / 38.0; 2880 / 2880, 16 tokens (5760)
// 131.2 / 130.1; 4 of 64, 3584 / 512, 20 tokens (7168) 56.2 / 53.6; output: 2048 / 1024 (2048) 21.1 / 21.3; 512 / 3584 (7168) 32.9 / 31.4; 1024 / 4096 (8192)
// 23.5 / 17.2; many rows of an expert: 8 of 128, 2048 / 768, 64 tokens, hidden (4096) 133.9 / 136.1.  Beyond the line and slower: 2 of 8, 4096 /
// 14336, 5 tokens 205 / 213 (8192) and 108 / 119 (28672).  float32, hidden: 4 of 64, 512 / 3584 (2048) 107.9 / 122.9; 3 of 13, 1003 / 1411, 5 tokens
// (4012) 29.9 / 28.1; 8 of 128, 2048 / 768, 64 tokens (8192) 252.0 / 246.9; 2 of 16, 4096 / 1024, 16 tokens (16384) 92.2 / 76.8; output: 2048 / 768
// 132.2 / 147.9 (shorter than the line); 1003 / 1411 (5644) 21.1 / 17.0; 2880 / 2880, 12 tokens (11520) 138.3 / 130.1; slower: 4096 / 1024 (4096) 42.0 / 50.5.
static constexpr int LONG_ROW = 3500;                        // bytes
template <typename T>
static bool few_per_workgroup(const RoutedLayerArgs& a, int length) {
  return (int64_t)length * (int64_t)sizeof(T) >= LONG_ROW && (sizeof(T) == 4 || a.T * a.k <= 2 * a.E);
}
template <typename T, int GROUPS>
static int launch_streams(const RoutedLayerArgs& a, hipStream_t st) {
  if constexpr (GROUPS == 1) {
    if (int rc = few_per_workgroup<T>(a, a.d) ? launch_hidden<T, 1, 16>(a, st) : launch_hidden<T, 1, 32>(a, st)) return rc;
    if (int rc = few_per_workgroup<T>(a, a.F) ? launch_out_tiles<T, 1, 16>(a, st) : launch_out_tiles<T, 1, 32>(a, st)) return rc;
  } else {
    if (int rc = launch_hidden<T, GROUPS, 32>(a, st)) return rc;
    if (int rc = launch_out_tiles<T, GROUPS, 32>(a, st)) return rc;
  }
  hipLaunchKernelGGL(layer_join_kernel<T>, dim3((a.d + 255) / 256, a.T), dim3(256), 0, st, a);
  return launch_status("layer_join_kernel");
}

template <typename T>
static int launch_t(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(layer_logits_kernel<T>, dim3((a.E + DOT_ROWS - 1) / DOT_ROWS, a.T), dim3(DOT_NW * 64), 0, st, a);
  if (int rc = launch_status("layer_logits_kernel")) return rc;
  const bool streams = a.sxk == 1 && a.sw1k == 1 && a.sw2k == 1 && std::min(a.d, a.F) >= Few<T>::PER;
  if (streams && a.T <= FEWEST) return launch_fewest<T>(a, st);
  hipLaunchKernelGGL(layer_select_kernel, dim3(a.T), dim3(64), 0, st, a);
  if (int rc = launch_status("layer_select_kernel")) return rc;
  if (streams) {
    // Groups per pass by the rows that an expert gets on average; experts with more take several passes.  Fewer groups leave registers
    // for more waves: us of the output's launch, 64 tokens over 128 experts, 1 / 2 / 4 groups 75 / 82 / 92, 17 over 32 74 / 74 / 81.
    const int rows = a.T * a.k;
    if (rows <= 4 * a.E) return launch_streams<T, 1>(a, st);
    return rows <= 8 * a.E ? launch_streams<T, 2>(a, st) : launch_streams<T, 4>(a, st);
  }
  hipLaunchKernelGGL(layer_hidden_any_kernel<T>, dim3((a.F + 3) / 4, a.T * a.k), dim3(256), 0, st, a);
  if (int rc = launch_status("layer_hidden_any_kernel")) return rc;
  hipLaunchKernelGGL(layer_out_any_kernel<T>, dim3((a.d + 3) / 4, a.T), dim3(256), 0, st, a);
  return launch_status("layer_out_any_kernel");
}

int launch_routed_layer(RoutedLayerArgs a, void* workspace, int dtype, hipStream_t st) {
  const int64_t L = (int64_t)a.T * a.k;
  char* w = (char*)workspace;
  a.experts = (int*)w;
  a.gates = (float*)(w + rows_bytes(L));
  a.hidden = (float*)(w + 2 * rows_bytes(L));
  a.out_rows = (float*)(w + 2 * rows_bytes(L) + hidden_bytes(L, a.F));
  a.ldh = (int)hidden_ld(a.F);
  switch (dtype) {
    case SMOE_F32: return launch_t<float>(a, st);
    case SMOE_BF16: return launch_t<bf16_t>(a, st);
    case SMOE_F16: return launch_t<f16_t>(a, st);
    default: set_error("smoe_routed_glu_mlp: unknown dtype %d", dtype); return SMOE_ERR_DTYPE;
  }
}

}  // namespace smoe
