// A whole gated mixture-of-experts layer for a few tokens, from the tokens to the layer's output:
//   l[t, e] = sum_c X[t, c] WR[e, c]                        (float32; returned)
//   S[t, :] = the k largest of l[t, :],  g[t, j] = softmax(l[t, :])[S[t, j]]  (divided by their sum when renormalised)
//   h[t, j] = a * silu(b),  (a, b) the halves of W1[e] X[t] + b1[e],  e = S[t, j]
//   OUT[t]  = sum_j g[t, j] (W2[e] h[t, j] + b2[e])
// in three launches: routing (one workgroup per token), hidden rows, output.  The hidden rows, like every sum, stay in
// float32; the only rounding of the layer is the output's.
//
// Counterpart in the reference: the router, softmax and top-k of its Hugging Face injection (scattermoe/utils/replace_moe.py:60-95)
// and GLUMLP.forward (scattermoe/mlp.py:74-95) behind them.
#include "few_rows.hpp"
#include "router_select.hpp"
#include <algorithm>

namespace smoe {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// This lane's share of the dot product of two strided vectors
template <typename A, typename B>
__device__ __forceinline__ float lane_dot(const A* __restrict__ a, int64_t sa, const B* __restrict__ b, int64_t sb, int n) {
  float v = 0.0f;
  for (int i = lane_id(); i < n; i += 64) v = fmaf(to_f32(a[i * sa]), to_f32(b[i * sb]), v);
  return v;
}

// ---- routing: one workgroup per token -------------------------------------------------------------------------------
static constexpr int ROUTE_NT = 1024, ROUTE_E = 4, ROUTE_P = 2;
// The logits of ROUTE_E experts by one wave, contiguous rows: ROUTE_P pieces of 64 x 16 bytes of each at a time
template <typename T>
__device__ __forceinline__ void route_dots(const T* __restrict__ x, const T* const (&w)[ROUTE_E], int d, float (&v)[ROUTE_E]) {
  constexpr int PER = Few<T>::PER;
  typedef T V __attribute__((ext_vector_type(PER)));
#pragma unroll
  for (int j = 0; j < ROUTE_E; ++j) v[j] = 0.0f;
  for (int k0 = lane_id() * PER; k0 < d; k0 += 64 * PER * ROUTE_P) {
    i32x4 xv[ROUTE_P], wv[ROUTE_E][ROUTE_P];
#pragma unroll
    for (int p = 0; p < ROUTE_P; ++p) {
      const int left = d - k0 - 64 * PER * p;
      xv[p] = load_piece_of<T>(x + k0 + 64 * PER * p, left);
#pragma unroll
      for (int j = 0; j < ROUTE_E; ++j) wv[j][p] = load_piece_of<T>(w[j] + k0 + 64 * PER * p, left);
    }
#pragma unroll
    for (int p = 0; p < ROUTE_P; ++p)
#pragma unroll
      for (int j = 0; j < ROUTE_E; ++j)
#pragma unroll
        for (int i = 0; i < PER; ++i)
          v[j] = fmaf(to_f32(__builtin_bit_cast(V, xv[p])[i]), to_f32(__builtin_bit_cast(V, wv[j][p])[i]), v[j]);
  }
#pragma unroll
  for (int j = 0; j < ROUTE_E; ++j) v[j] = wave_sum(v[j]);
}

template <typename T>
__global__ __launch_bounds__(ROUTE_NT) void layer_route_kernel(RoutedLayerArgs a) {
  __shared__ float logits[64 * ROUTER_MAX_PER_LANE];
  const int t = blockIdx.x, wave = threadIdx.x >> 6;
  const T* x = (const T*)a.X + t * a.sxm;
  for (int e0 = wave * ROUTE_E; e0 < a.E; e0 += ROUTE_NT / 64 * ROUTE_E) {
    float v[ROUTE_E];
    if (a.sxk == 1 && a.srk == 1) {
      const T* w[ROUTE_E];
#pragma unroll
      for (int j = 0; j < ROUTE_E; ++j) w[j] = (const T*)a.WR + min(e0 + j, a.E - 1) * a.sre;
      route_dots<T>(x, w, a.d, v);
    } else {
#pragma unroll
      for (int j = 0; j < ROUTE_E; ++j)
        v[j] = wave_sum(lane_dot(x, a.sxk, (const T*)a.WR + min(e0 + j, a.E - 1) * a.sre, a.srk, a.d));
    }
#pragma unroll
    for (int j = 0; j < ROUTE_E; ++j) {
      if (lane_id() == 0 && e0 + j < a.E) {
        logits[e0 + j] = v[j];
        a.LOGITS[(int64_t)t * a.E + e0 + j] = v[j];
      }
    }
  }
  __syncthreads();
  if (wave != 0) return;
  const float w = select_experts(
      a.E, a.k, a.renorm != 0, [&](int e) { return logits[e]; }, [](float v) { return expf(v); },
      [&](int j, int e) { a.experts[t * a.k + j] = e; });
  if (lane_id() < a.k) a.gates[t * a.k + lane_id()] = w;
}

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
  if (lane_id() == 0) a.hidden[(int64_t)row * a.F + f] = (a.act & 1) ? glu_h(a.act, first, second) : glu_h(a.act, second, first);
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
// values do not depend on its place.
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

// Hidden values are held as two parts of the operand's type (float32: one), rows of `ldh` elements
template <typename T> static constexpr int HIDDEN_PARTS = sizeof(T) == 4 ? 1 : 2;

// Hidden rows: a workgroup of four waves has 8 NT hidden values (16 NT weight rows, each value's two next to each other) of one
// expert's rows; the waves take the contraction's blocks in turn and are added up in LDS.
static constexpr int HID_NW = 4, HID_NT = 2;
template <typename T, int MT>
__device__ __forceinline__ void hidden_tile(const RoutedLayerArgs& a, int e, int f0, const int* rows, int M, float (*part)[64 * 4]) {
  constexpr int PER = Few<T>::PER, STEP = FEW_STEP<T>, BLOCK = FEW_BLOCK<T>;
  const int lane = lane_id(), wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const T* w[HID_NT];
  const T* x[MT];
#pragma unroll
  for (int j = 0; j < HID_NT; ++j) {
    const int f = min(f0 + 8 * j + (r >> 1), a.F - 1);
    w[j] = (const T*)a.W1 + e * a.sw1e + (f + (r & 1 ? a.F : 0)) * a.sw1n + q * PER;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = (const T*)a.X + rows[min(16 * i + r, M - 1)] / a.k * a.sxm + q * PER;
  f32x4 acc[MT][HID_NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < HID_NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int whole = a.d / BLOCK;
  for (int b = wave; b < whole; b += HID_NW) {
    const int k0 = b * BLOCK;
    constexpr int SIDE = MT > 2 ? 2 : 4;
#pragma unroll
    for (int s0 = 0; s0 < 4; s0 += SIDE) {
      i32x4 wv[HID_NT][SIDE], xv[MT][SIDE];
#pragma unroll
      for (int s = 0; s < SIDE; ++s) {
#pragma unroll
        for (int j = 0; j < HID_NT; ++j) wv[j][s] = load_piece<T, true>(w[j] + k0 + (s0 + s) * STEP);
#pragma unroll
        for (int i = 0; i < MT; ++i) xv[i][s] = load_piece<T, false>(x[i] + k0 + (s0 + s) * STEP);
      }
#pragma unroll
      for (int s = 0; s < SIDE; ++s)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < HID_NT; ++j) acc[i][j] = Few<T>::mma(wv[j][s], xv[i][s], acc[i][j]);
    }
  }
  if (wave == whole % HID_NW) {
    for (int k0 = whole * BLOCK; k0 < a.d; k0 += STEP) {
      const int left = a.d - k0 - q * PER;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const i32x4 xv = load_piece_of<T>(x[i] + k0, left);
#pragma unroll
        for (int j = 0; j < HID_NT; ++j) acc[i][j] = Few<T>::mma(load_piece_of<T>(w[j] + k0, left), xv, acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < HID_NT; ++j) *(f32x4*)(part[(wave * MT + i) * HID_NT + j] + lane * 4) = acc[i][j];
  __syncthreads();
  // lane (r, q) of group (i, j) held row 16 i + r, hidden values f0 + 8 j + 2 q and the next: first half, second half of each
  const T* b1 = a.b1 ? (const T*)a.b1 + e * a.sb1e : nullptr;
  for (int p = threadIdx.x; p < MT * HID_NT * 128; p += HID_NW * 64) {
    const int g = p >> 7, l = (p >> 1) & 63, h = p & 1;
    const int m = 16 * (g / HID_NT) + (l & 15), f = f0 + 8 * (g % HID_NT) + 2 * (l >> 4) + h;
    if (m >= M || f >= a.F) continue;
    float first = 0.0f, second = 0.0f;
#pragma unroll
    for (int v = 0; v < HID_NW; ++v) {
      const float* s = part[(v * MT) * HID_NT + g] + l * 4 + 2 * h;
      first += s[0];
      second += s[1];
    }
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

template <typename T, int MAX_MT>
__global__ __launch_bounds__(HID_NW * 64) void layer_hidden_kernel(RoutedLayerArgs a) {
  __shared__ float part[HID_NW * MAX_MT * HID_NT][64 * 4];
  __shared__ RowLists s;
  list_rows<HID_NW * 64>(a.experts, a.T * a.k, a.E, s);
  if ((int)blockIdx.y >= s.hits) return;
  const int e = s.hit[blockIdx.y], f0 = blockIdx.x * 8 * HID_NT, M = s.count[e];
  const int* rows = s.rows + s.first[e];
  if (MAX_MT == 1 || M <= 16) hidden_tile<T, 1>(a, e, f0, rows, M, part);
  else if (M <= 32) hidden_tile<T, MAX_MT == 1 ? 1 : 2>(a, e, f0, rows, M, part);
  else hidden_tile<T, MAX_MT>(a, e, f0, rows, M, part);
}

// Output: a workgroup has 16 output columns of all tokens.  The blocks of the contraction over all hit experts are dealt to
// its waves in pieces of equal length; a wave adds what its share of an expert gives, times the gates, to sums of its
// own per token in LDS, and the waves' sums are added up at the end in their order.
static constexpr int OUT_NW = 16, OUT_LD = 20;
template <typename T, int MT>
__device__ __forceinline__ void out_share(const RoutedLayerArgs& a, int e, const int* rows, int M, int n0, int b0, int b1, float* sums) {
  constexpr int PER = Few<T>::PER, STEP = FEW_STEP<T>, BLOCK = FEW_BLOCK<T>, P = HIDDEN_PARTS<T>;
  const int lane = lane_id(), r = lane & 15, q = lane >> 4;
  const T* w = (const T*)a.W2 + e * a.sw2e + min(n0 + r, a.d - 1) * a.sw2n + q * PER;
  const T* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = (const T*)a.hidden + (int64_t)rows[min(16 * i + r, M - 1)] * P * a.ldh + q * PER;
  f32x4 acc[MT][P];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int p = 0; p < P; ++p) acc[i][p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int b = b0; b < b1; ++b) {
    const int k0 = b * BLOCK;
    if (k0 + BLOCK <= a.F) {
      constexpr int SIDE = MT > 2 ? 2 : 4;
#pragma unroll
      for (int s0 = 0; s0 < 4; s0 += SIDE) {
        i32x4 wv[SIDE], xv[MT][P][SIDE];
#pragma unroll
        for (int s = 0; s < SIDE; ++s) {
          const int k = k0 + (s0 + s) * STEP;
          wv[s] = load_piece<T, true>(w + k);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int p = 0; p < P; ++p) xv[i][p][s] = *(const i32x4*)(x[i] + p * a.ldh + k);
        }
#pragma unroll
        for (int s = 0; s < SIDE; ++s)
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int p = 0; p < P; ++p) acc[i][p] = Few<T>::mma(wv[s], xv[i][p][s], acc[i][p]);
      }
    } else {
      for (int k = k0; k < a.F; k += STEP) {
        const int left = a.F - k - q * PER;
        const i32x4 wv = load_piece_of<T>(w + k, left);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int p = 0; p < P; ++p) acc[i][p] = Few<T>::mma(wv, load_piece_of<T>(x[i] + p * a.ldh + k, left), acc[i][p]);
      }
    }
  }
  // lane (r, q) holds, of row 16 i + r, columns n0 + 4 q and the next three
  f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.b2 && b0 == 0) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n0 + 4 * q + c < a.d) bias[c] = to_f32(((const T*)a.b2)[e * a.sb2e + (n0 + 4 * q + c) * a.sb2n]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = 16 * i + r;
    if (m >= M) continue;
    const int row = rows[m];
    const float g = a.gates[row];
    f32x4* to = (f32x4*)(sums + row / a.k * OUT_LD + 4 * q);
    f32x4 v = acc[i][0];
    if constexpr (P == 2) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = fmaf(acc[i][1][c], 1.0f / Few<T>::LOW, v[c]);
    }
    f32x4 old = *to;
#pragma unroll
    for (int c = 0; c < 4; ++c) old[c] = fmaf(g, v[c] + bias[c], old[c]);
    *to = old;
  }
}

template <typename T, int MAX_MT>
__global__ __launch_bounds__(OUT_NW * 64) void layer_out_kernel(RoutedLayerArgs a) {
  __shared__ __attribute__((aligned(16))) float sums[OUT_NW][MAX_MT * 16 * OUT_LD];
  __shared__ RowLists s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16;
  for (int i = lane_id(); i < a.T * OUT_LD; i += 64) sums[wave][i] = 0.0f;
  list_rows<OUT_NW * 64>(a.experts, a.T * a.k, a.E, s);
  const int nb = (a.F + FEW_BLOCK<T> - 1) / FEW_BLOCK<T>, total = s.hits * nb;
  const int last = (int)((int64_t)total * (wave + 1) / OUT_NW);
  for (int u = (int)((int64_t)total * wave / OUT_NW); u < last;) {
    const int h = u / nb, b0 = u - h * nb, b1 = min(nb, b0 + last - u);
    const int e = s.hit[h], M = s.count[e];
    const int* rows = s.rows + s.first[e];
    if (MAX_MT == 1 || M <= 16) out_share<T, 1>(a, e, rows, M, n0, b0, b1, sums[wave]);
    else if (M <= 32) out_share<T, MAX_MT == 1 ? 1 : 2>(a, e, rows, M, n0, b0, b1, sums[wave]);
    else out_share<T, MAX_MT>(a, e, rows, M, n0, b0, b1, sums[wave]);
    u += b1 - b0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * 16; i += OUT_NW * 64) {
    const int t = i >> 4, n = n0 + (i & 15);
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < OUT_NW; ++w) v += sums[w][t * OUT_LD + (i & 15)];
    if (n < a.d) ((T*)a.OUT)[t * a.som + n] = from_f32<T>(v);
  }
}

// The workspace: experts and gates of the T * k rows, then their hidden values, in two parts of two bytes or one of four.
static size_t rows_bytes(int64_t L) { return (size_t)(L * 4 + 255) / 256 * 256; }
static int64_t hidden_ld(int64_t F) { return (F + 7) / 8 * 8; }
size_t routed_layer_workspace_bytes(int64_t T, int k, int64_t F) {
  const int64_t L = T * k;
  return 2 * rows_bytes(L) + (size_t)L * hidden_ld(F) * sizeof(float);
}

template <typename T, int MAX_MT>
static int launch_streams(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((layer_hidden_kernel<T, MAX_MT>), dim3((a.F + 8 * HID_NT - 1) / (8 * HID_NT), std::min(a.E, a.T * a.k)),
                     dim3(HID_NW * 64), 0, st, a);
  if (int rc = launch_status("layer_hidden_kernel")) return rc;
  hipLaunchKernelGGL((layer_out_kernel<T, MAX_MT>), dim3((a.d + 15) / 16), dim3(OUT_NW * 64), 0, st, a);
  return launch_status("layer_out_kernel");
}

template <typename T>
static int launch_t(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(layer_route_kernel<T>, dim3(a.T), dim3(ROUTE_NT), 0, st, a);
  if (int rc = launch_status("layer_route_kernel")) return rc;
  if (a.sxk == 1 && a.sw1k == 1 && a.sw2k == 1)
    return a.T <= 16 ? launch_streams<T, 1>(a, st) : launch_streams<T, 4>(a, st);
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
  a.ldh = (int)hidden_ld(a.F);
  switch (dtype) {
    case SMOE_F32: return launch_t<float>(a, st);
    case SMOE_BF16: return launch_t<bf16_t>(a, st);
    case SMOE_F16: return launch_t<f16_t>(a, st);
    default: set_error("smoe_routed_glu_mlp: unknown dtype %d", dtype); return SMOE_ERR_DTYPE;
  }
}

}  // namespace smoe
