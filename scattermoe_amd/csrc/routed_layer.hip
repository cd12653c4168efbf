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
#include "router_select.hpp"

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
static constexpr int ROUTE_NT = 1024;
template <typename T>
__global__ __launch_bounds__(ROUTE_NT) void layer_route_kernel(RoutedLayerArgs a) {
  __shared__ float logits[64 * ROUTER_MAX_PER_LANE];
  const int t = blockIdx.x, wave = threadIdx.x >> 6;
  const T* x = (const T*)a.X + t * a.sxm;
  for (int e = wave; e < a.E; e += ROUTE_NT / 64) {
    const float v = wave_sum(lane_dot(x, a.sxk, (const T*)a.WR + e * a.sre, a.srk, a.d));
    if (lane_id() == 0) {
      logits[e] = v;
      a.LOGITS[(int64_t)t * a.E + e] = v;
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

// The workspace: experts and gates of the T * k rows, then their hidden values.
static size_t rows_bytes(int64_t L) { return (size_t)(L * 4 + 255) / 256 * 256; }
size_t routed_layer_workspace_bytes(int64_t T, int k, int64_t F) {
  const int64_t L = T * k;
  return 2 * rows_bytes(L) + (size_t)L * F * sizeof(float);
}

template <typename T>
static int launch_t(const RoutedLayerArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(layer_route_kernel<T>, dim3(a.T), dim3(ROUTE_NT), 0, st, a);
  if (int rc = launch_status("layer_route_kernel")) return rc;
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
  switch (dtype) {
    case SMOE_F32: return launch_t<float>(a, st);
    case SMOE_BF16: return launch_t<bf16_t>(a, st);
    case SMOE_F16: return launch_t<f16_t>(a, st);
    default: set_error("smoe_routed_glu_mlp: unknown dtype %d", dtype); return SMOE_ERR_DTYPE;
  }
}

}  // namespace smoe
