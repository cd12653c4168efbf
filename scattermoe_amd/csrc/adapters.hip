// Low-rank adapters of many requests beside a shared projection.  Row t carries the adapter a = ids[t]; a row whose id
// lies outside [0, R) carries none:
//   U[t] = s[a] A[a] X[t]                 (r values, float32)
//   Y[t] = W X[t] + bias + B[a] U[t]
// The backward pass is made of the same two products with the factors exchanged (V[t] = s[a] B[a]^T DY[t],
// DX[t] = W^T DY[t] + A[a]^T V[t]) and of the adapters' own gradients, sums over the rows that carry them:
//   DA[a] = sum_t V[t] X[t]^T,   DB[a] = sum_t DY[t] U[t]^T.
//
// The reference has no counterpart; the rows pick their weights by id as in scattermoe/parallel_experts.py:148-182.
#include "common.hpp"

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
  const int64_t t0 = (int64_t)blockIdx.y * PBM;
  const int n0 = blockIdx.x * PBN, tid = threadIdx.x;
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
  const int64_t lo = id ? a.off[id - 1] : 0, hi = a.off[id];
  for (int j0 = 0; j0 < a.r; j0 += GRAD_RANKS) {
    float acc[GRAD_RANKS] = {};
    for (int64_t i = lo + wave; i < hi; i += 4) {
      const int64_t t = a.idx ? a.idx[i] : i;
      const float m = c < a.C ? to_f32(((const T*)a.M)[t * a.smm + c]) : 0.0f;
#pragma unroll
      for (int j = 0; j < GRAD_RANKS; ++j)
        if (j0 + j < a.r) acc[j] = fmaf(a.P[t * a.r + j0 + j], m, acc[j]);
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

template <typename T>
static int low_t(const AdapterLowArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(adapter_low_any_kernel<T>, dim3((unsigned)a.T), dim3(256), 0, st, a);
  return launch_status("adapter_low_any_kernel");
}
template <typename T>
static int project_t(const AdapterProjectArgs& a, hipStream_t st) {
  const int64_t rows = cdiv64(a.T, PBM);
  if (rows > 65535) { set_error("smoe_adapter_project: too many rows for this layout"); return SMOE_ERR_RANGE; }
  hipLaunchKernelGGL(adapter_project_any_kernel<T>, dim3((a.N + PBN - 1) / PBN, (unsigned)rows), dim3(PT), 0, st, a);
  return launch_status("adapter_project_any_kernel");
}
template <typename T>
static int grad_t(const AdapterGradArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(adapter_grad_any_kernel<T>, dim3((a.C + 63) / 64, a.R), dim3(256), 0, st, a);
  return launch_status("adapter_grad_any_kernel");
}

int launch_adapter_low(const AdapterLowArgs& a, int dtype, hipStream_t st) {
  return dtype == SMOE_F32 ? low_t<float>(a, st) : dtype == SMOE_BF16 ? low_t<bf16_t>(a, st) : low_t<f16_t>(a, st);
}
int launch_adapter_project(const AdapterProjectArgs& a, int dtype, hipStream_t st) {
  return dtype == SMOE_F32 ? project_t<float>(a, st) : dtype == SMOE_BF16 ? project_t<bf16_t>(a, st) : project_t<f16_t>(a, st);
}
int launch_adapter_grad(const AdapterGradArgs& a, int dtype, hipStream_t st) {
  return dtype == SMOE_F32 ? grad_t<float>(a, st) : dtype == SMOE_BF16 ? grad_t<bf16_t>(a, st) : grad_t<f16_t>(a, st);
}

}  // namespace smoe
