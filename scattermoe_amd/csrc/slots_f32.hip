// What follows the experts' rows of products in 8 bits, whose rows stay float32 until a token's are added up: the sum over a token's slots,
// weighted or not, and the gates' gradient.  A row that is rounded to 16 bits first costs as much precision as the result's own rounding
// (bf16, against 64 bits: 2.35e-3 for 1.66e-3), and float16 cannot hold one beyond 65504 that a gate below 1 brings back.  Both
// passes are bound by the rows they read, once, 16 bytes a lane: 8192 tokens x 8 rows of 2048, bf16, 571 MB in 97 us and 604 MB in 88 us (5.9 and
// 6.8 TB/s); 4099 x 2 rows of 4096, 169 MB in 33 us.
#include "eight_bit.hpp"

namespace smoe {

typedef float s_f32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Four { T v[4]; };

// out[t] = sum_j gates[t, j] rows[t k + j], one token per workgroup, four columns a thread (VEC) or one, the slots in order, four of them on
// their way.  A slot whose id is no expert's is left out, whatever its gate and its row.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void slots_combine_kernel(const float* __restrict__ Y, int64_t sy, const T* __restrict__ G, int64_t sgt, int64_t sgk,
                                                           const int64_t* __restrict__ ids, int E, T* __restrict__ O, int64_t so, int k, int N) {
  const int64_t t = blockIdx.x;
  const float* y0 = Y + t * k * sy;
  auto there = [&](int j) { return !ids || (uint64_t)ids[t * k + j] < (uint64_t)E; };
  auto gate = [&](int j) { return G ? to_f32(G[t * sgt + j * sgk]) : 1.0f; };
  if constexpr (VEC) {
    for (int c = threadIdx.x * 4; c < N; c += 1024) {
      s_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      int j = 0;
      for (; j + 4 <= k; j += 4) {
        s_f32x4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = __builtin_nontemporal_load((const s_f32x4*)(y0 + (j + u) * sy + c));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (!there(j + u)) continue;
          const float g = gate(j + u);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[q] = fmaf(g, x[u][q], acc[q]);
        }
      }
      for (; j < k; ++j) {
        const s_f32x4 x = __builtin_nontemporal_load((const s_f32x4*)(y0 + j * sy + c));
        if (!there(j)) continue;
        const float g = gate(j);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] = fmaf(g, x[q], acc[q]);
      }
      Four<T> o;
#pragma unroll
      for (int q = 0; q < 4; ++q) o.v[q] = from_f32<T>(acc[q]);
      __builtin_memcpy(__builtin_assume_aligned((char*)(O + t * so + c), 4 * sizeof(T)), &o, sizeof(o));
    }
  } else {
    for (int c = threadIdx.x; c < N; c += 256) {
      float acc = 0.0f;
      for (int j = 0; j < k; ++j)
        if (there(j)) acc = fmaf(gate(j), y0[j * sy + c], acc);
      O[t * so + c] = from_f32<T>(acc);
    }
  }
}
template <typename T>
static int slots_combine(const float* Y, int64_t sy, const void* G, int64_t sgt, int64_t sgk, const int64_t* ids, int E, void* O, int64_t so, int64_t Tn,
                         int k, int N, hipStream_t st) {
  const bool vec = ((N | sy | so) & 3) == 0 && ((uintptr_t)Y & 15) == 0 && ((uintptr_t)O & (4 * sizeof(T) - 1)) == 0;
  if (vec) slots_combine_kernel<T, true><<<(unsigned)Tn, 256, 0, st>>>(Y, sy, (const T*)G, sgt, sgk, ids, E, (T*)O, so, k, N);
  else slots_combine_kernel<T, false><<<(unsigned)Tn, 256, 0, st>>>(Y, sy, (const T*)G, sgt, sgk, ids, E, (T*)O, so, k, N);
  return launch_status("slots_combine");
}
int launch_slots_combine(const float* Y, int64_t sy, const void* G, int64_t sgt, int64_t sgk, const int64_t* ids, int E, void* O, int64_t so, int64_t Tn,
                         int k, int N, int dtype, hipStream_t st) {
  if (dtype == SMOE_BF16) return slots_combine<bf16_t>(Y, sy, G, sgt, sgk, ids, E, O, so, Tn, k, N, st);
  if (dtype == SMOE_F16) return slots_combine<f16_t>(Y, sy, G, sgt, sgk, ids, E, O, so, Tn, k, N, st);
  return slots_combine<float>(Y, sy, G, sgt, sgk, ids, E, O, so, Tn, k, N, st);
}

// dgates[t, j] = <rows[t k + j], dout[t]>: a wave per slot, whose token's other slots are read beside it (dout comes from memory once)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void slots_gate_grad_kernel(const float* __restrict__ Y, int64_t sy, const T* __restrict__ D, int64_t sd, T* __restrict__ DG,
                                                             int64_t sgt, int64_t sgk, int64_t slots, int k, int N) {
  const int64_t s = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (s >= slots) return;
  const int64_t t = s / k;
  const float* y = Y + s * sy;
  const T* d = D + t * sd;
  const int l = lane_id();
  float acc = 0.0f;
  if constexpr (VEC) {
#pragma unroll 4
    for (int c = l * 4; c < N; c += 256) {
      const s_f32x4 x = __builtin_nontemporal_load((const s_f32x4*)(y + c));
      Four<T> o;
      __builtin_memcpy(&o, __builtin_assume_aligned((const char*)(d + c), 4 * sizeof(T)), sizeof(o));
#pragma unroll
      for (int q = 0; q < 4; ++q) acc = fmaf(x[q], to_f32(o.v[q]), acc);
    }
  } else {
    for (int c = l; c < N; c += 64) acc = fmaf(y[c], to_f32(d[c]), acc);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) acc += __shfl_xor(acc, m);
  if (l == 0) DG[t * sgt + (s - t * k) * sgk] = from_f32<T>(acc);
}
template <typename T>
static int slots_gate_grad(const float* Y, int64_t sy, const void* D, int64_t sd, void* DG, int64_t sgt, int64_t sgk, int64_t Tn, int k, int N,
                           hipStream_t st) {
  const bool vec = ((N | sy | sd) & 3) == 0 && ((uintptr_t)Y & 15) == 0 && ((uintptr_t)D & (4 * sizeof(T) - 1)) == 0;
  const int64_t slots = Tn * k;
  const unsigned grid = (unsigned)((slots + 3) / 4);
  if (vec) slots_gate_grad_kernel<T, true><<<grid, 256, 0, st>>>(Y, sy, (const T*)D, sd, (T*)DG, sgt, sgk, slots, k, N);
  else slots_gate_grad_kernel<T, false><<<grid, 256, 0, st>>>(Y, sy, (const T*)D, sd, (T*)DG, sgt, sgk, slots, k, N);
  return launch_status("slots_gate_grad");
}
int launch_slots_gate_grad(const float* Y, int64_t sy, const void* D, int64_t sd, void* DG, int64_t sgt, int64_t sgk, int64_t Tn, int k, int N, int dtype,
                           hipStream_t st) {
  if (dtype == SMOE_BF16) return slots_gate_grad<bf16_t>(Y, sy, D, sd, DG, sgt, sgk, Tn, k, N, st);
  if (dtype == SMOE_F16) return slots_gate_grad<f16_t>(Y, sy, D, sd, DG, sgt, sgk, Tn, k, N, st);
  return slots_gate_grad<float>(Y, sy, D, sd, DG, sgt, sgk, Tn, k, N, st);
}

}  // namespace smoe
