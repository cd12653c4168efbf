// Router front end: softmax over the expert logits of every token, top-k selection and optional renormalisation
// of the selected probabilities, in one pass over the (T, E) logits.
//
// Counterpart in the reference: the three torch calls of the Granite injection,
// scattermoe/utils/replace_moe.py:67-71 (softmax in float -> topk -> divide by the sum of the selected ones);
// every Hugging Face MoE block the reference patches computes its routing weights this way.
//
// One wave per token (select_experts in router_select.hpp).
#include "router_select.hpp"

namespace smoe {

template <typename T>
__global__ __launch_bounds__(256) void topk_softmax_kernel(const T* __restrict__ logits, int64_t slt, int64_t sle,
                                                          float* __restrict__ w_out, int64_t swt, int64_t swk,
                                                          int64_t* __restrict__ i_out, int64_t sit, int64_t sik,
                                                          int64_t Tn, int E, int k, int renorm) {
  const int lane = lane_id();
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= Tn) return;
  const float w = select_experts(
      E, k, renorm != 0, [&](int e) { return to_f32(logits[t * slt + e * sle]); }, [](float x) { return __expf(x); },
      [&](int j, int e) { i_out[t * sit + j * sik] = e; });
  if (lane < k) w_out[t * swt + lane * swk] = w;
}

int launch_topk_softmax(const void* logits, int64_t slt, int64_t sle, float* w, int64_t swt, int64_t swk,
                        int64_t* idx, int64_t sit, int64_t sik, int64_t Tn, int E, int k, int renorm, int dtype,
                        hipStream_t st) {
  const dim3 grid((unsigned)((Tn + 3) / 4)), block(256);
  switch (dtype) {
    case SMOE_F32:
      hipLaunchKernelGGL(topk_softmax_kernel<float>, grid, block, 0, st, (const float*)logits, slt, sle, w, swt, swk,
                         idx, sit, sik, Tn, E, k, renorm);
      break;
    case SMOE_BF16:
      hipLaunchKernelGGL(topk_softmax_kernel<bf16_t>, grid, block, 0, st, (const bf16_t*)logits, slt, sle, w, swt, swk,
                         idx, sit, sik, Tn, E, k, renorm);
      break;
    case SMOE_F16:
      hipLaunchKernelGGL(topk_softmax_kernel<f16_t>, grid, block, 0, st, (const f16_t*)logits, slt, sle, w, swt, swk,
                         idx, sit, sik, Tn, E, k, renorm);
      break;
    default:
      set_error("unknown dtype %d", dtype);
      return SMOE_ERR_DTYPE;
  }
  return launch_status("topk_softmax_kernel");
}

}  // namespace smoe
