// window_attention.hip — launch rules of the sliding-window attention (window_attention_kernel.h).
#include <algorithm>

#include "window_attention_kernel.h"

namespace {
WindowArgs args_of(const f5hip_window_attention_args& a) {
  WindowArgs w{};
  w.q = a.q; w.k = a.k; w.v = a.v; w.out = a.out;
  for (int i = 0; i < 3; ++i) { w.q_stride[i] = a.q_stride[i]; w.k_stride[i] = a.k_stride[i]; w.v_stride[i] = a.v_stride[i]; w.out_stride[i] = a.out_stride[i]; }
  w.kv_len = a.kv_len; w.q_len = a.q_len;
  w.batch = a.batch; w.tq = a.q_tokens; w.tk = a.kv_tokens; w.heads = a.heads; w.kv_heads = a.kv_heads; w.group = a.heads / a.kv_heads; w.dim = a.head_dim;
  w.left = a.window_left; w.right = a.window_right; w.sinks = a.sinks; w.align_end = a.align_end;
  w.scale_log2 = a.scale * 1.4426950408889634f;
  return w;
}
}  // namespace

int64_t window_attention_workspace(const f5hip_window_attention_args&) { return 0; }

hipError_t launch_window_attention(const f5hip_window_attention_args& a, hipStream_t s) {
  const WindowArgs w = args_of(a);
  const dim3 grid((unsigned)((int64_t)a.q_tokens * a.batch * a.heads));
  if (a.dtype == F5HIP_T_FP16) hipLaunchKernelGGL((window_attention_simple_kernel<f16>), grid, dim3(64), 0, s, w);
  else if (a.dtype == F5HIP_T_BF16) hipLaunchKernelGGL((window_attention_simple_kernel<bf16>), grid, dim3(64), 0, s, w);
  else hipLaunchKernelGGL((window_attention_simple_kernel<float>), grid, dim3(64), 0, s, w);
  return hipGetLastError();
}
