// window_attention_kernel.h — sliding-window attention with sinks (include/f5hip.h f5hip_window_attention); the launch rules are in
// window_attention.hip.
#pragma once
#include <math.h>

#include "operators.h"

namespace {

struct WindowArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];  // batch, token, head
  const int32_t *kv_len, *q_len;
  int batch, tq, tk, heads, kv_heads, group, dim;
  int left, right, sinks, align_end;
  float scale_log2;  // scale * log2(e)
};

// One wave per query row: 64 keys at a time, a lane per key for the scores, a lane per column for the product with v.
template <typename T>
__global__ __launch_bounds__(64) void window_attention_simple_kernel(WindowArgs a) {
  const int lane = threadIdx.x, bh = blockIdx.x / a.tq, i = blockIdx.x - bh * a.tq, b = bh / a.heads, head = bh - b * a.heads;
  const int n = a.kv_len ? min(max(a.kv_len[b], 0), a.tk) : a.tk, nq = a.q_len ? min(max(a.q_len[b], 0), a.tq) : a.tq;
  if (i >= nq) return;
  const int p = a.align_end ? n - nq + i : i;
  const int end = a.right < 0 ? n : max(0, min(n, p + a.right + 1)), begin = a.left < 0 ? 0 : min(max(0, p - a.left), end);
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + head * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + (head / a.group) * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + (head / a.group) * a.v_stride[2];
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  const auto keys = [&](int from, int to) {
    for (int j0 = from; j0 < to; j0 += 64) {
      float s = -INFINITY;
      if (j0 + lane < to) {
        s = 0.f;
        for (int d = 0; d < a.dim; ++d) s = fmaf((float)q[d], (float)k[(int64_t)(j0 + lane) * a.k_stride[1] + d], s);
        s *= a.scale_log2;
      }
      const float mn = fmaxf(m, wave_max(s)), al = exp2f(m - mn), w = exp2f(s - mn);
      m = mn;
      l = l * al + wave_sum(w);
      o0 *= al;
      o1 *= al;
      for (int t = 0; t < min(64, to - j0); ++t) {
        const float wt = __shfl(w, t, 64);
        const T* r = v + (int64_t)(j0 + t) * a.v_stride[1];
        if (lane < a.dim) o0 = fmaf(wt, (float)r[lane], o0);
        if (lane + 64 < a.dim) o1 = fmaf(wt, (float)r[lane + 64], o1);
      }
    }
  };
  keys(0, min(a.sinks, begin));
  keys(begin, end);
  T* o = static_cast<T*>(a.out) + b * a.out_stride[0] + i * a.out_stride[1] + head * a.out_stride[2];
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  if (lane < a.dim) o[lane] = (T)(o0 * inv);
  if (lane + 64 < a.dim) o[lane + 64] = (T)(o1 * inv);
}
}  // namespace
