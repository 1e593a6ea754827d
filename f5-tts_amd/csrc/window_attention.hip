// window_attention.hip — launch rules of the sliding-window attention (window_attention_kernel.h).
#include <algorithm>

#include "window_attention_kernel.h"

namespace {
// Few rows (window_few_kernel: waves along the keys) up to 32 rows of a key head, many (window_rows_kernel: waves along the rows) above.
// Many rows: 128 rows a workgroup, or, up to 64 columns and where that makes fewer than four workgroups a CU, 64 rows whose two waves share the keys
// (KG = 2).  Measured on an MI355X: 2 x 1406 frames, 16 heads of 64, 1026 keys seen (352 blocks of 128 rows) 23 us with 64 rows, 33 us with 128; 16 ragged
// utterances of 12 heads (1920 blocks) 56 and 50 us; 2 x 8192 frames (2048 blocks) 157 and 148 us; with 128 columns (6 chunks of 200 tokens, 32 heads on 8,
// 336 blocks) 81 and 75 us: there the tiles are twice as large, and loading them for 64 rows costs more than the better balance brings.
// Ranges of keys over workgroups, joined by window_join_kernel, where the blocks alone leave CUs without two workgroups: at least 256 keys each (few
// rows: 512, two tiles a wave).  More ranges balance better and lose it to the partial results' way out and back (the chunks in two ranges 75 us, three 81,
// four 89).
struct Plan {
  bool few;
  int ranges;  // many rows: key ranges of a workgroup (window_rows_kernel's KG)
  int nblk, nsplit;
};
Plan plan_of(const f5hip_window_attention_args& a) {
  const int group = a.heads / a.kv_heads;
  const int64_t rows = (int64_t)a.q_tokens * group, units = (int64_t)a.batch * a.kv_heads;
  Plan p{};
  p.few = rows <= 32;
  p.ranges = a.head_dim <= 64 && units * ((rows + 127) / 128) < 1024 ? 2 : 1;
  const int per = p.few ? 32 : 128 / p.ranges;
  p.nblk = (int)((rows + per - 1) / per);
  // the most keys that a block's queries can see
  int64_t keys = a.kv_tokens;
  if (a.window_left >= 0 && a.window_right >= 0)
    keys = std::min<int64_t>(keys, (int64_t)a.window_left + a.window_right + std::min<int64_t>(a.q_tokens, per / group + 2) + std::min(a.sinks, a.kv_tokens));
  const int64_t blocks = units * p.nblk, want = (512 + blocks - 1) / blocks, most = keys / (p.few ? 512 : 256);
  p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, most), 64));
  return p;
}
int64_t parts(const f5hip_window_attention_args& a, const Plan& p) { return (int64_t)a.batch * a.heads * a.q_tokens * p.nsplit; }

template <typename T>
hipError_t launch(const WindowArgs& w, const Plan& p, hipStream_t s) {
  const auto go = [&](auto DP) {
    constexpr int dp = decltype(DP)::value;
    if (p.few) hipLaunchKernelGGL((window_few_kernel<T, dp>), dim3((unsigned)w.nwg), dim3(64 * FEW_WAVES<T>), 0, s, w);
    else if (p.ranges == 1) hipLaunchKernelGGL((window_rows_kernel<T, dp, 1>), dim3((unsigned)w.nwg), dim3(256), 0, s, w);
    else if constexpr (dp == 64) hipLaunchKernelGGL((window_rows_kernel<T, dp, 2>), dim3((unsigned)w.nwg), dim3(256), 0, s, w);
  };
  if (w.dim <= 64) go(std::integral_constant<int, 64>{});
  else if (w.dim <= 96) go(std::integral_constant<int, 96>{});
  else go(std::integral_constant<int, 128>{});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || w.nsplit == 1) return e;
  const int64_t threads = (int64_t)w.batch * w.heads * w.tq * (w.dim / 4);
  hipLaunchKernelGGL((window_join_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, w);
  return hipGetLastError();
}
}  // namespace

int64_t window_attention_workspace(const f5hip_window_attention_args& a) {
  const Plan p = plan_of(a);
  return p.nsplit == 1 ? 0 : parts(a, p) * (a.head_dim + 2) * 4;
}

hipError_t launch_window_attention(const f5hip_window_attention_args& a, hipStream_t s) {
  const Plan p = plan_of(a);
  WindowArgs w{};
  w.q = a.q; w.k = a.k; w.v = a.v; w.out = a.out;
  for (int i = 0; i < 3; ++i) { w.q_stride[i] = a.q_stride[i]; w.k_stride[i] = a.k_stride[i]; w.v_stride[i] = a.v_stride[i]; w.out_stride[i] = a.out_stride[i]; }
  w.kv_len = a.kv_len; w.q_len = a.q_len;
  w.batch = a.batch; w.tq = a.q_tokens; w.tk = a.kv_tokens; w.heads = a.heads; w.kv_heads = a.kv_heads; w.group = a.heads / a.kv_heads; w.dim = a.head_dim;
  w.left = a.window_left; w.right = a.window_right; w.sinks = a.sinks; w.align_end = a.align_end;
  w.scale_log2 = std::max(std::fabs(a.scale) * 1.4426950408889634f, 1e-30f);  // (0 would turn a masked score into NaN)
  w.negate = a.scale < 0 ? (a.dtype == F5HIP_T_FP32 ? 0x80000000u : 0x80008000u) : 0u;
  w.nblk = p.nblk; w.nsplit = p.nsplit;
  w.nwg = (int)((int64_t)a.batch * a.kv_heads * p.nblk * p.nsplit);
  const int units = a.batch * a.kv_heads;
  w.xcd_units = units % 8 == 0 && units <= 64 ? units / 8 : 0;
  w.part_o = static_cast<float*>(a.workspace);
  w.part_ml = w.part_o ? w.part_o + parts(a, p) * a.head_dim : nullptr;
  if (a.dtype == F5HIP_T_FP16) return launch<f16>(w, p, s);
  if (a.dtype == F5HIP_T_BF16) return launch<bf16>(w, p, s);
  return launch<float>(w, p, s);
}
