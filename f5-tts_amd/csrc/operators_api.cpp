// operators_api.cpp — entry points of the operators (include/f5hip.h, "operators"): argument checks, device guard, per-thread error text.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "operators.h"
#ifndef F5_HIPEMU
#include <hip/hip_runtime.h>
#endif

int f5hip_set_thread_error(int code, const char* text);  // api.cpp: the text f5hip_last_error(NULL) returns

namespace {
int elt_bytes(int dtype) { return dtype == F5HIP_T_FP32 ? 4 : 2; }

// every element's offset in bytes stays far below 2^63, so 64-bit offsets cannot wrap (no address space has more than 2^57)
bool strides_ok(const int64_t (&st)[3], const int64_t (&ext)[3], bool output) {
  __int128 span = 0;
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0 || st[i] > (int64_t(1) << 40)) return false;
    if (output && st[i] == 0 && ext[i] > 1) return false;
    if (ext[i] > 1) span += (__int128)(ext[i] - 1) * st[i];
  }
  return span < (int64_t(1) << 55);
}
// an axis of at most one element may carry any stride: none
void drop_idle_strides(int64_t (&st)[3], int64_t batch, int64_t tokens, int64_t heads) {
  if (batch <= 1) st[0] = 0;
  if (tokens <= 1) st[1] = 0;
  if (heads <= 1) st[2] = 0;
}
f5hip_rotary_args plain(const f5hip_rotary_args& args) {
  f5hip_rotary_args a = args;
  drop_idle_strides(a.q_stride, a.batch, a.tokens, a.heads_q);
  drop_idle_strides(a.q_out_stride, a.batch, a.tokens, a.heads_q);
  drop_idle_strides(a.k_stride, a.batch, a.tokens, a.heads_k);
  drop_idle_strides(a.k_out_stride, a.batch, a.tokens, a.heads_k);
  return a;
}
f5hip_window_attention_args plain(const f5hip_window_attention_args& args) {
  f5hip_window_attention_args a = args;
  drop_idle_strides(a.q_stride, a.batch, a.q_tokens, a.heads);
  drop_idle_strides(a.out_stride, a.batch, a.q_tokens, a.heads);
  drop_idle_strides(a.k_stride, a.batch, a.kv_tokens, a.kv_heads);
  drop_idle_strides(a.v_stride, a.batch, a.kv_tokens, a.kv_heads);
  return a;
}
// a buffer as runs of `run` bytes: at `base` plus any multiples x_i < n_i of the strides, in bytes
struct Runs {
  const void* base;
  int64_t run, n[3], stride[3];
  Runs(const void* p, int64_t bytes) : base(p), run(p ? bytes : 0), n{1, 1, 1}, stride{0, 0, 0} {}
  Runs(const void* p, int dim, int eb, const int64_t (&st)[3], const int64_t (&ext)[3]) : Runs(p, (int64_t)dim * eb) {
    for (int i = 0; i < 3; ++i) {
      if (ext[i] < 1) run = 0;  // no element
      if (ext[i] > 1 && st[i] > 0) { n[i] = ext[i]; stride[i] = st[i] * eb; }
    }
  }
  uintptr_t begin() const { return reinterpret_cast<uintptr_t>(base); }
  uintptr_t end() const { return begin() + (uintptr_t)(run + (n[0] - 1) * stride[0] + (n[1] - 1) * stride[1] + (n[2] - 1) * stride[2]); }
};
// Is there a sum of c_i s_i, low_i <= c_i <= high_i, between `above` and `below` — with `moved`, one whose c_i are not all 0?  Strides in falling order,
// so what the smaller ones reach leaves few c_i to try: for views of one buffer a handful.  Strides that leave more than 2^16 are taken for a yes.
struct Reach {
  int dims = 0, left = 1 << 16;
  int64_t s[6], low[6], high[6];
  void add(int64_t stride, int64_t from, int64_t to) {
    if (!stride) return;
    int i = 0;
    while (i < dims && s[i] > stride) ++i;
    if (i == dims || s[i] != stride) {
      for (int j = dims++; j > i; --j) { s[j] = s[j - 1]; low[j] = low[j - 1]; high[j] = high[j - 1]; }
      s[i] = stride;
      low[i] = high[i] = 0;
    }
    low[i] += from;
    high[i] += to;
  }
  bool between(int64_t above, int64_t below, bool moved, int i = 0) {
    if (i == dims) return above < 0 && 0 < below && moved;
    int64_t least = 0, most = 0;
    for (int j = i + 1; j < dims; ++j) { least += low[j] * s[j]; most += high[j] * s[j]; }
    // the c with above < c s + (something in [least, most]) < below
    const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    const int64_t from = std::max(low[i], floor_div(above - most, s[i]) + 1), to = std::min(high[i], -floor_div(least - below, s[i]) - 1);
    for (int64_t c = from; c <= to; ++c)
      if (--left < 0 || between(above - c * s[i], below - c * s[i], moved || c != 0, i + 1)) return true;
    return false;
  }
};
bool share_memory(const Runs& a, const Runs& b) {
  if (!a.run || !b.run || a.end() <= b.begin() || b.end() <= a.begin()) return false;
  Reach r;
  for (int i = 0; i < 3; ++i) {
    r.add(a.stride[i], 0, a.n[i] - 1);
    r.add(b.stride[i], 1 - b.n[i], 0);
  }
  const int64_t apart = (int64_t)(b.begin() - a.begin());
  return r.between(apart - a.run, apart + b.run, true);
}
bool elements_overlap(const Runs& a) {
  Reach r;
  for (int i = 0; i < 3; ++i) r.add(a.stride[i], 1 - a.n[i], a.n[i] - 1);
  int64_t inner = a.run;  // each stride past what the smaller ones reach (two equal ones overlap): the ordinary tensor
  bool nested = a.run > 0;
  for (int i = r.dims - 1; i >= 0; --i) {
    nested = nested && r.s[i] >= inner;
    inner += r.high[i] * r.s[i];
  }
  int axes = 0;
  for (int64_t st : a.stride) axes += st > 0;
  return a.run > 0 && (axes != r.dims || (!nested && r.between(-a.run, a.run, false)));
}
bool same_strides(const int64_t (&x)[3], const int64_t (&y)[3]) { return x[0] == y[0] && x[1] == y[1] && x[2] == y[2]; }
bool aligned(const void* p, int a) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(a - 1)) == 0; }

// the calling thread's device while an operator launches, restored on every path
struct DeviceGuard {
  int before = -1;
  bool changed = false;
  hipError_t enter(int device) {
    hipError_t e = hipGetDevice(&before);
    if (e != hipSuccess || before == device) return e;
    e = hipSetDevice(device);
    changed = e == hipSuccess;
    return e;
  }
  ~DeviceGuard() {
    if (changed) (void)hipSetDevice(before);
  }
};

template <typename F>
int on_device(int device, F&& launch) {
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || n == 0) return f5hip_set_thread_error(F5HIP_ERR_HIP, "no HIP device: there is no CPU fallback");
  if (device < 0 || device >= n) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "device ordinal out of range");
  DeviceGuard guard;
  hipError_t e = guard.enter(device);
  if (e == hipSuccess) e = launch();
  if (e == hipSuccess) return F5HIP_OK;
  char b[128];
  snprintf(b, sizeof(b), "operator launch failed: %s", hipGetErrorString(e));
  return f5hip_set_thread_error(F5HIP_ERR_HIP, b);
}
}  // namespace

const char* check_rotary(const f5hip_rotary_args& a) {
  if (a.dtype < F5HIP_T_FP32 || a.dtype > F5HIP_T_BF16) return "rotary: dtype must be fp32, fp16 or bf16";
  if (a.layout != F5HIP_ROTARY_INTERLEAVED && a.layout != F5HIP_ROTARY_HALF) return "rotary: unknown layout";
  if (a.batch < 0 || a.tokens < 0 || a.heads_q < 1 || a.heads_k < 0 || a.head_dim < 2) return "rotary: batch, tokens >= 0, heads_q >= 1, heads_k >= 0, head_dim >= 2";
  if (a.rot_dim < 2 || (a.rot_dim & 1) || a.rot_dim > a.head_dim) return "rotary: rot_dim must be even and in [2, head_dim]";
  if (a.rot_heads < -1) return "rotary: rot_heads must be -1 (all) or a number of heads";
  if (a.head_dim > 4096 || a.heads_q > 65536 || a.heads_k > 65536) return "rotary: head_dim <= 4096, heads <= 65536";
  if ((int64_t)a.tokens * a.head_dim * ((int64_t)a.heads_q + a.heads_k) >= (int64_t(1) << 38)) return "rotary: more than 2^38 elements in a sequence";
  if (!std::isfinite(a.amplitude)) return "rotary: amplitude must be finite";
  if (a.batch == 0 || a.tokens == 0) return nullptr;  // nothing to do: empty tensors have no pointers
  if (!a.q || !a.q_out || !a.inv_freq || (a.heads_k && (!a.k || !a.k_out))) return "rotary: null pointer";
  const int eb = elt_bytes(a.dtype);
  if (!aligned(a.q, eb) || !aligned(a.q_out, eb) || (a.heads_k && (!aligned(a.k, eb) || !aligned(a.k_out, eb)))) return "rotary: pointer not aligned to its elements";
  if (!aligned(a.inv_freq, 8) || (a.positions && !aligned(a.positions, 8))) return "rotary: inv_freq / positions not aligned to 8 bytes";
  const int64_t eq[3] = {a.batch, a.tokens, a.heads_q}, ek[3] = {a.batch, a.tokens, a.heads_k};
  if (!strides_ok(a.q_stride, eq, false) || !strides_ok(a.q_out_stride, eq, true) ||
      (a.heads_k && (!strides_ok(a.k_stride, ek, false) || !strides_ok(a.k_out_stride, ek, true))))
    return "rotary: strides must lie in [0, 2^40] and a tensor must span less than 2^55 elements, an output's strides must not be 0";
  if (a.position_stride < 0 || a.position_stride > (int64_t(1) << 40) || (a.positions && (__int128)a.position_stride * a.batch >= int64_t(1) << 55))
    return "rotary: position_stride must lie in [0, 2^40] and the positions must span less than 2^55 elements";
  // (the last token's position is worked out in 64 bits)
  if (!a.positions && a.first > INT64_MAX - a.tokens) return "rotary: first + tokens must stay below 2^63";
  const Runs q(a.q, a.head_dim, eb, a.q_stride, eq), qo(a.q_out, a.head_dim, eb, a.q_out_stride, eq);
  const Runs k(a.heads_k ? a.k : nullptr, a.head_dim, eb, a.k_stride, ek), ko(a.heads_k ? a.k_out : nullptr, a.head_dim, eb, a.k_out_stride, ek);
  if (elements_overlap(qo) || elements_overlap(ko)) return "rotary: an output's elements must not overlap";
  // (strides of idle axes have been dropped: equal ones are the same view)
  const bool q_in_place = a.q == a.q_out && same_strides(a.q_stride, a.q_out_stride), k_in_place = a.k == a.k_out && same_strides(a.k_stride, a.k_out_stride);
  if ((!q_in_place && share_memory(qo, q)) || (!k_in_place && share_memory(ko, k)) || share_memory(qo, k) || share_memory(ko, q) || share_memory(qo, ko))
    return "rotary: an output may be its own input with the same strides, or memory of its own";
  const Runs freq(a.inv_freq, a.rot_dim / 2 * 8);
  Runs at(a.positions, (int64_t)a.tokens * 8);
  if (a.position_stride > 0) { at.n[0] = a.batch; at.stride[0] = a.position_stride * 8; }
  for (const Runs& in : {freq, at})
    if (share_memory(qo, in) || share_memory(ko, in)) return "rotary: an output must share no memory with inv_freq and positions";
  if (rotary_threads(a) > ROTARY_THREADS) return "rotary: a sequence of more than 2^31 pieces (of up to 16 bytes, as alignment allows)";
  return nullptr;
}

const char* check_window_attention(const f5hip_window_attention_args& a) {
  if (a.dtype < F5HIP_T_FP32 || a.dtype > F5HIP_T_BF16) return "window attention: dtype must be fp32, fp16 or bf16";
  if (a.batch < 0 || a.q_tokens < 0 || a.kv_tokens < 0 || a.heads < 1 || a.kv_heads < 1) return "window attention: batch, tokens >= 0, heads >= 1";
  if (a.heads % a.kv_heads) return "window attention: kv_heads must divide heads";
  const int eb = elt_bytes(a.dtype);
  if (a.head_dim < 1 || a.head_dim > 128 || (a.head_dim * eb) % 16) return "window attention: head_dim must be at most 128 and a whole multiple of 16 bytes";
  if (a.sinks < 0) return "window attention: sinks must be >= 0";
  if (a.align_end != 0 && a.align_end != 1) return "window attention: align_end must be 0 or 1";
  if (!std::isfinite(a.scale * 1.4426950408889634f)) return "window attention: scale times log2(e) must be finite";  // (what the kernels multiply by)
  constexpr int lim = 1 << 30;  // sums of two of them stay in 32 bits
  if (a.q_tokens >= lim || a.kv_tokens >= lim || a.window_left >= lim || a.window_right >= lim || a.sinks >= lim)
    return "window attention: tokens, window and sinks must be below 2^30";
  // the grid's threads stay below 2^32
  if ((int64_t)a.batch * a.heads >= (1 << 22)) return "window attention: batch * heads must be below 2^22";
  if ((int64_t)a.batch * a.heads * a.q_tokens >= lim) return "window attention: batch * heads * q_tokens must be below 2^30";
  if (a.batch == 0 || a.q_tokens == 0) return nullptr;
  if (!a.q || !a.out || (a.kv_tokens && (!a.k || !a.v))) return "window attention: null pointer";
  if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16)) return "window attention: pointers must be aligned to 16 bytes";
  if (!aligned(a.kv_len, 4) || !aligned(a.q_len, 4)) return "window attention: lengths must be aligned to 4 bytes";
  const int64_t eq[3] = {a.batch, a.q_tokens, a.heads}, ek[3] = {a.batch, a.kv_tokens, a.kv_heads};
  if (!strides_ok(a.q_stride, eq, false) || !strides_ok(a.out_stride, eq, true) || !strides_ok(a.k_stride, ek, false) || !strides_ok(a.v_stride, ek, false))
    return "window attention: strides must lie in [0, 2^40] and a tensor must span less than 2^55 elements, the output's strides must not be 0";
  const int64_t (*all[4])[3] = {&a.q_stride, &a.k_stride, &a.v_stride, &a.out_stride};
  for (auto* st : all)
    for (int i = 0; i < 3; ++i)
      if (((*st)[i] * eb) % 16) return "window attention: strides must be whole multiples of 16 bytes";
  // a 64-key tile is addressed with 31-bit byte offsets from its first key
  if (a.k_stride[1] * eb * 64 >= (int64_t(1) << 31) || a.v_stride[1] * eb * 64 >= (int64_t(1) << 31)) return "window attention: 64 key rows must span less than 2 GiB";
  const Runs out(a.out, a.head_dim, eb, a.out_stride, eq);
  if (elements_overlap(out)) return "window attention: out's elements must not overlap";
  const Runs q(a.q, a.head_dim, eb, a.q_stride, eq), k(a.k, a.head_dim, eb, a.k_stride, ek), v(a.v, a.head_dim, eb, a.v_stride, ek);
  const Runs kv_len(a.kv_len, (int64_t)a.batch * 4), q_len(a.q_len, (int64_t)a.batch * 4);
  for (const Runs* in : {&q, &k, &v, &kv_len, &q_len})
    if (share_memory(out, *in)) return "window attention: out must share no memory with q, k and v, nor with the lengths";
  return nullptr;
}

const char* scale_rotary_frequencies(double* f, int rot_dim, int scaling, double factor, int64_t original_length, double low, double high, double* amplitude) {
  if (scaling < F5HIP_ROPE_NONE || scaling > F5HIP_ROPE_YARN) return "rotary frequencies: unknown scaling";
  if (scaling != F5HIP_ROPE_NONE && (!(factor > 0) || !std::isfinite(factor))) return "rotary frequencies: factor must be positive";
  if (scaling == F5HIP_ROPE_NTK && rot_dim < 4) return "rotary frequencies: the base change needs rot_dim >= 4";
  if (scaling == F5HIP_ROPE_YARN) {
    if (low == 0 && high == 0) { low = 1; high = 32; }
    if (original_length <= 0 || !(low >= 0) || !(high > low) || !std::isfinite(high) || !(factor >= 1))
      return "rotary frequencies: by parts needs original_length > 0, 0 <= low < high, factor >= 1";
  }
  for (int i = 0; i < rot_dim / 2; ++i) {
    if (scaling == F5HIP_ROPE_LINEAR) f[i] /= factor;
    if (scaling == F5HIP_ROPE_NTK) f[i] *= std::pow(factor, -2.0 * i / (rot_dim - 2));  // (base factor^(R / (R - 2)))^(-2i / R)
    if (scaling == F5HIP_ROPE_YARN) {
      const double r = (double)original_length * f[i] / 6.283185307179586476925;
      const double g = std::fmin(1.0, std::fmax(0.0, (r - low) / (high - low)));
      f[i] *= g + (1.0 - g) / factor;
    }
    if (!std::isfinite(f[i])) return "rotary frequencies: the base and the factor give an infinite frequency";
  }
  *amplitude = scaling == F5HIP_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
  return nullptr;
}

extern "C" {
int f5hip_rotary_frequencies(int rot_dim, double base, int scaling, double factor, int64_t original_length, double low, double high, double* inv_freq,
                             double* amplitude) {
  if (!inv_freq || !amplitude) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "rotary frequencies: null pointer");
  if (rot_dim < 2 || (rot_dim & 1)) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "rotary frequencies: rot_dim must be even and >= 2");
  if (!(base > 0) || !std::isfinite(base)) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "rotary frequencies: base must be positive");
  for (int i = 0; i < rot_dim / 2; ++i) inv_freq[i] = std::pow(base, -2.0 * i / rot_dim);
  if (const char* why = scale_rotary_frequencies(inv_freq, rot_dim, scaling, factor, original_length, low, high, amplitude))
    return f5hip_set_thread_error(F5HIP_ERR_INVALID, why);
  return F5HIP_OK;
}

int f5hip_rotary(const f5hip_rotary_args* args, int device, void* stream) {
  if (!args) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "rotary: null argument");
  const f5hip_rotary_args a = plain(*args);
  if (const char* why = check_rotary(a)) return f5hip_set_thread_error(F5HIP_ERR_INVALID, why);
  if (a.batch == 0 || a.tokens == 0) return F5HIP_OK;
  return on_device(device, [&] { return launch_rotary(a, (hipStream_t)stream); });
}

int64_t f5hip_window_attention_workspace(const f5hip_window_attention_args* args) {
  const char* why = args ? check_window_attention(plain(*args)) : "window attention: null argument";
  if (why) { f5hip_set_thread_error(F5HIP_ERR_INVALID, why); return -1; }
  return args->batch == 0 || args->q_tokens == 0 ? 0 : window_attention_workspace(*args);
}

int f5hip_window_attention(const f5hip_window_attention_args* args, int device, void* stream) {
  if (!args) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "window attention: null argument");
  const f5hip_window_attention_args a = plain(*args);
  if (const char* why = check_window_attention(a)) return f5hip_set_thread_error(F5HIP_ERR_INVALID, why);
  if (a.batch == 0 || a.q_tokens == 0) return F5HIP_OK;
  const int64_t need = window_attention_workspace(a);
  if (a.workspace_bytes < need || (need && (!a.workspace || !aligned(a.workspace, 16))))
    return f5hip_set_thread_error(F5HIP_ERR_INVALID, "window attention: workspace missing, too small or not aligned to 16 bytes");
  const int64_t eq[3] = {a.batch, a.q_tokens, a.heads}, ek[3] = {a.batch, a.kv_tokens, a.kv_heads};
  const int eb = elt_bytes(a.dtype);
  for (const Runs& other : {Runs(a.out, a.head_dim, eb, a.out_stride, eq), Runs(a.q, a.head_dim, eb, a.q_stride, eq), Runs(a.k, a.head_dim, eb, a.k_stride, ek),
                            Runs(a.v, a.head_dim, eb, a.v_stride, ek), Runs(a.kv_len, (int64_t)a.batch * 4), Runs(a.q_len, (int64_t)a.batch * 4)})
    if (share_memory(Runs(a.workspace, need), other)) return f5hip_set_thread_error(F5HIP_ERR_INVALID, "window attention: the workspace must share no memory with the tensors");
  return on_device(device, [&] { return launch_window_attention(a, (hipStream_t)stream); });
}
}  // extern "C"
