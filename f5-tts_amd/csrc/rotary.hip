// rotary.hip — rotary positions of q and k in one launch (include/f5hip.h f5hip_rotary).
//
// (x, y) -> a (x cos - y sin, x sin + y cos) with the angle p f_i: three flops a value against 4 (16-bit types) to 8 (fp32) bytes moved, so
// the operator is a copy that computes on the way.  A thread owns one piece of a head's columns (16 bytes where sizes and alignment allow:
// VEC elements of both members of its pairs) at one token, and walks over the heads of q and then of k in steps of `hg`: its sines and cosines are
// computed once for all of them.  Consecutive threads take consecutive pieces, then consecutive heads, so a wave's access is one contiguous
// run wherever the heads are.  Heads per thread grow with the size of the call (launch_rotary): one at a time for single tokens, where only
// the number of threads hides latency, up to eight where the chip is full and the angle work is worth sharing.
//
// The angle: turns t = p f / 2 pi in 64 bits, reduced to t - rint(t) in [-1/2, 1/2] in 64 bits (at p = 2^31 the product is 2^-22 turns exact),
// then sin / cos of pi times twice that in fp32.  In fp32 from the start the product alone would be off by 2^-24 p f radians: 0.008 at
// position 131 072.
#include <algorithm>

#include "operators.h"

namespace {

struct RotaryArgs {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_stride[3], k_stride[3], q_out_stride[3], k_out_stride[3];  // batch, token, head
  const double* inv_freq;
  const int64_t* positions;
  int64_t position_stride, first;
  int batch, tokens, heads_q, heads, turned_q, turned_k;  // heads = heads_q + heads_k; turned: the first so many of each rotate
  int rot, nitem, npair, step, off_b;  // items of a head (the first npair rotate, the others copy); columns from item to item, to the partners
  int hg;                              // head step of a thread
  int keep_q, keep_k;                  // in place: what does not rotate stays untouched
  float amplitude, sign;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Piece {
  T v[N];
};

// TWO = false: an item is VEC / 2 interleaved pairs in one piece.  TWO = true: an item is VEC first members and, off_b columns on, their
// partners (the half layout; also, with VEC = 1, interleaved pairs that are not aligned to be read together).  U heads are loaded before
// the first of them is stored: an output may be its input, so the compiler does not move a load over a store by itself.
template <typename T, int VEC, bool TWO, int U>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  using P = Piece<T, VEC>;
  constexpr int NP = TWO ? VEC : VEC / 2;  // pairs of an item
  const uint32_t slots = (uint32_t)a.nitem * (uint32_t)a.hg;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x, token = id / slots;
  if (token >= (uint32_t)a.tokens) return;
  const uint32_t slot = id - token * slots;
  const int h0 = (int)(slot / (uint32_t)a.nitem), item = (int)(slot - (uint32_t)h0 * (uint32_t)a.nitem);
  const bool pair = item < a.npair;
  const int col = pair ? item * a.step : a.rot + (item - a.npair) * VEC;
  for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
    float c[NP], s[NP];
    if (pair) {
      const int64_t p = a.positions ? a.positions[(int64_t)b * a.position_stride + token] : a.first + (int64_t)token;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const double turns = (double)p * (a.inv_freq[item * NP + i] * 0.15915494309189533577);  // 1 / 2 pi
        const double r = turns - rint(turns);
#ifdef F5_HIPEMU
        c[i] = (float)cos(6.283185307179586477 * r);
        s[i] = (float)sin(6.283185307179586477 * r);
#else
        sincospif(2.0f * (float)r, &s[i], &c[i]);
#endif
        c[i] *= a.amplitude;
        s[i] *= a.amplitude * a.sign;
      }
    }
    for (int h = h0; h < a.heads; h += U * a.hg) {
      P x[U], y[U];
      T* out[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int hu = h + u * a.hg;
        out[u] = nullptr;
        if (hu >= a.heads) continue;
        const bool isq = hu < a.heads_q;
        const int hh = isq ? hu : hu - a.heads_q;
        const bool turn = pair && hh < (isq ? a.turned_q : a.turned_k);
        if (!turn && (isq ? a.keep_q : a.keep_k)) continue;
        const int64_t* si = isq ? a.q_stride : a.k_stride;
        const int64_t* so = isq ? a.q_out_stride : a.k_out_stride;
        const T* in = static_cast<const T*>(isq ? a.q : a.k) + b * si[0] + (int64_t)token * si[1] + hh * si[2] + col;
        out[u] = static_cast<T*>(isq ? a.q_out : a.k_out) + b * so[0] + (int64_t)token * so[1] + hh * so[2] + col;
        x[u] = *reinterpret_cast<const P*>(in);
        if (TWO && pair) y[u] = *reinterpret_cast<const P*>(in + a.off_b);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!out[u]) continue;
        const int hu = h + u * a.hg;
        const bool turn = pair && (hu < a.heads_q ? hu < a.turned_q : hu - a.heads_q < a.turned_k);
        if (turn) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            T& tx = x[u].v[TWO ? i : 2 * i];
            T& ty = TWO ? y[u].v[i] : x[u].v[TWO ? i : 2 * i + 1];
            const float fx = (float)tx, fy = (float)ty;
            tx = (T)(fx * c[i] - fy * s[i]);  // rounded once, to the nearest
            ty = (T)(fx * s[i] + fy * c[i]);
          }
        }
        *reinterpret_cast<P*>(out[u]) = x[u];
        if (TWO && pair) *reinterpret_cast<P*>(out[u] + a.off_b) = y[u];
      }
    }
  }
}

template <typename T, int VEC, bool TWO>
hipError_t launch(RotaryArgs& r, int head_dim, hipStream_t s) {
  r.npair = TWO ? r.rot / 2 / VEC : r.rot / VEC;
  r.nitem = r.npair + (head_dim - r.rot) / VEC;
  // Heads per thread: one until the call has more items than the chip keeps in flight (256 CUs x 2048 threads / 4), then up to eight.
  const int64_t items = (int64_t)r.batch * r.tokens * r.heads * r.nitem;
  const int per = (int)std::max<int64_t>(1, std::min<int64_t>(8, items / (256 * 512)));
  r.hg = (r.heads + per - 1) / per;
  const int64_t threads = (int64_t)r.tokens * r.nitem * r.hg;
  if (threads > 0x7fffff00) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((threads + 255) / 256), (unsigned)std::min(r.batch, 65535));
  if (per == 1) hipLaunchKernelGGL((rotary_kernel<T, VEC, TWO, 1>), grid, dim3(256), 0, s, r);
  else hipLaunchKernelGGL((rotary_kernel<T, VEC, TWO, 4>), grid, dim3(256), 0, s, r);
  return hipGetLastError();
}

template <typename T, int VEC>
hipError_t launch_layout(RotaryArgs& r, int head_dim, bool half, hipStream_t s) {
  if (half) {
    r.step = VEC;
    r.off_b = r.rot / 2;
    return launch<T, VEC, true>(r, head_dim, s);
  }
  if constexpr (VEC > 1) {
    r.step = VEC;
    r.off_b = 0;
    return launch<T, VEC, false>(r, head_dim, s);
  } else {
    r.step = 2;
    r.off_b = 1;
    return launch<T, 1, true>(r, head_dim, s);
  }
}

template <typename T>
hipError_t launch_type(RotaryArgs& r, int head_dim, bool half, int vec, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch_layout<T, 8>(r, head_dim, half, s);
  if (vec >= 4) return launch_layout<T, 4>(r, head_dim, half, s);
  if (vec >= 2) return launch_layout<T, 2>(r, head_dim, half, s);
  return launch_layout<T, 1>(r, head_dim, half, s);
}
}  // namespace

hipError_t launch_rotary(const f5hip_rotary_args& a, hipStream_t s) {
  RotaryArgs r{};
  r.q = a.q; r.k = a.k; r.q_out = a.q_out; r.k_out = a.k_out;
  for (int i = 0; i < 3; ++i) {
    r.q_stride[i] = a.q_stride[i]; r.q_out_stride[i] = a.q_out_stride[i];
    r.k_stride[i] = a.k_stride[i]; r.k_out_stride[i] = a.k_out_stride[i];
  }
  r.inv_freq = a.inv_freq; r.positions = a.positions; r.position_stride = a.position_stride; r.first = a.first;
  r.batch = a.batch; r.tokens = a.tokens; r.heads_q = a.heads_q; r.heads = a.heads_q + a.heads_k;
  r.turned_q = a.rot_heads < 0 ? a.heads_q : std::min(a.rot_heads, a.heads_q);
  r.turned_k = a.rot_heads < 0 ? a.heads_k : std::min(a.rot_heads, a.heads_k);
  r.rot = a.rot_dim;
  r.amplitude = a.amplitude;
  r.sign = a.inverse ? -1.0f : 1.0f;
  const auto same = [](const int64_t (&x)[3], const int64_t (&y)[3]) { return x[0] == y[0] && x[1] == y[1] && x[2] == y[2]; };
  r.keep_q = a.q == a.q_out && same(a.q_stride, a.q_out_stride);
  r.keep_k = a.k == a.k_out && same(a.k_stride, a.k_out_stride);
  // The widest piece (16 bytes at most) that divides the rotated columns (their half in the half layout), the columns behind them, every
  // stride and every pointer.
  const int eb = a.dtype == F5HIP_T_FP32 ? 4 : 2;
  const bool half = a.layout == F5HIP_ROTARY_HALF;
  int vec = 16 / eb;
  const auto fits = [&](int v) {
    if ((half ? a.rot_dim / 2 : a.rot_dim) % v || (a.head_dim - a.rot_dim) % v) return false;
    for (int i = 0; i < 3; ++i)
      if (a.q_stride[i] % v || a.q_out_stride[i] % v || (a.heads_k && (a.k_stride[i] % v || a.k_out_stride[i] % v))) return false;
    uintptr_t p = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out);
    if (a.heads_k) p |= reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out);
    return p % (uintptr_t)(v * eb) == 0;
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  if (a.dtype == F5HIP_T_FP16) return launch_type<f16>(r, a.head_dim, half, vec, s);
  if (a.dtype == F5HIP_T_BF16) return launch_type<bf16>(r, a.head_dim, half, vec, s);
  return launch_type<float>(r, a.head_dim, half, vec, s);
}
