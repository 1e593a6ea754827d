// rotary.hip — rotary positions of q and k in one launch (include/f5hip.h f5hip_rotary).
//
// (x, y) -> a (x cos - y sin, x sin + y cos) with the angle p f_i: three flops a value against 4 (16-bit types) to 8 (fp32) bytes moved, so
// the operator is a copy that computes on the way.  A thread owns one piece of a head's columns (16 bytes where sizes and alignment allow:
// VEC elements of both members of its pairs) at one token, in one or two of the heads of q and k, `hg` apart.  Consecutive threads take
// consecutive pieces, then consecutive heads, so a wave's access is one contiguous run wherever the heads are.  Heads per thread grow with the size of the call (launch_rotary): one at a time for single tokens, where only
// the number of threads hides latency, two where the chip is full.
// A workgroup's threads cover a few tokens; it works out each of their angles once, while its loads are under way, and hands the cosines and sines
// round through LDS (eight angles a thread by itself cost 2000 cycles and 100 registers: 4 x 8192 tokens of 40 heads of 128 took 176 us; now 134 us,
// 5.0 TB/s, which is what a large copy reaches on this card).
//
// The angle: p f turns by 1 / 2 pi, in units of a turn as p (w + e), w the 64-bit product f / 2 pi and e what its rounding and the constant's left behind.
// p w less the nearest whole number is one fused operation, so for |p| up to 2^53 the turn, in [-1/2, 1/2], is that of the exact product to 2^-53, whatever
// was reduced; then sin / cos of pi times twice that in fp32.  (In 64 bits without e it is off by 2^-22 turns at 2^31, in fp32 from the start by 2^-24 p f
// radians: 0.008 at position 131 072.)
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

// Stores past the cache: each XCD's L2 is written back at the kernel's end and whoever reads the output next sits on any XCD, so keeping it there buys
// nothing (4 x 8192 tokens of 40 heads of 128: 144 us with ordinary stores, 134 us with these).
template <typename P>
__device__ __forceinline__ void store_past_cache(P* p, const P& v) {
#ifdef F5_HIPEMU
  *p = v;
#else
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  using W = std::conditional_t<sizeof(P) == 16, u32x4, std::conditional_t<sizeof(P) == 8, u32x2, std::conditional_t<sizeof(P) == 4, unsigned, unsigned short>>>;
  static_assert(sizeof(W) == sizeof(P), "pieces of 2 to 16 bytes");
  __builtin_nontemporal_store(__builtin_bit_cast(W, v), reinterpret_cast<W*>(p));
#endif
}

// TWO = false: an item is VEC / 2 interleaved pairs in one piece.  TWO = true: an item is VEC first members and, off_b columns on, their
// partners (the half layout; also, with VEC = 1, interleaved pairs that are not aligned to be read together).  The thread's U heads, hg apart, are
// loaded before its angles are worked out and before the first is stored (an output may be its input, so the compiler moves no load over a store).
template <typename T, int VEC, bool TWO, int U>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  using P = Piece<T, VEC>;
  constexpr int NP = TWO ? VEC : VEC / 2;  // pairs of an item
  F5_DYN_LDS(float2, turns_lds);  // [tokens of the workgroup][rot / 2] (cos, sin)
  const uint32_t slots = (uint32_t)a.nitem * (uint32_t)a.hg;
  const uint32_t id = blockIdx.x * 256u + threadIdx.x, token = id / slots;
  const uint32_t token0 = blockIdx.x * 256u / slots, token1 = min((blockIdx.x * 256u + 255u) / slots, (uint32_t)a.tokens - 1u);
  const bool exists = token < (uint32_t)a.tokens;
  const int half_rot = a.rot / 2, nangle = (int)(token1 - token0 + 1u) * half_rot;
  const uint32_t slot = id - token * slots;
  const int h0 = (int)(slot / (uint32_t)a.nitem), item = (int)(slot - (uint32_t)h0 * (uint32_t)a.nitem);
  const bool pair = item < a.npair;
  const int col = pair ? item * a.step : a.rot + (item - a.npair) * VEC;
  for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
    P x[U], y[U];
    bool turn[U], live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * a.hg;
      const bool isq = h < a.heads_q;
      const int hh = isq ? h : h - a.heads_q;
      turn[u] = pair && hh < (isq ? a.turned_q : a.turned_k);
      live[u] = exists && h < a.heads && (turn[u] || !(isq ? a.keep_q : a.keep_k));
      if (!live[u]) continue;
      const int64_t* st = isq ? a.q_stride : a.k_stride;
      const T* in = static_cast<const T*>(isq ? a.q : a.k) + b * st[0] + (int64_t)token * st[1] + hh * st[2] + col;
      x[u] = *reinterpret_cast<const P*>(in);
      if (TWO && pair) y[u] = *reinterpret_cast<const P*>(in + a.off_b);
    }
    for (int i = threadIdx.x; i < nangle; i += 256) {
      const int t = i / half_rot, f = i - t * half_rot;
      const int64_t tok = (int64_t)token0 + t, p = a.positions ? a.positions[(int64_t)b * a.position_stride + tok] : a.first + tok;
      constexpr double hi = 0x1.45f306dc9c883p-3, lo = -0x1.6b01ec5417056p-57;  // 1 / 2 pi
      const double freq = a.inv_freq[f], w = freq * hi, e = fma(freq, lo, fma(freq, hi, -w)), at = (double)p;
      const double r = fma(at, w, -rint(at * w)) + at * e;
      float2 cs;
#ifdef F5_HIPEMU
      cs.x = (float)cos(6.283185307179586477 * r);
      cs.y = (float)sin(6.283185307179586477 * r);
#else
      sincospif(2.0f * (float)r, &cs.y, &cs.x);
#endif
      cs.x *= a.amplitude;
      cs.y *= a.amplitude * a.sign;
      turns_lds[i] = cs;
    }
    __syncthreads();
    float c[NP], s[NP];
    if (pair && exists) {
      const float2* at = turns_lds + (token - token0) * (uint32_t)half_rot + item * NP;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        c[i] = at[i].x;
        s[i] = at[i].y;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!live[u]) continue;
      const int h = h0 + u * a.hg;
      const bool isq = h < a.heads_q;
      if (turn[u]) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          T& tx = x[u].v[TWO ? i : 2 * i];
          T& ty = TWO ? y[u].v[i] : x[u].v[TWO ? i : 2 * i + 1];
          const float fx = (float)tx, fy = (float)ty;
          tx = (T)(fx * c[i] - fy * s[i]);  // rounded once, to the nearest
          ty = (T)(fx * s[i] + fy * c[i]);
        }
      }
      const int64_t* st = isq ? a.q_out_stride : a.k_out_stride;
      T* out = static_cast<T*>(isq ? a.q_out : a.k_out) + b * st[0] + (int64_t)token * st[1] + (isq ? h : h - a.heads_q) * st[2] + col;
      store_past_cache(reinterpret_cast<P*>(out), x[u]);
      if (TWO && pair) store_past_cache(reinterpret_cast<P*>(out + a.off_b), y[u]);
    }
    __syncthreads();  // the next sequence's angles take the place of these
  }
}

// the pieces of a call and their threads
struct Plan {
  int vec, npair, nitem, hg;  // elements of a piece; pieces of a head that rotate, all of them; heads of a thread stand hg apart
  bool two;                   // a thread's pairs are in two pieces
  int per;                    // heads of a thread
  int64_t threads;            // of a sequence
};
Plan plan_of(const f5hip_rotary_args& a) {
  Plan p{};
  // The widest piece (16 bytes at most) that divides the rotated columns (their half in the half layout), the columns behind them, every
  // stride and every pointer.
  const int eb = a.dtype == F5HIP_T_FP32 ? 4 : 2;
  const bool half = a.layout == F5HIP_ROTARY_HALF;
  const auto fits = [&](int v) {
    if ((half ? a.rot_dim / 2 : a.rot_dim) % v || (a.head_dim - a.rot_dim) % v) return false;
    for (int i = 0; i < 3; ++i)
      if (a.q_stride[i] % v || a.q_out_stride[i] % v || (a.heads_k && (a.k_stride[i] % v || a.k_out_stride[i] % v))) return false;
    uintptr_t p = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out);
    if (a.heads_k) p |= reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out);
    return p % (uintptr_t)(v * eb) == 0;
  };
  p.vec = 16 / eb;
  while (p.vec > 1 && !fits(p.vec)) p.vec /= 2;
  p.two = half || p.vec == 1;
  p.npair = p.two ? a.rot_dim / 2 / p.vec : a.rot_dim / p.vec;
  p.nitem = p.npair + (a.head_dim - a.rot_dim) / p.vec;
  // Heads per thread: one until the call has half as many items as the chip holds threads (256 CUs x 2048), two above (4 x 8192 tokens of 40 heads of
  // 128: 134 us, with four heads and their registers 139 us, with one 135 us; 2 x 1406 tokens of 32 heads of 64: 6.6, 7.8, 7.6 us).
  const int heads = a.heads_q + a.heads_k;
  const int64_t items = (int64_t)a.batch * a.tokens * heads * p.nitem;
  p.per = items < 256 * 1024 ? 1 : 2;
  p.hg = (heads + p.per - 1) / p.per;
  p.threads = (int64_t)a.tokens * p.nitem * p.hg;
  return p;
}

template <typename T, int VEC, bool TWO>
hipError_t launch(const RotaryArgs& r, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.threads + 255) / 256), (unsigned)std::min(r.batch, 65535));
  // 256 threads touch at most 256 / slots + 2 tokens: 48 KiB for the largest head, under 17 KiB for the smallest
  const int64_t slots = (int64_t)p.nitem * p.hg;
  const size_t lds = (size_t)(256 / slots + 2) * (r.rot / 2) * sizeof(float2);
  if (p.per == 1) hipLaunchKernelGGL((rotary_kernel<T, VEC, TWO, 1>), grid, dim3(256), lds, s, r);
  else hipLaunchKernelGGL((rotary_kernel<T, VEC, TWO, 2>), grid, dim3(256), lds, s, r);
  return hipGetLastError();
}

template <typename T, int VEC>
hipError_t launch_layout(RotaryArgs& r, const Plan& p, bool half, hipStream_t s) {
  if (half) {
    r.step = VEC;
    r.off_b = r.rot / 2;
    return launch<T, VEC, true>(r, p, s);
  }
  if constexpr (VEC > 1) {
    r.step = VEC;
    r.off_b = 0;
    return launch<T, VEC, false>(r, p, s);
  } else {
    r.step = 2;
    r.off_b = 1;
    return launch<T, 1, true>(r, p, s);
  }
}

template <typename T>
hipError_t launch_type(RotaryArgs& r, const Plan& p, bool half, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (p.vec == 8) return launch_layout<T, 8>(r, p, half, s);
  if (p.vec >= 4) return launch_layout<T, 4>(r, p, half, s);
  if (p.vec >= 2) return launch_layout<T, 2>(r, p, half, s);
  return launch_layout<T, 1>(r, p, half, s);
}
}  // namespace

int64_t rotary_threads(const f5hip_rotary_args& a) { return plan_of(a).threads; }

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
  const Plan p = plan_of(a);
  if (p.threads > ROTARY_THREADS) return hipErrorInvalidValue;  // (the entry point says why)
  r.npair = p.npair; r.nitem = p.nitem; r.hg = p.hg;
  const bool half = a.layout == F5HIP_ROTARY_HALF;
  if (a.dtype == F5HIP_T_FP16) return launch_type<f16>(r, p, half, s);
  if (a.dtype == F5HIP_T_BF16) return launch_type<bf16>(r, p, half, s);
  return launch_type<float>(r, p, half, s);
}
