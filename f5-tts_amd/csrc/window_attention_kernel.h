// window_attention_kernel.h — sliding-window attention with sinks (include/f5hip.h f5hip_window_attention).  A header so that tests/hipemu can
// compile the same source for the host; the launch rules are in window_attention.hip.
//
// Rows.  The query heads that share a key head are rows of one matrix: row R of (sequence, key head) is token R / group, head R % group, so
// a key tile is read once for all of them, and one new token of a model with grouped heads already fills part of a 32-row tile.
// Keys.  A block of rows visits [0, sinks) and the union of its rows' windows, [low, high) — or [0, high) where the two meet — in tiles that
// start at 0 and at `low`: whatever lies between, or past the last key, is not read (rows behind a tile's last key come from the buffer
// descriptor's bounds check as zeros).  Only tiles on a border of some row's window take the mask.
// Product.  S^T = K Q^T on 32x32 matrix instructions leaves a lane 16 keys of ONE query row, so maxima and sums are register work and one
// half-wave exchange; those registers are, as they stand, the other operand of O^T += V^T P^T (the contraction runs over keys in the
// accumulator's own order), so P never moves.  V^T fragments come from row-major V tiles by the transposing LDS read.
// fp32.  A number is the exact sum of three bf16 pieces of 8 bits each, high | middle | low; a product takes six of the nine piece products (the other
// three are below 2^-21 of it, below 2^-23 in the mean) on the bf16 matrix instructions, at 6 / 16 of the cost of the fp32 ones.  q is split once, K and V as
// they are staged, P in registers.
// Softmax.  exp2(c s - c m) with c = scale log2 e > 0 (a negative scale's sign is folded into q).  m is a reference, not the running maximum, and no
// maximum is taken on the common path: the weights of a tile are summed anyway, and only where a lane's sum passes LIMIT = 2^(BIAS + 8) — the reference is
// 2^3 to 2^8 too low, or none has been set — is the tile's maximum taken, O and l rescaled, and the tile's weights computed again.  The reference is set so
// that the row's largest weight is 2^BIAS: in fp16 2^7, so that weights up to 2^15 are finite and those as small as 2^-21 of the largest are normal numbers,
// rounded relative to themselves; in bf16 and fp32 1, and O, at most 2^8 |v| for every 16 keys, is finite where 16 |v| keys < 2^128.
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
  float scale_log2;       // |scale| log2(e), > 0
  uint32_t negate;        // sign bits to flip in q (a negative scale)
  int nblk, nsplit, nwg;  // row blocks of a (sequence, key head), key ranges of a row block, workgroups
  int xcd_units;          // (sequence, key head) units of each XCD whose blocks take turns; 0: one unit after the other
  float *part_o, *part_ml;  // nsplit > 1: [rows, nsplit, dim] unnormalised, [rows, nsplit, 2] (c m - BIAS, l); rows = (sequence, head, token)
};

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Win;  // what differs between the element types
template <>
struct Win<f16> {
  static constexpr float BIAS = 7.0f, LIMIT = 32768.0f;
  static __device__ __forceinline__ void mma(f32x16& c, const uint4& a, const uint4& b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const f16x2 v = {(f16)x, (f16)y};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ float add2(uint32_t p, float acc) { return f5_sum2_f16(p, acc); }
};
template <>
struct Win<bf16> {
  static constexpr float BIAS = 0.0f, LIMIT = 256.0f;
  static __device__ __forceinline__ void mma(f32x16& c, const uint4& a, const uint4& b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const bf16x2 v = {(bf16)x, (bf16)y};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ float add2(uint32_t p, float acc) {
#ifdef F5_HIPEMU
    return acc + (__builtin_bit_cast(float, p << 16) + __builtin_bit_cast(float, p & 0xffff0000u));
#else
    const bf16x2 ones = {(bf16)1.0f, (bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), ones, acc, false);
#endif
  }
};
template <>
struct Win<float> : Win<bf16> {};  // of the pieces

// two fp32 numbers -> their pieces, a pair a plane.  Truncation: each remainder is exact, and what is left behind the second has 8 bits.
__device__ __forceinline__ void split_pair(uint32_t x, uint32_t y, uint32_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
#ifdef F5_HIPEMU
    p[i] = (x >> 16) | (y & 0xffff0000u);
#else
    p[i] = __builtin_amdgcn_perm(y, x, 0x07060302);  // the high halves
#endif
    if (i == 2) break;
    x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, x) - __builtin_bit_cast(float, x & 0xffff0000u));
    y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, y) - __builtin_bit_cast(float, y & 0xffff0000u));
  }
}
// c += a b over 16 contracted elements of one (16-bit types) or three (fp32) planes, the small products first
template <typename T>
__device__ __forceinline__ void mma_planes(f32x16& c, const uint4* a, const uint4* b) {
  if constexpr (sizeof(T) == 4) {
    Win<T>::mma(c, a[2], b[0]);
    Win<T>::mma(c, a[0], b[2]);
    Win<T>::mma(c, a[1], b[1]);
    Win<T>::mma(c, a[1], b[0]);
    Win<T>::mma(c, a[0], b[1]);
  }
  Win<T>::mma(c, a[0], b[0]);
}

// 4 rows of a row-major 16-bit tile, transposed: lanes 4 r + c of a group of 16 name 4 columns (8 bytes) of row r, lane i gets column i of the
// four rows (ds_read_b64_tr_b16)
__device__ __forceinline__ uint2 lds_read_transposed(const char* p) {
#ifdef F5_HIPEMU
  return hipemu::ds_read_tr16(p);
#else
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
#endif
}

// 16 bytes a lane from a buffer to LDS, lane l's at p + 16 l (p wave-uniform); what lies past the descriptor's end arrives as zeros
__device__ __forceinline__ void load_to_lds(BufRsrc r, uint32_t offset, char* p) {
#ifdef F5_HIPEMU
  const uint4 v = buffer_load_b128(r, offset);
  memcpy(p + 16 * hipemu::blk->cur->lane, &v, 16);
#else
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)p, 16, (int)offset, 0, 0, 0);
#endif
}
__device__ __forceinline__ void loads_to_lds_landed() {  // the wave's; a barrier makes them the workgroup's
#ifndef F5_HIPEMU
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#endif
}

// max over the lane and its partner in the other half-wave (the same query row)
__device__ __forceinline__ float both_halves_max(float x) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
  f5_swap32(a, b);
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float both_halves_sum(float x) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
  f5_swap32(a, b);
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// the windows of tokens: [low(p), high(p)) and, of the sinks, [0, min(sinks, high(p)))
struct Span {
  int n, left, right;
  __device__ __forceinline__ int high(int p) const { return right < 0 ? n : max(0, min(n, p + right + 1)); }
  __device__ __forceinline__ int low(int p) const { return left < 0 ? 0 : max(0, p - left); }
};

// a tile's rows through a buffer descriptor: rows at and past `rows`, and columns past the head's, read as zeros
__device__ __forceinline__ BufRsrc tile_rsrc(const char* base, int64_t stride_bytes, int key0, int rows, int dim_bytes) {
  const uint32_t bytes = rows > 0 ? (uint32_t)((rows - 1) * (int)stride_bytes + dim_bytes) : 0u;
  return make_rsrc(base + (int64_t)key0 * stride_bytes, bytes);
}

// the running softmax of one 32-row group: O^T (32 columns a block), reference maximum, row sum
template <typename T, int DP>
struct Rows {
  static constexpr int EB = sizeof(T), PL = EB == 4 ? 3 : 1, ND = DP / 32, NKS = DP / 16;  // planes, blocks of 32 columns, steps of 16
  static constexpr int K_ROWB = DP * 2 + 16;            // of a plane in LDS: 32 rows read 16 bytes each without conflicts
  static constexpr int V_ROWB = DP == 64 ? 192 : 320;   // 4 rows start 64 bytes apart in the 256-byte bank row
  static constexpr float UNSET = -3.402823466e38f, LIMIT = Win<T>::LIMIT;
  f32x16 o[ND];
  float mc, l;  // c m - BIAS (UNSET: no key seen, any score passes the limit), this lane's share of the row sum
  int lo, hi;      // the lane's row: its window
  uint4 fq[NKS][PL];

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    mc = UNSET;
    l = 0.f;
  }

  // the lane's row of q: columns 16 k + 8 half .. + 7 for each step, in planes; `negate` flips signs
  __device__ __forceinline__ void load_q(const T* q, bool live, int dim, int half, uint32_t negate) {
#pragma unroll
    for (int k = 0; k < NKS; ++k) {
      const int col = k * 16 + half * 8;
      uint4 u[EB / 2];
#pragma unroll
      for (int i = 0; i < EB / 2; ++i) {
        const int at = col + i * (16 / EB);
        u[i] = live && at < dim ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
        u[i].x ^= negate; u[i].y ^= negate; u[i].z ^= negate; u[i].w ^= negate;
      }
      planes(u, fq[k]);
    }
  }
  // 8 columns as loaded -> operand pieces
  static __device__ __forceinline__ void planes(const uint4 (&u)[EB / 2], uint4 (&f)[PL]) {
    if constexpr (EB == 2) {
      f[0] = u[0];
    } else {
      uint32_t p[4][3];
      split_pair(u[0].x, u[0].y, p[0]);
      split_pair(u[0].z, u[0].w, p[1]);
      split_pair(u[1].x, u[1].y, p[2]);
      split_pair(u[1].z, u[1].w, p[3]);
#pragma unroll
      for (int i = 0; i < 3; ++i) f[i] = make_uint4(p[0][i], p[1][i], p[2][i], p[3][i]);
    }
  }
  // a 16-byte piece of a K or V row, as loaded -> its place in the planes (plane bytes apart) of row `at`
  static __device__ __forceinline__ void stage(char* at, int plane, int piece, const uint4& u) {
    if constexpr (EB == 2) {
      *reinterpret_cast<uint4*>(at + piece * 16) = u;
    } else {
      uint32_t a[3], b[3];
      split_pair(u.x, u.y, a);
      split_pair(u.z, u.w, b);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(at + i * plane + piece * 8) = make_uint2(a[i], b[i]);
    }
  }

  // the keys of NB blocks of 32 that the lane's row does not see -> -inf.  `high`, `low`, `sink` (wave-uniform): which borders the tile can
  // touch — one compare and one select a score for each.
  template <int NB>
  __device__ __forceinline__ void mask(f32x16 (&s)[NB], int key0, int kend, int half, bool high, bool low, int sinks) {
    const int base = key0 + 4 * half, e = min(hi, kend) - base, b = lo - base, k = sinks - base;
    if (high) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = n * 32 + (r & 3) + 8 * (r >> 2) < e ? s[n][r] : -INFINITY;
    }
    if (low) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int off = n * 32 + (r & 3) + 8 * (r >> 2);
          s[n][r] = ((off >= b) | (off < k)) ? s[n][r] : -INFINITY;
        }
    }
  }

  // the reference raised to the tile's maximum (O, l rescaled); rows that see nothing keep theirs
  template <int NB>
  __device__ __forceinline__ void raise(const f32x16 (&s)[NB], float c) {
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    const float to = fmaxf(mc, fmaf(both_halves_max(mx), c, -Win<T>::BIAS)), al = __builtin_amdgcn_exp2f(mc - to);
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] *= al;
    l *= al;
    mc = to;
  }

  // A tile is worked through in phases of 16 keys, two for each 32: the lane's are 16 g + 4 half + 0..3 and 8 on.  V^T operands of a phase, from V rows at
  // sv (planes `plane` bytes apart):
  struct VFrag {
    uint4 v[ND][PL];
  };
  static __device__ __forceinline__ void read_v(VFrag& f, int g, const char* sv, int plane, int lane) {
    const char* at = sv + (g * 16 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * V_ROWB + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const uint2 v0 = lds_read_transposed(at + i * plane + d * 64), v1 = lds_read_transposed(at + i * plane + 8 * V_ROWB + d * 64);
        f.v[d][i] = make_uint4(v0.x, v0.y, v1.x, v1.y);
      }
  }
  // ... from rows without padding whose places are exchanged (window_rows_kernel): `at` holds the lane's place of each column block
  template <int ROWB>
  static __device__ __forceinline__ void read_v_exchanged(VFrag& f, int g, const char* sv, const uint32_t (&at)[ND]) {
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const char* p = sv + at[d] + g * 16 * ROWB;
      const uint2 v0 = lds_read_transposed(p), v1 = lds_read_transposed(p + 8 * ROWB);
      f.v[d][0] = make_uint4(v0.x, v0.y, v1.x, v1.y);
    }
  }
  // the weights of a tile's keys, as the second product takes them (pairs, in planes), and the row sum; the reference raised where it has to be
  template <int NB>
  struct Weights {
    uint32_t p[PL][NB * 8];
  };
  template <int NB>
  __device__ __forceinline__ float weights_once(const f32x16 (&s)[NB], Weights<NB>& w, float c) const {
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[n][r], c, -mc)), y = __builtin_amdgcn_exp2f(fmaf(s[n][r + 1], c, -mc));
        if constexpr (EB == 2) {
          const uint32_t p = Win<T>::pack(x, y);
          w.p[0][n * 8 + r / 2] = p;
          sum = Win<T>::add2(p, sum);  // of the rounded weights: numerator and denominator see the same ones
        } else {
          uint32_t p[3];
          split_pair(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), p);
#pragma unroll
          for (int i = 0; i < PL; ++i) w.p[i][n * 8 + r / 2] = p[i];
          sum += x + y;
        }
      }
    return sum;
  }
  template <int NB>
  __device__ __forceinline__ void weigh(const f32x16 (&s)[NB], Weights<NB>& w, float c) {
    float sum = weights_once(s, w, c);
    if (f5_wave_any(sum > LIMIT)) {
      raise(s, c);
      sum = weights_once(s, w, c);
    }
    l += sum;
  }
  // O^T += V^T P^T over phase g's keys
  template <int NB>
  __device__ __forceinline__ void product(const Weights<NB>& w, int g, const VFrag& f) {
    uint4 p[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i) p[i] = make_uint4(w.p[i][4 * g], w.p[i][4 * g + 1], w.p[i][4 * g + 2], w.p[i][4 * g + 3]);
#pragma unroll
    for (int d = 0; d < ND; ++d) mma_planes<T>(o[d], f.v[d], p);
  }
  __device__ __forceinline__ float reference() const { return mc == UNSET ? -INFINITY : mc; }
};

// four neighbouring columns of an output row
template <typename T>
__device__ __forceinline__ void store4(T* p, float x0, float x1, float x2, float x3) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(x0, x1, x2, x3);
  else *reinterpret_cast<uint2*>(p) = make_uint2(Win<T>::pack(x0, x1), Win<T>::pack(x2, x3));
}

// XCD-aware placement: block b runs on XCD b % 8, so give each XCD a contiguous range of the order — the row blocks and key ranges of one key head
// are neighbours in it and share an L2.  A bijection for any grid.
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
}
// ... and deal the (sequence, key head) units to those ranges in turn: place i of the order is unit 0, 8, 16 ..., 1, 9 ...  Neighbouring units are heads of
// one sequence, so sequences of different lengths would otherwise load the XCDs differently.
__device__ __forceinline__ int spread_units(int i, int n) {
  const int q = n >> 3, r = n & 7, big = r * (q + 1);
  return i < big ? (i % (q + 1)) * 8 + i / (q + 1) : ((i - big) % q) * 8 + r + (i - big) / q;
}

// A workgroup's place in the order.  Blocks of rows go from the last one down: later tokens see more keys (a window cut off at the sequence's start is
// shorter), so what is left for the end of the launch is short.  Where every XCD has up to eight whole units, their blocks take turns, for the same reason (2 x 1406
// frames of 16 heads, 4 units an XCD: 22.3 -> 20.4 us, in fp32 79 -> 70 us; 2 x 8192 frames 142 -> 138 us); with more, a unit's blocks would be so far apart in
// time that its keys leave L2 between them (16 utterances of 12 heads, 24 units: 45 us one unit after the other, 49 us in turns).
struct Place {
  int ks, blk, bh;
};
__device__ __forceinline__ Place place_of(const WindowArgs& a, int block) {
  Place p;
  int i;
  if (a.xcd_units) {
    const int l = block >> 3;
    p.ks = l % a.nsplit;
    i = l / a.nsplit;
    p.bh = i % a.xcd_units * 8 + (block & 7);
    i /= a.xcd_units;
  } else {
    const int l = xcd_order(block, a.nwg);
    p.ks = l % a.nsplit;
    i = l / a.nsplit;
    p.bh = spread_units(i / a.nblk, a.batch * a.kv_heads);
    i %= a.nblk;
  }
  p.blk = a.nblk - 1 - i;
  return p;
}

// ---- many rows: K and V tiles of 64 keys shared through LDS, two stages ------------------------------------------------------------------------------
// Four waves: 4 / KG groups of 32 rows x KG ranges of keys.  KG = 1: 128 rows a workgroup, a wave takes whole tiles.  KG = 2: 64 rows, a wave takes one half
// of every tile and the two halves' results meet in LDS at the end — twice the workgroups, each half as long, where row blocks alone load the CUs unevenly.
// The tiles of a row block in order: keys [0, ea), then [bb, khigh).
// 16-bit tiles go from memory to LDS without registers on the way (2 x 8192 frames of 16 heads of 64: 148 -> 142 us, and the 40 registers saved make room for
// a fourth workgroup a CU: 139 us).  Such loads write 64 lanes' pieces side by side, so rows have no padding; instead the pieces of a row change places by its
// number — K: 16 bytes by all 8 or 16 places, so that 16 rows read at one column hit 16 different places of the 256-byte bank row; V: 64 bytes, so that the 4
// rows of a transposing read do — in the addresses that are loaded and in those that are read.  Rows of up to 96 and 128 columns take 256 bytes.
struct Tiles {
  int key0, kend;  // the tile's first key, its range's end
};

template <typename T, int DP, int KG>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP == 64 ? 4 : sizeof(T) == 4 && DP > 64 ? 1 : 2) void window_rows_kernel(WindowArgs a) {
  using R = Rows<T, DP>;
  // (fp32 planes are three times as large: 32 keys, or one stage)
  constexpr bool DMA = sizeof(T) == 2;
  constexpr int EB = R::EB, KT = DMA || KG == 2 ? 64 : 32, NB = KT / 32 / KG, ROWS = 128 / KG, STAGES = DMA || KG == 1 ? 2 : 1;
  constexpr int ROWB = DP == 64 ? 128 : 256, CPR = DMA ? ROWB / 16 : DP * EB / 16, NP = KT * CPR, NL = (NP + 255) / 256;  // pieces of 16 bytes: a row's, a tile's, a thread's
  constexpr int KPL = KT * (DMA ? ROWB : R::K_ROWB), VPL = KT * (DMA ? ROWB : R::V_ROWB), KB = R::PL * KPL, VB = R::PL * VPL;
  static_assert(!DMA || NP % 256 == 0, "whole wave instructions");
  // (an array a stage: the compiler then sees that what is read now is not what is being loaded)
  __shared__ __attribute__((aligned(1024))) char stage0[KB + VB];
  __shared__ __attribute__((aligned(1024))) char stage1[STAGES == 2 ? KB + VB : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, ql = lane & 31;
  const Place pl = place_of(a, (int)blockIdx.x);
  const int ks = pl.ks, blk = pl.blk, b = pl.bh / a.kv_heads, kvh = pl.bh - b * a.kv_heads;
  const int n = a.kv_len ? max(0, min(a.kv_len[b], a.tk)) : a.tk, nq = a.q_len ? max(0, min(a.q_len[b], a.tq)) : a.tq;
  const int first = blk * ROWS / a.group;
  if (first >= nq) return;  // (the whole workgroup: no barrier has been reached)
  const int p0 = a.align_end ? n - nq : 0;
  const Span sp{n, a.left, a.right};
  const int last = min(nq - 1, (blk * ROWS + ROWS - 1) / a.group);
  const int khigh = sp.high(p0 + last), klow = min(sp.low(p0 + first), khigh), ksink = min(a.sinks, khigh);
  const int ea = klow <= ksink ? 0 : ksink, bb = klow <= ksink ? 0 : klow;  // keys [0, ea) and [bb, khigh)
  const int na = (ea + KT - 1) / KT, nt = na + (khigh - bb + KT - 1) / KT;
  const int t0 = (int)((int64_t)ks * nt / a.nsplit), t1 = (int)((int64_t)(ks + 1) * nt / a.nsplit);

  // the wave's rows, the lane's row
  const int r0 = blk * ROWS + wave / KG * 32, kg = wave % KG, row = r0 + ql, tok = row / a.group, head = kvh * a.group + (row - tok * a.group);
  const bool live = tok < nq;
  const int wfirst = r0 / a.group, wlast = min(nq - 1, (r0 + 31) / a.group);
  // the tightest and widest borders of the wave's rows; no row at all: nothing is seen
  const int whi0 = sp.high(p0 + wfirst), whi1 = wfirst < nq ? sp.high(p0 + wlast) : 0, wlo0 = sp.low(p0 + wfirst), wlo1 = sp.low(p0 + wlast);
  R st;
  st.reset();
  st.lo = sp.low(p0 + tok);
  st.hi = live ? sp.high(p0 + tok) : 0;
  st.load_q(static_cast<const T*>(a.q) + b * a.q_stride[0] + tok * a.q_stride[1] + head * a.q_stride[2], live, a.dim, half, a.negate);

  const int64_t ksb = a.k_stride[1] * EB, vsb = a.v_stride[1] * EB;
  const int dimb = a.dim * EB;
  uint4 rk[NL], rv[NL];     // (fp32)
  uint32_t ok[NL], ov[NL];  // the thread's pieces of a tile (rows past its last key are past the descriptor's end, columns past the head's are put there)
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = tid + i * 256, r = c / CPR, at = c - r * CPR;
    const int ck = DMA ? at ^ (DP == 64 ? r >> 1 & 7 : r & 15) : at, cv = DMA ? at ^ (DP == 64 ? r >> 1 & 1 : r & 3) * 4 : at;
    const bool in = NP % 256 == 0 || c < NP;
    ok[i] = in && ck * 16 < dimb ? (uint32_t)(r * (int)ksb + ck * 16) : OOB_ROW;
    ov[i] = in && cv * 16 < dimb ? (uint32_t)(r * (int)vsb + cv * 16) : OOB_ROW;
  }
  uint32_t atk[R::NKS], atv[R::ND];  // (16-bit types) the lane's places of its K pieces and V blocks in a tile
#pragma unroll
  for (int k = 0; k < R::NKS; ++k) atk[k] = (kg * 32 * NB + ql) * ROWB + ((2 * k + half) ^ (DP == 64 ? ql >> 1 & 7 : ql & 15)) * 16;
#pragma unroll
  for (int d = 0; d < R::ND; ++d) {
    const int r = (lane & 15) >> 2;
    atv[d] = (kg * 32 * NB + 4 * half + r) * ROWB + (d ^ (DP == 64 ? r >> 1 : r)) * 64 + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
  }
  const char* kb = static_cast<const char*>(a.k) + (b * a.k_stride[0] + kvh * a.k_stride[2]) * EB;
  const char* vb = static_cast<const char*>(a.v) + (b * a.v_stride[0] + kvh * a.v_stride[2]) * EB;
  Tiles ahead{t0 < na ? t0 * KT : bb + (t0 - na) * KT, t0 < na ? ea : khigh};  // the tile to load next, and where its rows are
  const char *kp = kb + ahead.key0 * ksb, *vp = vb + ahead.key0 * vsb;
  const int64_t kstep = KT * ksb, vstep = KT * vsb;
  const auto advance = [&] {
    ahead.key0 += KT;
    kp += kstep;
    vp += vstep;
    if (ahead.key0 >= ahead.kend && ahead.kend != khigh) {
      ahead = Tiles{bb, khigh};
      kp = kb + bb * ksb;
      vp = vb + bb * vsb;
    }
  };
  const auto place = [&](auto S) { return decltype(S)::value ? stage1 : stage0; };
  const auto load = [&](auto S) {  // (a row's last piece may lie past the descriptor's end: zeros)
    const int rows = min(KT, ahead.kend - ahead.key0);
    const BufRsrc Kr = make_rsrc(kp, (uint32_t)((rows - 1) * (int)ksb + dimb)), Vr = make_rsrc(vp, (uint32_t)((rows - 1) * (int)vsb + dimb));
    if constexpr (DMA) {
      char* to = place(S) + wave * 1024;
#pragma unroll
      for (int i = 0; i < NL; ++i) load_to_lds(Kr, ok[i], to + i * 4096);
#pragma unroll
      for (int i = 0; i < NL; ++i) load_to_lds(Vr, ov[i], to + KB + i * 4096);
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) rk[i] = buffer_load_b128(Kr, ok[i]);
#pragma unroll
      for (int i = 0; i < NL; ++i) rv[i] = buffer_load_b128(Vr, ov[i]);
    }
  };
  const auto store = [&](auto S) {
    if constexpr (DMA) {
      loads_to_lds_landed();
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int c = tid + i * 256, r = c / CPR, col = c - r * CPR;
        if (NP % 256 == 0 || c < NP) {
          R::stage(place(S) + r * R::K_ROWB, KPL, col, rk[i]);
          R::stage(place(S) + KB + r * R::V_ROWB, VPL, col, rv[i]);
        }
      }
    }
  };
  const float c = a.scale_log2;
  const auto work = [&](const Tiles& t, auto S) {
    const int key0 = t.key0 + kg * 32 * NB;  // the wave's keys of the tile
    if (key0 >= min(whi1, t.kend) || (min(key0 + 32 * NB, t.kend) <= wlo0 && key0 >= a.sinks)) return;  // none of its rows sees one (wave-uniform)
    const char* sk = place(S) + (DMA ? 0 : (kg * 32 * NB + ql) * R::K_ROWB + half * 16);
    const char* sv = place(S) + KB + (DMA ? 0 : kg * 32 * NB * R::V_ROWB);
    f32x16 s[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[nb][r] = 0.f;
    // Operands are read from LDS one step ahead of the matrix instructions that take them — one or two steps of K, or the V pieces of a phase — and the scheduling
    // barriers keep the compiler from sinking the reads back to their uses (a wave then sits out an LDS round trip at each).
    constexpr int QS = R::PL == 3 ? 1 : 2, NQ = NB * R::NKS / QS, PH = 2 * NB;
    static_assert(NB * R::NKS % QS == 0, "whole steps of K pieces");
    uint4 fk[2][QS][R::PL];
    const auto read_k = [&](auto C) {
      constexpr int q = decltype(C)::value;
#pragma unroll
      for (int i = 0; i < QS; ++i)
#pragma unroll
        for (int p = 0; p < R::PL; ++p)
          fk[q & 1][i][p] = *reinterpret_cast<const uint4*>(sk + p * KPL + (QS * q + i) / R::NKS * 32 * (DMA ? ROWB : R::K_ROWB) +
                                                            (DMA ? atk[(QS * q + i) % R::NKS] : (QS * q + i) % R::NKS * 32));
    };
    const auto read_v = [&](typename R::VFrag& f, int g) {
      if constexpr (DMA) R::template read_v_exchanged<ROWB>(f, g, sv, atv);
      else R::read_v(f, g, sv, VPL, lane);
    };
    typename R::VFrag fv[2];
    read_k(std::integral_constant<int, 0>{});
    static_for<NQ>([&](auto Q) {
      constexpr int q = decltype(Q)::value;
      if constexpr (q + 1 < NQ) read_k(std::integral_constant<int, q + 1>{});
      else read_v(fv[0], 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < QS; ++i) mma_planes<T>(s[(QS * q + i) / R::NKS], fk[q & 1][i], st.fq[(QS * q + i) % R::NKS]);
      __builtin_amdgcn_sched_barrier(0);
    });
    st.mask(s, key0, t.kend, half, key0 + 32 * NB > min(whi0, t.kend), key0 < wlo1 && key0 + 32 * NB > a.sinks, a.sinks);
    typename R::template Weights<NB> w;
    st.weigh(s, w, c);
    static_for<PH>([&](auto G) {
      constexpr int g = decltype(G)::value;
      if constexpr (g + 1 < PH) read_v(fv[(g + 1) & 1], g + 1);
      __builtin_amdgcn_sched_barrier(0);
      st.product(w, g, fv[g & 1]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  if (t0 < t1) {
    Tiles at = ahead;
    constexpr std::integral_constant<int, 0> S0{};
    constexpr std::integral_constant<int, STAGES - 1> S1{};
    const auto step = [&](int t, auto S, auto next) {
      const bool more = t + 1 < t1;
      if (more) {
        advance();
        load(next);
      }
      work(at, S);
      if constexpr (STAGES == 1) __syncthreads();  // every wave has read the one stage
      if (more) store(next);
      __syncthreads();
      at = ahead;
    };
    load(S0);
    store(S0);
    __syncthreads();
    for (int t = t0; t < t1; t += STAGES) {
      step(t, S0, S1);
      if (STAGES == 2 && t + 1 < t1) step(t + 1, S1, S0);
    }
  }

#ifndef F5_HIPEMU
  // O as one register tuple behind the loop: left to itself the compiler gathers what the epilogue reads inside the loop, 32 moves behind every tile's
  // matrix instructions
#pragma unroll
  for (int d = 0; d < R::ND; ++d) asm volatile("" : "+v"(st.o[d]));
#endif
  float l = both_halves_sum(st.l), top = st.reference();
  if constexpr (KG == 2) {  // the second half's result through LDS (its places have been read: the loop ended at a barrier), columns as the lanes hold them
    constexpr int LANE_FLOATS = 16 * R::ND + 2;
    static_assert(KB + VB >= (3 - STAGES) * 64 * LANE_FLOATS * 4, "the halves meet in the tiles' place");
    float* x = reinterpret_cast<float*>(wave >= 2 && STAGES == 2 ? stage1 : stage0) + (STAGES == 1 ? wave / 2 * 64 * LANE_FLOATS : 0) + lane;
    if (kg == 1) {
#pragma unroll
      for (int d = 0; d < R::ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[(d * 16 + r) * 64] = st.o[d][r];
      x[16 * R::ND * 64] = top;
      x[(16 * R::ND + 1) * 64] = l;
    }
    __syncthreads();
    if (kg == 1) return;
    const float top1 = x[16 * R::ND * 64], l1 = x[(16 * R::ND + 1) * 64], both = fmaxf(top, top1);
    const float f0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - both), f1 = top1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top1 - both);
#pragma unroll
    for (int d = 0; d < R::ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.o[d][r] = st.o[d][r] * f0 + x[(d * 16 + r) * 64] * f1;
    l = l * f0 + l1 * f1;
    top = both;
  }
  if (!live) return;
  if (a.nsplit > 1) {
    const int64_t part = (((int64_t)b * a.heads + head) * a.tq + tok) * a.nsplit + ks;
    float* po = a.part_o + part * a.dim;
#pragma unroll
    for (int d = 0; d < R::ND; ++d)
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const int col = d * 32 + 8 * c4 + 4 * half;
        if (col < a.dim) *reinterpret_cast<float4*>(po + col) = make_float4(st.o[d][4 * c4], st.o[d][4 * c4 + 1], st.o[d][4 * c4 + 2], st.o[d][4 * c4 + 3]);
      }
    if (half == 0) {
      a.part_ml[part * 2] = top;
      a.part_ml[part * 2 + 1] = l;
    }
    return;
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  T* op = static_cast<T*>(a.out) + b * a.out_stride[0] + tok * a.out_stride[1] + head * a.out_stride[2];
#pragma unroll
  for (int d = 0; d < R::ND; ++d)
#pragma unroll
    for (int c4 = 0; c4 < 4; ++c4) {
      const int col = d * 32 + 8 * c4 + 4 * half;
      if (col < a.dim) store4(op + col, st.o[d][4 * c4] * inv, st.o[d][4 * c4 + 1] * inv, st.o[d][4 * c4 + 2] * inv, st.o[d][4 * c4 + 3] * inv);
    }
}

// ---- few rows: one 32-row group, the waves along the keys ----------------------------------------------------------------------------------------
// Every wave walks 32-key tiles of its own (tile t belongs to wave t % NW): K straight into operand registers, V through the wave's own LDS rows, no
// barrier on the way, the next tile's loads issued as soon as the registers are free; the waves' results meet in LDS at the end, in a fixed order.
// 8 waves; 4 in fp32, whose operands of one tile fill a 512-register wave.
template <typename T>
constexpr int FEW_WAVES = sizeof(T) == 4 ? 4 : 8;
template <typename T, int DP>
__global__ __launch_bounds__(64 * FEW_WAVES<T>, 1) void window_few_kernel(WindowArgs a) {
  using R = Rows<T, DP>;
  constexpr int NW = FEW_WAVES<T>, KT = 32, EB = R::EB, CPR = DP * EB / 16, NL = KT * CPR / 64;
  constexpr int VPL = KT * R::V_ROWB, VB = R::PL * VPL, MERGE = NW * 32 * 33 * 4, EK = EB / 2;  // EK: 16-byte loads of a lane's 8 columns of K
  __shared__ __attribute__((aligned(16))) char smem[NW * VB > MERGE ? NW * VB : MERGE];
  __shared__ float sml[NW][32][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, ql = lane & 31;
  const Place pl = place_of(a, (int)blockIdx.x);
  const int ks = pl.ks, blk = pl.blk, b = pl.bh / a.kv_heads, kvh = pl.bh - b * a.kv_heads;
  const int n = a.kv_len ? max(0, min(a.kv_len[b], a.tk)) : a.tk, nq = a.q_len ? max(0, min(a.q_len[b], a.tq)) : a.tq;
  const int first = blk * 32 / a.group;
  if (first >= nq) return;  // (the whole workgroup)
  const int p0 = a.align_end ? n - nq : 0;
  const Span sp{n, a.left, a.right};
  const int last = min(nq - 1, (blk * 32 + 31) / a.group);
  const int high0 = sp.high(p0 + first), khigh = sp.high(p0 + last), low1 = sp.low(p0 + last), klow = min(sp.low(p0 + first), khigh), ksink = min(a.sinks, khigh);
  const int ea = klow <= ksink ? 0 : ksink, bb = klow <= ksink ? 0 : klow;
  const int na = (ea + KT - 1) / KT, nt = na + (khigh - bb + KT - 1) / KT;
  const int t0 = (int)((int64_t)ks * nt / a.nsplit), t1 = (int)((int64_t)(ks + 1) * nt / a.nsplit);

  const int row = blk * 32 + ql, tok = row / a.group, g = row - tok * a.group, head = kvh * a.group + g;
  const bool live = tok < nq;
  R st;
  st.reset();
  st.lo = sp.low(p0 + tok);
  st.hi = live ? sp.high(p0 + tok) : 0;
  st.load_q(static_cast<const T*>(a.q) + b * a.q_stride[0] + tok * a.q_stride[1] + head * a.q_stride[2], live, a.dim, half, a.negate);
  const char* kb = static_cast<const char*>(a.k) + (b * a.k_stride[0] + kvh * a.k_stride[2]) * EB;
  const char* vb = static_cast<const char*>(a.v) + (b * a.v_stride[0] + kvh * a.v_stride[2]) * EB;
  const int64_t ksb = a.k_stride[1] * EB, vsb = a.v_stride[1] * EB;
  const int dimb = a.dim * EB;
  char* sv = smem + wave * VB;

  const auto tile = [&](int t, int& key0, int& kend) {
    key0 = t < na ? t * KT : bb + (t - na) * KT;
    kend = t < na ? ea : khigh;
  };
  uint4 fk[R::NKS][EK], rv[NL];
  uint32_t ok[R::NKS][EK], ov[NL];
#pragma unroll
  for (int k = 0; k < R::NKS; ++k)
#pragma unroll
    for (int i = 0; i < EK; ++i) {
      const int col = (k * 16 + half * 8) * EB + i * 16;  // bytes
      ok[k][i] = col < dimb ? (uint32_t)(ql * (int)ksb + col) : OOB_ROW;
    }
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = lane + i * 64, r = c / CPR, col = c - r * CPR;
    ov[i] = col * 16 < dimb ? (uint32_t)(r * (int)vsb + col * 16) : OOB_ROW;
  }
  const auto load_k = [&](int t) {
    int key0, kend;
    tile(t, key0, kend);
    const BufRsrc Kr = tile_rsrc(kb, ksb, key0, min(KT, kend - key0), dimb);
#pragma unroll
    for (int k = 0; k < R::NKS; ++k)
#pragma unroll
      for (int i = 0; i < EK; ++i) fk[k][i] = buffer_load_b128(Kr, ok[k][i]);
  };
  const auto load_v = [&](int t) {
    int key0, kend;
    tile(t, key0, kend);
    const BufRsrc Vr = tile_rsrc(vb, vsb, key0, min(KT, kend - key0), dimb);
#pragma unroll
    for (int i = 0; i < NL; ++i) rv[i] = buffer_load_b128(Vr, ov[i]);
  };
  if (t0 + wave < t1) {
    load_k(t0 + wave);
    load_v(t0 + wave);
  }
  for (int t = t0 + wave; t < t1; t += NW) {
    int key0, kend;
    tile(t, key0, kend);
    f32x16 s[1];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
    for (int k = 0; k < R::NKS; ++k) {
      uint4 f[R::PL];
      R::planes(fk[k], f);
      mma_planes<T>(s[0], f, st.fq[k]);
    }
    if (t + NW < t1) load_k(t + NW);  // as soon as its registers are free
    wave_lds_sync();                  // the last tile's reads of these rows come before
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = lane + i * 64, r = c / CPR, col = c - r * CPR;
      R::stage(sv + r * R::V_ROWB, VPL, col, rv[i]);
    }
    if (t + NW < t1) load_v(t + NW);
    st.mask(s, key0, kend, half, key0 + KT > min(high0, kend), key0 < low1 && key0 + KT > a.sinks, a.sinks);
    typename R::template Weights<1> w;
    st.weigh(s, w, a.scale_log2);
    wave_lds_sync();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      typename R::VFrag f;
      R::read_v(f, g, sv, VPL, lane);
      st.product(w, g, f);
    }
  }

  // the waves' parts: common reference, then 32 columns at a time through LDS, summed in the waves' order
  const float l = both_halves_sum(st.l);
  if (half == 0) {
    sml[wave][ql][0] = st.reference();
    sml[wave][ql][1] = l;
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) top = fmaxf(top, sml[w][ql][0]);
  const float mine = sml[wave][ql][0], f = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - top);
  float* sm = reinterpret_cast<float*>(smem);
  for (int d = 0; d < R::ND; ++d) {
    __syncthreads();  // the V rows, or the columns before, have been read
#pragma unroll
    for (int dd = 0; dd < R::ND; ++dd)  // (a register array is indexed with constants only)
      if (dd == d)
#pragma unroll
        for (int r = 0; r < 16; ++r) sm[(wave * 32 + (r & 3) + 8 * (r >> 2) + 4 * half) * 33 + ql] = st.o[dd][r] * f;
    __syncthreads();
    for (int v = tid; v < 1024; v += 64 * NW) {
      const int rr = v >> 5, cc = v & 31, col = d * 32 + cc, orow = blk * 32 + rr, otok = orow / a.group;
      if (otok >= nq || col >= a.dim) continue;
      const int ohead = kvh * a.group + (orow - otok * a.group);
      float x = 0.f, rtop = -INFINITY, rl = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        x += sm[(w * 32 + cc) * 33 + rr];
        rtop = fmaxf(rtop, sml[w][rr][0]);
      }
#pragma unroll
      for (int w = 0; w < NW; ++w) rl += sml[w][rr][0] == -INFINITY ? 0.f : sml[w][rr][1] * __builtin_amdgcn_exp2f(sml[w][rr][0] - rtop);
      if (a.nsplit > 1) {
        const int64_t part = (((int64_t)b * a.heads + ohead) * a.tq + otok) * a.nsplit + ks;
        a.part_o[part * a.dim + col] = x;
        if (col == 0) { a.part_ml[part * 2] = rtop; a.part_ml[part * 2 + 1] = rl; }
      } else {
        T* op = static_cast<T*>(a.out) + b * a.out_stride[0] + otok * a.out_stride[1] + ohead * a.out_stride[2];
        op[col] = (T)(rl > 0.f ? x / rl : x * 0.f);  // nothing seen: 0; a NaN seen: NaN
      }
    }
  }
}

// ---- join of the key ranges: a thread per four columns of a row -----------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
  const int quads = a.dim / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / quads;
  if (row >= (int64_t)a.batch * a.heads * a.tq) return;
  const int col = (int)(id - row * quads) * 4, bh = (int)(row / a.tq), tok = (int)(row - (int64_t)bh * a.tq), b = bh / a.heads, head = bh - b * a.heads;
  const int nq = a.q_len ? max(0, min(a.q_len[b], a.tq)) : a.tq;
  if (tok >= nq) return;
  const float* ml = a.part_ml + row * a.nsplit * 2;
  const float* po = a.part_o + row * a.nsplit * a.dim + col;
  float top = -INFINITY;
  for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, ml[2 * s]);
  float l = 0.f, x0 = 0.f, x1 = 0.f, x2 = 0.f, x3 = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float f = ml[2 * s] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[2 * s] - top);
    const float4 x = *reinterpret_cast<const float4*>(po + (int64_t)s * a.dim);
    l += f * ml[2 * s + 1];
    x0 += f * x.x; x1 += f * x.y; x2 += f * x.z; x3 += f * x.w;
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  T* op = static_cast<T*>(a.out) + b * a.out_stride[0] + tok * a.out_stride[1] + head * a.out_stride[2] + col;
  store4(op, x0 * inv, x1 * inv, x2 * inv, x3 * inv);
}
}  // namespace
