// Pieces shared by the attention kernels whose scores follow a rule (attn_scored.hip, attn_cached.hip): operands of 16 and
// 32 bits, the cap, and the products of a step of 32 streamed rows with an own row per MFMA column.
#pragma once

#include <cfloat>
#include <type_traits>

#include "attn_tile.h"
#include "sa_common.h"

namespace {

constexpr int kStep = 32;          // streamed rows per step, own rows per wave
constexpr int kMostRadius = 1024;  // distances that a bias tells apart
// A row's offset (log2 units) is left where it is until its maximum lies more than kAbove over it; then it is put kBelow under
// that. P stays below 2^kAbove. fp16 has no number under 2^-25 but zero: with the offset at the maximum itself, 45104 keys of
// 2^-25.5 behind a strong one lost 1e-3 of the row; this way what is below 2^-36 of the maximum is lost.
template <typename T>
constexpr float kAbove = std::is_same<T, _Float16>::value ? 15.f : 8.f;
template <typename T>
constexpr float kBelow = std::is_same<T, _Float16>::value ? 11.f : 0.f;

template <typename T>
__device__ inline float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __bf16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const sa_f16x2 h = __builtin_bit_cast(sa_f16x2, w);
  return make_float2((float)h[0], (float)h[1]);
}

// Sum of the products of two 16-byte chunks.
template <typename T>
__device__ inline float dot_chunk(sa_u32x4v x, sa_u32x4v y, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      s = fmaf(__uint_as_float(x[i]), __uint_as_float(y[i]), s);
    } else {
      const float2 u = unpack2<T>(x[i]), w = unpack2<T>(y[i]);
      s = fmaf(u.x, w.x, fmaf(u.y, w.y, s));
    }
  }
  return s;
}

// A 32 x 32 product over the 32 bytes of a row that chunks 2 s and 2 s + 1 hold (the order of the terms is the
// same for both operands, whatever it is).
template <typename T>
__device__ inline sa_f32x16 mfma_chunk(sa_u32x4v a, sa_u32x4v b, sa_f32x16 c) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  } else {
    return Elem<T>::mfma(Elem<T>::as8(a), Elem<T>::as8(b), c);
  }
}

// 16 weights of an own row (one register each in fp32, pairs otherwise).
template <typename T>
struct Weights {
  uint32_t w[8];
  __device__ inline void set(int e, float a, float b) { w[e >> 1] = Elem<T>::pack(a, b); }
  __device__ inline float sum(float s) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) s = Elem<T>::dot2_ones(w[i], s);
    return s;
  }
};
template <>
struct Weights<float> {
  sa_f32x16 w;
  __device__ inline void set(int e, float a, float b) {
    w[e] = a;
    w[e + 1] = b;
  }
  __device__ inline float sum(float s) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) s += w[i];
    return s;
  }
};

// Two weights as two terms of the type each, exact to its bits twice over. bf16: the upper halves of the floats, so that
// they are picked out of the registers, and the rest rounded (a dot product in place of the mask and the subtraction is
// slower: 266 us of a pass, not 250). fp16: what the first term leaves is one multiply-add that reads and writes fp16.
template <typename T>
__device__ __forceinline__ void set_two_terms(Weights<T>& hi, Weights<T>& lo, int e, float a, float b) {
  if constexpr (std::is_same<T, float>::value) {
    hi.set(e, a, b);
  } else if constexpr (std::is_same<T, __bf16>::value) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    hi.w[e >> 1] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    lo.set(e, a - __uint_as_float(x & 0xffff0000u), b - __uint_as_float(y & 0xffff0000u));
  } else {
    hi.set(e, a, b);
    float minus = -1.f;
    asm("" : "+v"(hi.w[e >> 1]), "+s"(minus));  // (so that they stay multiply-adds of the pair's halves)
    const sa_f16x2 h = __builtin_bit_cast(sa_f16x2, hi.w[e >> 1]);
    lo.set(e, fmaf((float)h[0], minus, a), fmaf((float)h[1], minus, b));
  }
}

// cap tanh(y) and 1 - tanh(y)^2, in one of two ways. Fine: below 0.6 the odd polynomial through tanh(y) / y at Chebyshev nodes
// (relative error 7e-8), because a small score would otherwise lose its bits. Else cap - 2 cap / (exp2(y') + 1), whose error is
// absolute, 2e-7 cap; y' = 2 log2(e) y is the argument. fp32 calls are fine, 16-bit ones where the cap is above kFineCap, whose
// 2e-7 is a tenth of fp16's rounding of P (at a cap of 1e4 scores were off by 0.002, at 1e7 by 1.7). The derivative 4 (r - r^2)
// of r = 1 / (exp2(y') + 1) keeps its bits above 0; towards minus the cap, where r is close to 1, it is off by 2^-22.
constexpr float kFineCap = 256.f, kLeastCap = 1e-12f;  // (below that fine, too: what the key pass hides pairs by counts in caps)
__device__ inline float bend_r(float y) { return __builtin_amdgcn_rcpf(fast_exp2(y) + 1.f); }
template <bool kFine, bool kSlope>
__device__ inline float bend(float y, float cap, float& slope) {
  if constexpr (kFine) {
    const float z = y * y;
    float p = 2.3734868e-3f;
    p = fmaf(p, z, -8.4125260e-3f);
    p = fmaf(p, z, 2.1789098e-2f);
    p = fmaf(p, z, -5.3961653e-2f);
    p = fmaf(p, z, 1.3333313e-1f);
    p = fmaf(p, z, -3.3333334e-1f);
    const float r = __builtin_amdgcn_rcpf(fast_exp2(y * (2.f * kLog2e)) + 1.f);
    const float t = fabsf(y) < 0.6f ? fmaf(y * z, p, y) : fmaf(r, -2.f, 1.f);
    if constexpr (kSlope) slope = fabsf(y) < 0.6f ? fmaf(-t, t, 1.f) : 4.f * fmaf(-r, r, r);
    return t * cap;
  } else {
    const float r = bend_r(y);
    if constexpr (kSlope) slope = 4.f * fmaf(-r, r, r);
    return fmaf(r, -2.f * cap, cap);
  }
}

// The capped products of a tile.
template <bool kFine, bool kSlope>
__device__ __forceinline__ void bend_all(float cap_in, float cap, sa_f32x16& S, sa_f32x16& slope) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float t = 0.f;
    S[e] = bend<kFine, kSlope>(S[e] * cap_in, cap, t);
    if constexpr (kSlope) slope[e] = t;
  }
}

// A call's cap as the kernels have it: the products' factor, the cap times log2(e), and the way.
struct Cap {
  float in, log2;
  int fine;
};
inline Cap cap_of(float sm_scale, float cap, int dtype) {
  Cap c{};
  if (!(cap > 0)) return c;
  c.fine = dtype == SA_DTYPE_F32 || cap > kFineCap || cap < kLeastCap;
  c.in = sm_scale / cap * (c.fine ? 1.f : 2.f * kLog2e);
  c.log2 = cap * kLog2e;
  return c;
}
// Caps and scales whose quotient is a normal number, with room for its factors.
inline bool cap_in_range(float sm_scale, float cap) {
  return !cap || (cap > 1e-30f && cap < 1e30f && sm_scale / cap * 3.f <= FLT_MAX && sm_scale / cap >= FLT_MIN);
}

__device__ inline float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == SA_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == SA_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}

// A step's rows of one matrix in LDS: kD * sizeof(T) / 128 pieces of 32 rows of 128 bytes, 16-byte chunks swizzled by the
// row. row(): where lane (col, hh) reads its part of chunks 2 c and 2 c + 1 of row col, for the first products' A operand.
// product(): to[d][own] += rows^T W, W in the layout of the first products' results. 16-bit types read 4 x 16 blocks
// transposed; fp32 reads value col of the 32 of a piece, of streamed row 8 (e / 4) + 4 hh + e % 4.
template <typename T, int kD>
struct TileReads {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int kPiece = kStep * 128;
  int ro[4], tr[kF32 ? 8 : 4];
  __device__ inline explicit TileReads(int lane) {
    const int col = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int s = 0; s < 4; ++s) ro[s] = 128 * col + 16 * ((2 * s + hh) ^ swz(col));
    if constexpr (kF32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = 8 * (e >> 2) + 4 * hh + (e & 3);
        tr[e] = 128 * r + 16 * ((col >> 2) ^ swz(r)) + 4 * (col & 3);
      }
    } else {
      const int i = lane & 15, dg = (lane >> 4) & 1;
#pragma unroll
      for (int dc = 0; dc < 2; ++dc)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int r = 8 * t + 4 * hh + (i >> 2);
          const int chunk = 4 * dc + 2 * dg + ((i & 3) >> 1);
          tr[2 * dc + t] = 128 * r + 16 * (chunk ^ swz(r)) + 8 * (i & 1);
        }
    }
  }
  __device__ inline const lds_u8* row(const lds_u8* mat, int c) const { return mat + ro[c & 3] + (c >> 2) * kPiece; }
  // 16-bit types: 64 columns transposed, and to += those columns' rows^T W.
  struct Columns {
    sa_u32x4v x[2][2];  // [16 streamed rows][32 columns]
  };
  __device__ __forceinline__ Columns columns(const lds_u8* mat, int hf) const {
    Columns r;
    if constexpr (!kF32) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dc = 0; dc < 2; ++dc) {
          const lds_u8* p = mat + hf * kPiece + 2048 * u;
          const uint2 r0 = lds_read_tr16(p + tr[2 * dc]), r1 = lds_read_tr16(p + tr[2 * dc + 1]);
          r.x[u][dc] = sa_u32x4v{r0.x, r0.y, r1.x, r1.y};
        }
    }
    return r;
  }
  __device__ __forceinline__ void product(const Columns& c, int hf, const Weights<T>& W, sa_f32x16 (&to)[kD / 32]) const {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dc = 0; dc < 2; ++dc)
        to[2 * hf + dc] = mfma_chunk<T>(c.x[u][dc], sa_u32x4v{W.w[4 * u], W.w[4 * u + 1], W.w[4 * u + 2], W.w[4 * u + 3]},
                                        to[2 * hf + dc]);
  }
  __device__ __forceinline__ void product(const lds_u8* mat, const Weights<T>& W, sa_f32x16 (&to)[kD / 32]) const {
    if constexpr (kF32) {
#pragma unroll
      for (int dc = 0; dc < kD / 32; ++dc)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = *reinterpret_cast<const __attribute__((address_space(3))) float*>(mat + dc * kPiece + tr[e & 7] +
                                                                                            2048 * (e >> 3));
          to[dc] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, W.w[e], to[dc], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int hf = 0; hf < kD / 64; ++hf) product(columns(mat, hf), hf, W, to);
    }
  }
};

}  // namespace
