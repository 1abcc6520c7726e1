// Rows in 8 bits: the two code formats and the helpers their kernels share (rows8.hip, gemm_i8.hip, act8_wgrad.hip).  gfx950 only.
//
//   row codes (the operands of the int8 product): one fp32 scale a row, s = max(fl32(max|x| / 127), 2^-126), code = the multiple of s nearest to x
//     (quotient x / s of the real numbers, ties to even).  A row that holds a NaN or an infinity has s = NaN and codes 0: whatever is computed from
//     it is NaN, an overflow is not turned into a number.
//   group codes (checkpoints): columns in groups of 64 that share a scale 2^e, e the smallest with max|x| <= 127 2^e, stored as the byte e + 127; a
//     group that holds a NaN or an infinity has the byte 255 and codes 0, and reads back as NaN.  The power of two costs up to one bit of the step
//     against max / 127 and buys two things: x 2^-e is exact, so no division decides a code, and code * 2^e has 7 significant bits, so it IS a number of
//     the 16-bit operand type -- a matrix product reads a checkpoint without rounding it a second time.
#pragma once
#include "common.h"

#define ROW_SCALE_PLAIN 0x1p96f          // (scaled_sum)
#define ACT8_GROUP 64
#define ACT8_BAD 255u
#define ACT8_EMAX 249u          // 2^122, the step of numbers above 127 * 2^121: their codes stop at 63, the largest that stands for a finite fp32 number
// smallest stored exponent: 2^-126 keeps every step a normal fp32 / bf16 number; IEEE half has none below 2^-24 (its own smallest subnormal), so the
// half build stops there -- an activation that came in that type has no finer bits
#if CLIMB_H16_F16
#define ACT8_EMIN (127 - 24)
#else
#define ACT8_EMIN 1
#endif

// biased exponent byte for the largest |x| of a group, given as fp32 bits without the sign (integer order = order of magnitude, NaN above inf above all
// numbers, so one integer maximum carries "holds a NaN").  max = 1.f 2^k: 127 = 1.984375 * 2^6, so e = k - 6 while 1.f <= 1.984375, else k - 5.
__device__ __forceinline__ unsigned act8_exp(unsigned mx) {
  if (mx >= 0x7f800000u) return ACT8_BAD;
  const int e = (int)(mx >> 23) - 6 + ((mx & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return (unsigned)(e < ACT8_EMIN ? ACT8_EMIN : e);
}
__device__ __forceinline__ float act8_step(unsigned e) { return __uint_as_float(e == ACT8_BAD ? 0x7fc00000u : e << 23); }      // 2^(e - 127); NaN
__device__ __forceinline__ float act8_inv(unsigned e) { return e == ACT8_BAD ? 0.f : __uint_as_float((254u - e) << 23); }
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// four codes in a word: x * inv (exact) + 1.5 * 2^23 rounds to the nearest integer, ties to even, in ONE fma and leaves it as the low byte in two's complement
__device__ __forceinline__ unsigned act8_pack4(float a, float b, float c, float d, unsigned e) {
  const float inv = act8_inv(e), magic = 12582912.f;
  if (e == ACT8_EMAX) {          // (64 steps of 2^122 would be 2^128, which reads back as an infinity)
    const float top = 63.f * 0x1p122f;
    a = fminf(fmaxf(a, -top), top); b = fminf(fmaxf(b, -top), top); c = fminf(fmaxf(c, -top), top); d = fminf(fmaxf(d, -top), top);
  }
  const unsigned ua = __float_as_uint(fmaf(a, inv, magic)), ub = __float_as_uint(fmaf(b, inv, magic));
  const unsigned uc = __float_as_uint(fmaf(c, inv, magic)), ud = __float_as_uint(fmaf(d, inv, magic));
  const unsigned r = __builtin_amdgcn_perm(ub, ua, 0x0c0c0400u) | __builtin_amdgcn_perm(ud, uc, 0x04000c0cu);
  return e == ACT8_BAD ? 0u : r;
}
// ... and back: byte ^ 128 is code + 128 in 0 .. 255, put in the low byte of 2^23 and taken off again (one byte permute and one subtraction at full rate, where a
// conversion is slower), then one exact product
__device__ __forceinline__ float4 act8_unpack4(unsigned w, float step) {
  const unsigned u = w ^ 0x80808080u;
  const float off = 8388736.f;          // 2^23 + 128
  return make_float4((__uint_as_float(__builtin_amdgcn_perm(0x4b000000u, u, 0x07060500u)) - off) * step, (__uint_as_float(__builtin_amdgcn_perm(0x4b000000u, u, 0x07060501u)) - off) * step,
                     (__uint_as_float(__builtin_amdgcn_perm(0x4b000000u, u, 0x07060502u)) - off) * step, (__uint_as_float(__builtin_amdgcn_perm(0x4b000000u, u, 0x07060503u)) - off) * step);
}

// ... as numbers of type T, of a group with exponent byte e.  A number of IEEE half above 65024 is kept as 64 steps of 2^10 = 65536, one step beyond the type's largest:
// where the half build reads that in 16 bits (a load, an MFMA operand, a recomputed activation) it is the largest again and no infinity
template <typename T>
__device__ __forceinline__ float4 act8_values4(unsigned w, unsigned e, float step) {
  float4 v = act8_unpack4(w, step);
#if CLIMB_H16_F16
  if (sizeof(T) == 2 && e == 127u + 10u) {
    auto top = [](float x) { return fabsf(x) == 65536.f ? copysignf(65504.f, x) : x; };
    v = make_float4(top(v.x), top(v.y), top(v.z), top(v.w));
  }
#endif
  return v;
}

// Phi(-|x|) = exp(-x^2 / 2) R(1 / (1 + p |x|)), R a polynomial without constant term fitted to erfcx(|x| / sqrt 2) / 2 on [0, 14] for the smallest largest
// RELATIVE error (weighted least squares, own fit): the tail keeps its digits, where 1 + erf would cancel them.  DEG 6: 8.3e-6 (results that are stored
// in 16 bits: a 470th of their half step), DEG 8: 1.5e-7 (fp32 results).  e2 returns exp(-x^2 / 2).
template <int DEG>
__device__ __forceinline__ float phi_lower(float x, float& e2) {
  const float z = fabsf(x);
  float r, t;
  if constexpr (DEG == 6) {
    t = __builtin_amdgcn_rcpf(fmaf(0.30f, z, 1.0f));
    r = fmaf(fmaf(fmaf(fmaf(fmaf(-0.07709959f, t, 0.21604484f), t, -0.01695827f), t, 0.1442025f), t, 0.11374025f), t, 0.1200744f);
  } else {
    t = __builtin_amdgcn_rcpf(fmaf(0.30f, z, 1.0f));
    r = fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(0.03567617f, t, -0.15720912f), t, 0.20636429f), t, -0.05369389f), t, 0.1285672f), t, 0.09991176f), t, 0.12075424f), t,
             0.11962928f);
  }
  e2 = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170368f);
  return r * t * e2;
}
template <typename T> struct GeluDeg { static constexpr int v = 6; };
template <> struct GeluDeg<float> { static constexpr int v = 8; };
// gelu(x) = x Phi(x): x >= 0: x - x q, x < 0: x q, q = Phi(-|x|)  =  max(x, 0) - |x| q.  (q and exp(-x^2 / 2) are 0 beyond |x| = 14.4: the factor is held
// at 64 there, so that an infinity gives its limit and not inf * 0)
template <typename T> __device__ __forceinline__ float gelu_phi(float x);
template <> __device__ __forceinline__ float gelu_phi<float>(float x) {
  float e2;
  const float q = phi_lower<8>(x, e2);
  return fmaf(-fminf(fabsf(x), 64.f), q, fmaxf(x, 0.f));
}
// For results stored in 16 bits: log2 Phi(-z) is close to a parabola, so one polynomial of degree 8 (own fit, as above) and ONE exponential give q: 11 full-rate
// operations and a transcendental, against 13 and two.  bfloat16 holds x q down to z = 13.2 and its half step is 2^-9 of a number at least, so the fit spans
// [0, 13.2] and may err more where q is small: relative error 1.8e-5 below 2, 8e-5 below 3, 3.8e-4 beyond; z stays at 14.5, where q underflows to the limit 0.
// IEEE half ends at 2^-25 (z = 5.6) with a finer step: fitted on [0, 10] to 2.6e-5, z stays at 10.  minimum / maximum: the NaN of a NaN argument goes through.
#if CLIMB_H16_F16
#define GELU16_END 10.f
#define GELU16_C {-1.00002384f, -1.15098619f, -0.458911031f, -0.0537272729f, 0.00850201212f, -0.000961354177f, 7.17434377e-05f, -3.12999009e-06f, 6.00354042e-08f}
#else
#define GELU16_END 14.5f
#define GELU16_C {-1.0000207f, -1.1508853f, -0.4593939f, -0.053093407f, 0.00815379f, -0.00086898665f, 5.9202197e-05f, -2.2890285e-06f, 3.7937127e-08f}
#endif
template <> __device__ __forceinline__ float gelu_phi<bf16_t>(float x) {
  constexpr float C[9] = GELU16_C;
  const float z = __builtin_elementwise_minimum(__builtin_fabsf(x), GELU16_END);
  float p = C[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) p = fmaf(p, z, C[i]);
  return fmaf(-z, __builtin_amdgcn_exp2f(p), __builtin_elementwise_maximum(x, 0.f));
}
// ... and gelu'(x) = Phi(x) + x exp(-x^2 / 2) / sqrt(2 pi)
template <int DEG>
__device__ __forceinline__ float gelu_phi_pair(float x, float& d) {
  float e2;
  const float q = phi_lower<DEG>(x, e2);
  const float z = fminf(fabsf(x), 64.f);
  d = fmaf(copysignf(z, x) * 0.39894228040143267794f, e2, x < 0.f ? q : 1.0f - q);
  return fmaf(-z, q, fmaxf(x, 0.f));
}

// Columns c .. c + N - 1 of a row of C (N = 4 or 8), zeros past its end.  MODE (row_mode): 1 whole rows of aligned pieces, C % N == 0; 0 any address and
// C >= N: the hardware reads unaligned words, and hipcc makes wide loads of the copy; 2 shorter rows.  The load itself is UNCONDITIONAL -- a piece at or past the end is
// read as the row's last N columns and shifted down -- because a load under a condition is waited for inside it: the pieces of a row would come one
// latency after the other.
template <int MODE, int N, typename T>
__device__ __forceinline__ void row_ld(const T* __restrict__ row, int c, int C, float (&v)[N]) {
  if constexpr (MODE == 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < C ? Act<T>::ld(row + c + i) : 0.f;
    return;
  }
  const int sh = max(c - (C - N), 0);
  const T* p = row + (sh ? C - N : c);
  if constexpr (MODE == 1) {
    if constexpr (N == 8 && sizeof(T) == 2) {
      const uint4 r = *reinterpret_cast<const uint4*>(p);
      v[0] = h16lo_to_f32(r.x); v[1] = h16hi_to_f32(r.x); v[2] = h16lo_to_f32(r.y); v[3] = h16hi_to_f32(r.y);
      v[4] = h16lo_to_f32(r.z); v[5] = h16hi_to_f32(r.z); v[6] = h16lo_to_f32(r.w); v[7] = h16hi_to_f32(r.w);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 r = ld4(p + i);
        v[i] = r.x; v[i + 1] = r.y; v[i + 2] = r.z; v[i + 3] = r.w;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sh ? 0.f : v[i];
  } else {
    T r[N];
    __builtin_memcpy(r, p, sizeof(r));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Act<T>::ld(r + i);
#pragma unroll
    for (int b = 1; b < N; b *= 2)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (sh & b) ? (i + b < N ? v[i + b] : 0.f) : v[i];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sh >= N ? 0.f : v[i];
  }
}
template <int MODE, int N, typename T>
__device__ __forceinline__ void row_st(T* __restrict__ p, int left, const float (&v)[N]) {
  if constexpr (MODE == 1) {
    if (left > 0) {
      if constexpr (N == 8 && sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
      } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) st4(p + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
      }
    }
  } else {
    if (left >= N) {
      T r[N];
#pragma unroll
      for (int i = 0; i < N; ++i) Act<T>::st(r + i, v[i]);
      __builtin_memcpy(p, r, sizeof(r));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) Act<T>::st(p + i, v[i]);
    }
  }
}
static inline int row_mode(bool aligned, int C, int N) { return C < N ? 2 : (aligned && C % N == 0 ? 1 : 0); }

// Reductions over W = 8, 16 or 64 neighbouring lanes without a trip through LDS: quad permutes, mirrors of 8 and 16 lanes (DPP), and the row / half swaps of
// gfx950 for 32 and 64.  Every lane ends with the result; the order of a sum is fixed.
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true); }
template <int W, typename F>
__device__ __forceinline__ unsigned lanes_reduce(unsigned x, F f) {
  x = f(x, dpp<0xB1>(x));          // quad_perm [1, 0, 3, 2]
  x = f(x, dpp<0x4E>(x));          // quad_perm [2, 3, 0, 1]
  x = f(x, dpp<0x141>(x));         // mirror within 8 lanes
  if constexpr (W >= 16) x = f(x, dpp<0x140>(x));          // mirror within 16 lanes
  if constexpr (W == 64) {
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f(r[0], r[1]);
    auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = f(h[0], h[1]);
  }
  return x;
}
// largest absolute value (as bits)
template <int W> __device__ __forceinline__ unsigned lanes_umax(unsigned m) {
  return lanes_reduce<W>(m, [](unsigned a, unsigned b) { return a > b ? a : b; });
}
__device__ __forceinline__ float lanes_sum(float v) {
  return __uint_as_float(lanes_reduce<64>(__float_as_uint(v), [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// True-quotient rounding.  x * (1 / s) is rounded to the nearest integer k by adding 1.5 * 2^23 in the same fma (k in the low bits), which may miss next to a
// half; the remainder r = x - k s is exact in one fma and settles it: k moves towards r's sign if 2 |r| > s, or 2 |r| = s and k is odd.  The sign and zero of
// 2 |r| - s are those of its bits as an integer (an exact zero is +0), so "bits + (k & 1) > 0" is both conditions at once.
__device__ __forceinline__ unsigned rowq(float x, float s, float rs) {
  const float magic = 12582912.f, u = fmaf(x, rs, magic), r = fmaf(magic - u, s, x), a = fmaf(2.f, fabsf(r), -s);
  const unsigned k = __float_as_uint(u);
  const int away = (__float_as_int(r) >> 31) | 1;
  return k + ((int)(__float_as_uint(a) + (k & 1u)) > 0 ? away : 0);
}
__device__ __forceinline__ float row_scale(unsigned mx) {
  return mx >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(mx) / 127.f, 1.1754943508222875e-38f);
}
// sum s t + b for an int32 sum and two row scales (both at least 2^-126, or NaN): s t itself may leave fp32's range where the result does not, so the sum takes the
// scales one after the other -- it is 0 or at least 1 in magnitude, so the first product keeps all its digits, and below 2^31, so it is finite for s <= 2^96.  Beyond
// that t goes first: if that product overflows, so does the result.  PLAIN: the caller knows that s <= 2^96 (or NaN); the same bits.
template <bool PLAIN = false>
__device__ __forceinline__ float scaled_sum(int sum, float s, float t, float b) {
  const bool far = !PLAIN && s > ROW_SCALE_PLAIN;
  return fmaf((float)sum * (far ? t : s), far ? s : t, b);
}
// Four codes.  |x| / s <= 127, so x * rs is within 127 * 2^-24 < 2^-17 of the quotient, and its distance from the nearest integer is off by less than 2^-25 more: only where
// that distance comes within 2^-16 of a half can the exact quotient round to the other side, and only a wave that holds such a one (0.8 % of the calls on random
// numbers) takes the exact steps.  Row codes of 12288 x 3072 in 16 bits 20 us, 22 with the exact steps for all.
__device__ __forceinline__ unsigned rowq4(const float (&v)[4], float s, float rs, bool bad) {
  const float magic = 12582912.f;
  unsigned k[4];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float u = fmaf(v[i], rs, magic);
    k[i] = __float_as_uint(u);
    far = fmaxf(far, fabsf(fmaf(v[i], rs, magic - u)));
  }
  if (__any(far > 0.5f - 0x1p-16f)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = rowq(v[i], s, rs);
  }
  const unsigned w = __builtin_amdgcn_perm(k[1], k[0], 0x0c0c0400u) | __builtin_amdgcn_perm(k[3], k[2], 0x04000c0cu);
  return bad ? 0u : w;
}
