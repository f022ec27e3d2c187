// Activations in 8 bits: 32 neighbouring columns of a row share a power of two (the layout of the open MXINT8 format: one
// exponent byte, e + 127, and signed bytes).
//
//   e     floor(log2 max|x|) of the group, in [-120, 127], one more where the largest value would round to 128 steps
//   code  x / 2^(e - 6), rounded to the nearest whole number (ties to even), in [-127, 127]: off by at most half a step
//   value code * 2^(e - 6).  Seven bits and a power of two: exact in bf16 and TF32, so that products on the tensor cores read the
//         values as they are, and scaling by powers of two makes every step above exact in fp32: no rounding but the one.
// A group that holds an infinity or a NaN has the byte 255, and all its values are NaN.
// Behind a ReLU codes are never negative, and the byte -128 is free: it stands for a positive value that rounds to zero.  The
// code says then whether the value was positive, which is what the ReLU's backward pass asks.
#pragma once
#include "values.cuh"

namespace tfk {

constexpr int kPackGroup = 32;

__device__ __forceinline__ float pack8_power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }  // e in [-126, 127]

// The group's exponent from the bits of its largest |value|; 128 for a group that is not finite.
__device__ __forceinline__ int pack8_exponent(unsigned top) {
  const int e = (int)(top >> 23) - 127;
  if (e == 128) return 128;
  if (e < -120) return -120;
  return min(127, e + ((top & 0x7fffffu) >= 0x7f0000u ? 1 : 0));
}
// A code in the low byte of the result, from x in steps of its group, at most 128 of them: adding 1.5 * 2^23 leaves the nearest whole
// number in the last bits, ties to even (a conversion instruction runs at a quarter of the rate).
template <bool RELU> __device__ __forceinline__ unsigned pack8_code(float steps) {
  if (!RELU) return __float_as_uint(steps + 12582912.f);
  return steps > 0.f && steps <= 0.5f ? 0x80u : __float_as_uint(fmaxf(steps, 0.f) + 12582912.f);
}
// A value in steps: exact but far below the group's largest, where a positive one (rounded up) does not become zero.
__device__ __forceinline__ float pack8_steps(float v, float power) { return __fmul_ru(v, power); }
__device__ __forceinline__ float unpack8_step(unsigned byte) {  // 2^(e - 6), NaN for 255
  return byte == 255 ? __int_as_float(0x7fc00000) : __uint_as_float((byte - 6) << 23);
}
__device__ __forceinline__ float unpack8_value(int code, float step) { return (float)(code == -128 ? 0 : code) * step; }
// Four codes at a time.  With c + 128 in a byte (128 where it was zero, which stands for the code zero), that byte behind 2^23 is the
// float 2^23 + 128 + c; one multiplication and addition leaves c steps, exactly.  The step times 2^23 must be a number: SMALL is for
// steps up to 2^96; larger ones take the subtraction first.
__device__ __forceinline__ unsigned unpack8_biased(unsigned w) {
  w ^= 0x80808080u;
  const unsigned any = (w & 0x7f7f7f7fu) + 0x7f7f7f7fu;  // top bit of a byte: one of the lower seven is set
  return w | (~(any | w) & 0x80808080u);
}
template <bool SMALL> __device__ __forceinline__ void unpack8_word(unsigned w, float step, float *v) {
  w = unpack8_biased(w);
  const float less = -8388736.f * step;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i));
    v[i] = SMALL ? fmaf(f, step, less) : (f - 8388736.f) * step;
  }
}
template <int N> __device__ __forceinline__ void unpack8_values(const Pack<signed char, N> &c, float step, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
    const unsigned *w = reinterpret_cast<const unsigned *>(&c);
    if (fabsf(step) <= 0x1p96f) {  // (a NaN is not)
#pragma unroll
      for (int i = 0; i < N; i += 4) unpack8_word<true>(w[i / 4], step, &v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) unpack8_word<false>(w[i / 4], step, &v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = unpack8_value(c.v[i], step);
  }
}

// A thread's N neighbouring values (N divides 32), the other lanes of the group holding the rest: codes in the low bytes, and the
// exponent.
template <int N, bool RELU> __device__ __forceinline__ int pack8_lanes(const float (&v)[N], unsigned (&code)[N]) {
  float m = 0.f;
  if constexpr (N == 1) m = RELU ? max3(m, v[0], v[0]) : max3_abs(m, v[0], v[0]);
  else {
#pragma unroll
    for (int i = 0; i < N; i += 2) m = RELU ? max3(m, v[i], v[i + 1]) : max3_abs(m, v[i], v[i + 1]);
  }
  unsigned top = __float_as_uint(m) & 0x7fffffffu;  // (a NaN is above the infinity)
#pragma unroll
  for (int k = kPackGroup / N / 2; k; k >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, k));
  const int e = pack8_exponent(top);
  if (e >= 127) {  // rare: the last power of two, where 128 steps stay 127, or a group that is not finite: its codes say what was positive
    const float power = e == 127 ? pack8_power(6 - e) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      code[i] = e == 127 ? pack8_code<RELU>(fminf(fmaxf(pack8_steps(v[i], power), -127.f), 127.f)) : RELU && v[i] > 0.f ? 0x80u : 0u;
  } else {
    const float power = pack8_power(6 - e);
#pragma unroll
    for (int i = 0; i < N; ++i) code[i] = pack8_code<RELU>(pack8_steps(v[i], power));
  }
  return e;
}
template <int N> __device__ __forceinline__ void store_codes(signed char *p, const unsigned (&code)[N]) {
  if constexpr (N % 4 == 0) {
    Pack<unsigned, N / 4> a;
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      a.v[i] = __byte_perm(__byte_perm(code[4 * i], code[4 * i + 1], 0x0040), __byte_perm(code[4 * i + 2], code[4 * i + 3], 0x0040), 0x5410);
    *reinterpret_cast<Pack<unsigned, N / 4> *>(p) = a;
  } else {
    Pack<unsigned char, N> a;
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = (unsigned char)code[i];
    *reinterpret_cast<Pack<unsigned char, N> *>(p) = a;
  }
}

}  // namespace tfk
