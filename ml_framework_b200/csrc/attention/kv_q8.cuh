// A paged cache in 8 bits: cache[num_blocks][2 (K, V)][block_size][Hkv][128] numbers of one byte, e4m3 or int8, and
// scale[num_blocks][2][Hkv] fp32; a value is its number times the scale of its block, side and head.
//
// Scales that the kernels write are powers of two, 2^-40 .. 2^40: the smallest under which the block's largest magnitude fits
// (448 for e4m3, 127 for int8). Dividing by one is exact, so that a number is rounded once, and a block whose scale grows
// while rows are appended to it is rounded to the coarser step without a second error of the division. A reader takes any
// positive scale, and a block that came with one keeps it until rows need a larger one.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace mlf {

constexpr int Q8_D = 128;
enum Q8Format { Q8_E4M3 = 0, Q8_INT8 = 1 };
constexpr int Q8_EXP_MAX = 40;

// The smallest power of two from 2^-40 to 2^40 under which magnitudes up to amax fit. amax = (1 + m / 2^23) 2^e by its bits;
// 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6 decide whether 2^(e - 8) (2^(e - 6)) is enough.
template <int FMT>
__device__ __forceinline__ float q8_scale_for(float amax) {
  const unsigned u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127;
  const unsigned m = u & 0x7fffffu;
  int x = FMT == Q8_E4M3 ? e - 8 + (m > 0x600000u ? 1 : 0) : e - 6 + (m > 0x7e0000u ? 1 : 0);
  x = max(-Q8_EXP_MAX, min(Q8_EXP_MAX, x));
  return __uint_as_float((unsigned)(x + 127) << 23);
}

// Numbers (already divided by their scale) rounded to 8 bits, the first one in the low byte. Magnitudes beyond the largest become the
// largest; a NaN stays one in e4m3 and becomes 0 in int8.
template <int FMT>
__device__ __forceinline__ unsigned q8_pack4(float a, float b, float c, float d) {
  if (FMT == Q8_E4M3)
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) | (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
  // conversion and packing saturate above, the comparison below (-128 is no number of the format)
  int x = __float2int_rn(a), y = __float2int_rn(b), z = __float2int_rn(c), w = __float2int_rn(d);
  x = max(x, -127); y = max(y, -127); z = max(z, -127); w = max(w, -127);
  unsigned hi, all;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(w), "r"(z));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(all) : "r"(y), "r"(x), "r"(hi));
  return all;
}

// Numbers in 8 bits under a scale that came with the block and is no power of two: times its inverse, which is rounded, a number half way
// between two steps came to the wrong one of them, and to different ones in an append and in a write.
__device__ __forceinline__ bool q8_power_of_two(float scale) { return (__float_as_uint(scale) & 0x7fffffu) == 0; }
template <int FMT>
__device__ __forceinline__ unsigned q8_divide4(float a, float b, float c, float d, float scale) {
  return q8_pack4<FMT>(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale));
}

// The four numbers of a word as two f16 pairs, (byte 0, byte 1) and (byte 2, byte 3): every one of both types is exact in f16.
// int8: the byte with its sign bit turned over, as the low mantissa bits of 1024 + x, less 1152.
template <int FMT>
__device__ __forceinline__ void q8_unpack4(unsigned w, unsigned& lo, unsigned& hi) {
  if (FMT == Q8_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const unsigned x = w ^ 0x80808080u;
    const unsigned a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));     // 1152
    const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&a), off), h = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const unsigned*>(&l);
    hi = *reinterpret_cast<const unsigned*>(&h);
  }
}
template <int FMT>
__device__ __forceinline__ float4 q8_floats(unsigned w) {
  unsigned lo, hi;
  q8_unpack4<FMT>(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_float4(a.x, a.y, b.x, b.y);
}
// Held numbers in units of a new scale: rounded again.
template <int FMT>
__device__ __forceinline__ unsigned q8_shrink4(unsigned w, float ratio) {
  const float4 f = q8_floats<FMT>(w);
  return q8_pack4<FMT>(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio);
}

}  // namespace mlf
