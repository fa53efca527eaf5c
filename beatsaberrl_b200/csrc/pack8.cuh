// Activations in 8 bits: blocks of 32 neighbouring values of a row share a power of two, 2^(E - 127), and hold one code each.
//
// int8: codes -127 .. 127.  e4m3: codes on the e4m3 grid with magnitude at most 240.  E is the least one with which the code of the
// block's largest magnitude, rounded to nearest, stays in that range; in the top binade of the values' own type E stays one lower
// and the codes clamp, so that what they stand for is finite in that type.  E = 0: a block of zeros (largest magnitude below
// 2^-120, e4m3 2^-119).  E = 255 with codes of zero: a block that held a value that is not finite; 0 x infinity makes all 32 NaN
// wherever they are read, without a test.
//
// The scale is a power of two so that every value has at most 8 significant bits: bf16 holds it exactly, fp16 where its range does, and
// 16-bit matrix operands made of codes lose nothing more.  With the largest magnitude itself as the scale int8's step would be between 1 and 1/2
// of this one.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace bsrl {
namespace p8 {

constexpr int kBlock = 32;
enum Kind { kInt8 = 0, kE4m3 = 1 };

__host__ __device__ __forceinline__ int64_t pitch_of(int64_t d) { return (d + kBlock - 1) / kBlock * kBlock; }

// ---- loads and stores of V neighbouring elements (V = 8: 16-byte aligned; V = 1: any)
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two 16-bit elements of a word <-> two floats
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b);
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// V elements as they lie in memory: few registers between the request and the use
template <typename T, int V>
struct Raw {
  T v[V];
  __device__ __forceinline__ void load(const T* p) { v[0] = *p; }
  __device__ __forceinline__ void zero() { v[0] = from_f32<T>(0.f); }
  __device__ __forceinline__ void get(float (&f)[V]) const { f[0] = to_f32(v[0]); }
  __device__ __forceinline__ void set(const float (&f)[V]) { v[0] = from_f32<T>(f[0]); }
  __device__ __forceinline__ void store(T* p) const { *p = v[0]; }
};
template <>
struct Raw<float, 8> {
  float4 v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = reinterpret_cast<const float4*>(p)[0];
    v[1] = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = v[0].x; f[1] = v[0].y; f[2] = v[0].z; f[3] = v[0].w;
    f[4] = v[1].x; f[5] = v[1].y; f[6] = v[1].z; f[7] = v[1].w;
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v[0] = make_float4(f[0], f[1], f[2], f[3]);
    v[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = v[0];
    reinterpret_cast<float4*>(p)[1] = v[1];
  }
};
template <typename T>
struct Raw16x8 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    unpack2<T>(v.x, f[0], f[1]);
    unpack2<T>(v.y, f[2], f[3]);
    unpack2<T>(v.z, f[4], f[5]);
    unpack2<T>(v.w, f[6], f[7]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
};
template <>
struct Raw<__half, 8> : Raw16x8<__half> {};
template <>
struct Raw<__nv_bfloat16, 8> : Raw16x8<__nv_bfloat16> {};

// V codes
template <int V>
struct Codes {
  uint8_t v;
  __device__ __forceinline__ void load(const uint8_t* p) { v = *p; }
  __device__ __forceinline__ void store(uint8_t* p) const { *p = v; }
  __device__ __forceinline__ void zero() { v = 0; }
};
template <>
struct Codes<8> {
  uint2 v;
  __device__ __forceinline__ void load(const uint8_t* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void store(uint8_t* p) const { *reinterpret_cast<uint2*>(p) = v; }
  __device__ __forceinline__ void zero() { v = make_uint2(0, 0); }
};

// ---- the shared exponent
__device__ __forceinline__ float max_nan(float a, float b) {      // NaN wins
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// largest magnitude (its bits; NaN above all) of the block whose values the V-wide lanes of a group hold
template <int V>
__device__ __forceinline__ uint32_t block_max_bits(const float (&f)[V]) {
  if constexpr (V == 1) {
    return __reduce_max_sync(0xffffffffu, __float_as_uint(f[0]) & 0x7fffffffu);
  } else {
    float m = fabsf(f[0]);
#pragma unroll
    for (int i = 1; i < V; ++i) m = max_nan(m, fabsf(f[i]));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
    return __float_as_uint(m) & 0x7fffffffu;
  }
}

// Per kind: log2 of the range's top binade, and what is added to the largest magnitude's bits so that a mantissa whose code would
// round past the range (127.5 / 64, 248 / 128: ties go to the even code, which lies past it) carries into the next exponent.
template <int KIND>
struct KindOf {
  static constexpr int kUp = KIND == kInt8 ? 6 : 7;
  static constexpr uint32_t kCarry = KIND == kInt8 ? 0x10000u : 0x80000u;
  static constexpr float kTop = KIND == kInt8 ? 127.f / 64.f : 240.f / 128.f;      // times 2^top binade: the largest value
};
// exponent of the type's top binade
template <typename T>
__device__ constexpr int top_binade() { return 127; }
template <>
__device__ constexpr int top_binade<__half>() { return 15; }

// E of a block, the factor that takes its values to codes, and -- in the top binade only, or where something is not finite -- the
// values themselves brought into the range.
template <typename T, int KIND, int V>
__device__ __forceinline__ uint32_t block_exp(uint32_t bits, float (&f)[V], float& inv) {
  using K = KindOf<KIND>;
  constexpr uint32_t kPast = (uint32_t)(top_binade<T>() + 128) << 23;                // 2^(top + 1); fp32: infinity
  uint32_t e = (bits + K::kCarry) >> 23;
  if (bits + K::kCarry >= kPast) {
    if (bits >= 0x7f800000u) {
      inv = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = 0.f;
      return 255;
    }
    constexpr float kMost = K::kTop * (top_binade<T>() == 15 ? 32768.f : 1.7014118346046923e38f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = fminf(fmaxf(f[i], -kMost), kMost);
    e = bits >> 23;
  }
  e = e > K::kUp ? e - K::kUp : 0;
  inv = e ? __uint_as_float((254u - e) << 23) : 0.f;
  return e;
}

// ---- codes
template <int KIND>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
  if constexpr (KIND == kInt8) {
    // 1.5 x 2^23 + t: the integer nearest to t in the low bits, ties to even
    const uint32_t u0 = __float_as_uint(fmaf(a, inv, 12582912.f)), u1 = __float_as_uint(fmaf(b, inv, 12582912.f));
    const uint32_t u2 = __float_as_uint(fmaf(c, inv, 12582912.f)), u3 = __float_as_uint(fmaf(d, inv, 12582912.f));
    return __byte_perm(__byte_perm(u0, u1, 0x0040), __byte_perm(u2, u3, 0x0040), 0x5410);
  } else {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a * inv), "f"(b * inv), "f"(c * inv), "f"(d * inv));
    return r;
  }
}
template <int KIND>
__device__ __forceinline__ void encode(const float (&f)[8], float inv, Codes<8>& c) {
  c.v.x = encode4<KIND>(f[0], f[1], f[2], f[3], inv);
  c.v.y = encode4<KIND>(f[4], f[5], f[6], f[7], inv);
}
template <int KIND>
__device__ __forceinline__ void encode(const float (&f)[1], float inv, Codes<1>& c) {
  c.v = (uint8_t)encode4<KIND>(f[0], 0.f, 0.f, 0.f, inv);
}

// codes as numbers, without the scale
template <int KIND>
__device__ __forceinline__ void decode4(uint32_t w, float& a, float& b, float& c, float& d) {
  if constexpr (KIND == kInt8) {
    w ^= 0x80808080u;                                   // code + 128, as the low byte of 2^23 + .
    a = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650)) - 8388736.f;
    b = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7651)) - 8388736.f;
    c = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7652)) - 8388736.f;
    d = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7653)) - 8388736.f;
  } else {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
    unpack2<__half>(lo, a, b);
    unpack2<__half>(hi, c, d);
  }
}
template <int KIND>
__device__ __forceinline__ void decode(const Codes<8>& c, float (&f)[8]) {
  decode4<KIND>(c.v.x, f[0], f[1], f[2], f[3]);
  decode4<KIND>(c.v.y, f[4], f[5], f[6], f[7]);
}
template <int KIND>
__device__ __forceinline__ void decode(const Codes<1>& c, float (&f)[1]) {
  float x, y, z;
  decode4<KIND>(c.v, f[0], x, y, z);
}
// 2^(E - 127); E = 0: 0, E = 255: infinity
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e << 23); }

}  // namespace p8
}  // namespace bsrl
