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

// ---- eight neighbouring elements of a row
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

// as they lie in memory: few registers between the request and the use.  load, store: on 16 bytes, fp32 on 32
template <typename T>
struct Raw8 {                                    // 16 bits
  static constexpr int kWords = 4;
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) unpack2<T>(w[j], f[2 * j], f[2 * j + 1]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack2<T>(f[2 * j], f[2 * j + 1]);
  }
  __device__ __forceinline__ void load1(const T* p, int e) {       // element e, the others of its word kept
    const uint32_t v = *reinterpret_cast<const uint16_t*>(p + e);
    w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | v << 16 : (w[e >> 1] & 0xffff0000u) | v;
  }
  __device__ __forceinline__ void store1(T* p, int e) const { *reinterpret_cast<uint16_t*>(p + e) = (uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1]); }
};
template <>
struct Raw8<float> {
  static constexpr int kWords = 8;
  uint32_t w[8];
  __device__ __forceinline__ void load(const float* p) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
  }
  // whole 32-byte sectors: two stores of 16 bytes, 32 apart from lane to lane, each write half of every sector (expand to fp32 272 -> 198 us
  // for 475,136 x 512)
  __device__ __forceinline__ void store(float* p) const {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7])
                 : "memory");
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 0;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(f[j]);
  }
  __device__ __forceinline__ void load1(const float* p, int e) { w[e] = *reinterpret_cast<const uint32_t*>(p + e); }
  __device__ __forceinline__ void store1(float* p, int e) const { *reinterpret_cast<uint32_t*>(p + e) = w[e]; }
};

// eight numbers as four pairs: two fp32 operations per instruction
struct Eight {
  uint64_t p[4];
  template <typename T>
  __device__ __forceinline__ static Eight of(const Raw8<T>& r) {
    float f[8];
    r.get(f);
    return of(f);
  }
  __device__ __forceinline__ static Eight of(const float (&f)[8]) {
    Eight e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.p[i] = f2_make(f[2 * i], f[2 * i + 1]);
    return e;
  }
  __device__ __forceinline__ static Eight all(float v) {
    Eight e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.p[i] = f2_make(v, v);
    return e;
  }
  __device__ __forceinline__ void split(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f2_split(p[i], f[2 * i], f[2 * i + 1]);
  }
  __device__ __forceinline__ float sum() const {
    float a, b;
    f2_split(f2_add(f2_add(p[0], p[1]), f2_add(p[2], p[3])), a, b);
    return a + b;
  }
};
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Where a matrix's bytes begin and end: pieces that do not start on 16 bytes are read by the aligned 16 bytes around them, inside these
struct Span {
  const uint8_t* lo;
  const uint8_t* hi;
};
template <typename T>
__host__ __device__ __forceinline__ Span span_of(const T* p, int64_t rows, int64_t d, int64_t ld) {
  return Span{reinterpret_cast<const uint8_t*>(p), reinterpret_cast<const uint8_t*>(p + (rows - 1) * ld + d)};
}

// N 32-bit words from byte `by` (0 .. 15, a multiple of the element's size) of the words c
template <int N, bool HALVES, int M>
__device__ __forceinline__ void take_words(uint32_t (&c)[M], int by, uint32_t* out) {
  static_assert(M >= N + 4, "");
  const int k = by >> 2;
#pragma unroll
  for (int j = 0; j + 1 < M; ++j) c[j] = k & 1 ? c[j + 1] : c[j];
#pragma unroll
  for (int j = 0; j + 2 < M; ++j) c[j] = k & 2 ? c[j + 2] : c[j];
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = HALVES ? __funnelshift_r(c[j], c[j + 1], (by & 2) * 8) : c[j];
}
// A piece anywhere in memory, of which `n` elements exist (the others read as zero)
template <typename T>
__device__ __forceinline__ void load_any(Raw8<T>& r, const T* p, int n, const Span& s) {
  constexpr int W = Raw8<T>::kWords;
  const int by = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  const uint8_t* from = reinterpret_cast<const uint8_t*>(p) - by;
  if (n >= 8 && by == 0 && W == 4) {
    r.load(p);
  } else if (n >= 8 && by == 0) {                  // fp32, on 16 bytes but maybe not on 32
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(from + j * 4);
      r.w[j] = v.x; r.w[j + 1] = v.y; r.w[j + 2] = v.z; r.w[j + 3] = v.w;
    }
  } else if (from >= s.lo && from + W * 4 + 16 <= s.hi) {
    uint32_t c[W + 4];
#pragma unroll
    for (int j = 0; j < W + 4; j += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(from + j * 4);
      c[j] = v.x; c[j + 1] = v.y; c[j + 2] = v.z; c[j + 3] = v.w;
    }
    take_words<W, W == 4>(c, by, r.w);
    if (n < 8) {                                   // what follows the row
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int left = W == 8 ? 2 * (n - j) : n - 2 * j;       // halves of word j that belong to it
        r.w[j] = left >= 2 ? r.w[j] : left == 1 ? r.w[j] & 0xffffu : 0u;
      }
    }
  } else {
    r.zero();
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) r.load1(p, e);
  }
}
// The same the other way.  The aligned 16 bytes that two neighbouring pieces share are written by the later one: `prev` holds the last
// 16 bytes of the piece ahead where that is whole and in this call (`ahead`); `behind`: the next one is whole and takes this one's end.
template <typename T>
__device__ __forceinline__ void store_any(const Raw8<T>& r, T* p, int n, const uint32_t (&prev)[4], bool ahead, bool behind) {
  constexpr int W = Raw8<T>::kWords, SIZE = (int)sizeof(T);
  const int by = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  if (n >= 8 && by == 0) {
    if constexpr (W == 4) {
      r.store(p);
    } else {
      reinterpret_cast<uint4*>(p)[0] = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
      reinterpret_cast<uint4*>(p)[1] = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
    }
    return;
  }
  int head = 0, tail = 8;                          // elements below head and from tail on go one by one
  if (n >= 8) {
    uint32_t c[W + 4], o[W];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = prev[j];
#pragma unroll
    for (int j = 0; j < W; ++j) c[4 + j] = r.w[j];
    take_words<W, W == 4>(c, 16 - by, o);
    uint8_t* to = reinterpret_cast<uint8_t*>(p) - by;
    if (ahead) *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
    else head = (16 - by) / SIZE;
    if constexpr (W == 8) *reinterpret_cast<uint4*>(to + 16) = make_uint4(o[4], o[5], o[6], o[7]);
    if (!behind) tail = 8 - by / SIZE;
  } else {
    head = n;
  }
  if (head > 0 || tail < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < head || e >= tail) r.store1(p, e);
  }
}

// eight codes
struct Codes {
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
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// largest magnitude (its bits; NaN above all) of the block that four lanes hold
__device__ __forceinline__ uint32_t block_max_bits(const float (&f)[8]) {
  float m = max_abs(max_abs(max_abs(f[0], f[1], f[2]), f[3], f[4]), max_abs(f[5], f[6], f[7]), 0.f);
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  return __float_as_uint(m) & 0x7fffffffu;
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
template <typename T, int KIND>
__device__ __forceinline__ uint32_t block_exp(uint32_t bits, float (&f)[8], float& inv) {
  using K = KindOf<KIND>;
  constexpr uint32_t kPast = (uint32_t)(top_binade<T>() + 128) << 23;                // 2^(top + 1); fp32: infinity
  uint32_t e = (bits + K::kCarry) >> 23;
  if (bits + K::kCarry >= kPast) {
    if (bits >= 0x7f800000u) {
      inv = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
      return 255;
    }
    constexpr float kMost = K::kTop * (top_binade<T>() == 15 ? 32768.f : 1.7014118346046923e38f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fminf(fmaxf(f[i], -kMost), kMost);
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
__device__ __forceinline__ void encode(const float (&f)[8], float inv, Codes& c) {
  c.v.x = encode4<KIND>(f[0], f[1], f[2], f[3], inv);
  c.v.y = encode4<KIND>(f[4], f[5], f[6], f[7], inv);
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
__device__ __forceinline__ void decode(const Codes& c, float (&f)[8]) {
  decode4<KIND>(c.v.x, f[0], f[1], f[2], f[3]);
  decode4<KIND>(c.v.y, f[4], f[5], f[6], f[7]);
}
// 2^(E - 127); E = 0: 0, E = 255: infinity
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e << 23); }

}  // namespace p8
}  // namespace bsrl
