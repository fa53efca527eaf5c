// Elementwise operators around activations kept in 8 bits (pack8.cuh): pack, expand, exact GELU forward (which keeps its input)
// and backward (which reads it).
//
// Pure streams: 16-bit elements cost 2 bytes read and 1 1/32 written (pack), the same the other way round (expand), 5 1/32 (GELU
// forward: x, y, codes; backward: gy, codes, gx).  The rows' codes are dense with a pitch of whole blocks, so a work item's
// place among the codes is its place among all items; only the rows of 16- or 32-bit elements have a pitch, and where those are
// dense too (and the width a multiple of 32) all rows are taken as one.
//
// Eight neighbouring elements per thread, four threads to a block, whose largest magnitude travels by two shuffles; several such pieces of a
// thread are requested before the first is used.  Rows that 16 bytes do not divide (odd widths or pitches, unaligned first elements) are
// read by the aligned 16 bytes around a piece and shifted into place, and written the same way, with the end of the neighbouring lane's
// piece: 40.9 M bf16 elements in rows of 1,363, one element per thread 166 us, 75 us so.
#include "kernels.cuh"
#include "pack8.cuh"

namespace bsrl {
namespace {
using namespace p8;

constexpr int kThreads = 256;
enum Op { kPack, kExpand, kGelu, kGeluBwd };

struct ElemArgs {
  const void* in;        // x; gy (GELU backward)
  void* out;             // y; gx; the expanded rows
  uint8_t* codes;
  uint8_t* exps;
  int64_t rows, d;       // rows = 1: d may be the elements of all rows
  int64_t ld_in, ld_out;
  int64_t pieces;        // pieces of eight elements, padding included
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// log2 of Phi(-a) for two magnitudes at a time, and its power: the fits of common.cuh.  Results that are rounded to fp16 take the short
// one, whose Phi(-a) is off by 9e-8 at most; bf16, whose range is fp32's, and fp32 the long one.  Its Phi(-a) is off by 6e-7 of itself at 2, 5e-6
// at 4, 4e-5 at 6, 3e-4 at 8, 1e-3 at 10, 9e-3 at 12.9 (more than half a step of bf16 from 10 on), and zero past 12.95, where it leaves fp32's normal numbers.
template <typename T>
__device__ __forceinline__ void tails(const float (&a)[8], float (&p)[8]) {
  constexpr bool SHORT = top_binade<T>() == 15;
  constexpr int N = SHORT ? 9 : 13;
  auto c = [](int i) { return SHORT ? kGeluQ[i < 9 ? i : 0] : kGeluQ32[i]; };
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint64_t aa = f2_make(a[j], a[j + 1]);
    uint64_t q = f2_make(c(N - 1), c(N - 1));
#pragma unroll
    for (int i = N - 2; i >= 0; --i) q = f2_fma(q, aa, f2_make(c(i), c(i)));
    f2_split(q, p[j], p[j + 1]);
    p[j] = gelu_ex2(p[j]);
    p[j + 1] = gelu_ex2(p[j + 1]);
  }
}
constexpr float kFar = 1e18f;      // past any finite tail; keeps infinity times zero out
// x Phi(x) = max(x, 0) - |x| Phi(-|x|)
template <typename T>
__device__ __forceinline__ void gelu_values(const float (&x)[8], float (&y)[8]) {
  float a[8], p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = min_nan(fabsf(x[j]), kFar);
  tails<T>(a, p);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = fmaf(-a[j], p[j], fmaxf(x[j], 0.f));
}
// the slope Phi(x) + x phi(x) = t for x < 0, 1 - t else, with t = Phi(-|x|) - |x| phi(|x|).  In the tail |x| phi(|x|) is x^2 times the other, and
// t is off by 2e-6 of itself at -6, 1.2e-5 at -10, 5e-5 at -12.9.  Its zero, x = -0.752, is a difference of near numbers: 1e-7 absolute there.
template <typename T>
__device__ __forceinline__ void gelu_slopes(const float (&x)[8], float (&s)[8]) {
  float a[8], p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = min_nan(fabsf(x[j]), kFar);
  tails<T>(a, p);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // phi(a) = 2^(log2(1 / sqrt(2 pi)) - a^2 log2(e) / 2)
    const float phi = gelu_ex2(fmaf(a[j] * a[j], -0.72134752044448170368f, -1.32574806473616302f));
    const float t = fmaf(-a[j], phi, p[j]);
    s[j] = x[j] < 0.f ? t : 1.f - t;
  }
}

// How the rows lie: all as one dense row; rows that 16 bytes divide; any
enum Rows { kFlat, kAligned, kAny };
template <typename T>
constexpr int unroll_of(int mode) { return sizeof(T) == 4 || mode == kAny ? 2 : 4; }
template <int OP, typename T, int KIND, int MODE>
__global__ void __launch_bounds__(kThreads) elem8_kernel(ElemArgs p) {
  constexpr int U = unroll_of<T>(MODE);
  constexpr bool ALIGNED = MODE != kAny;
  constexpr bool READS_CODES = OP == kExpand || OP == kGeluBwd;
  const int64_t per_row = pitch_of(p.d) / 8;
  const Span span_in = OP != kExpand && !ALIGNED ? span_of(static_cast<const T*>(p.in), p.rows, p.d, p.ld_in) : Span{};
  pdl_begin();
  for (int64_t tile = blockIdx.x; tile * (kThreads * U) < p.pieces; tile += gridDim.x) {
    const int64_t first = tile * (kThreads * U) + threadIdx.x;
    Raw8<T> in[U];
    Codes codes[U];
    uint32_t exps[U];
    int64_t out_at[U];
    int live[U], piece[U];               // elements of the row that the piece holds; its place in the row
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = first + u * kThreads;
      int64_t row = 0, col = i * 8;
      piece[u] = 1;
      if (MODE != kFlat && p.rows > 1) {
        row = div_index(i, (int)per_row, &piece[u]);
        col = (int64_t)piece[u] * 8;
      }
      if (MODE == kFlat) live[u] = i < p.pieces ? 8 : 0;
      else live[u] = i >= p.pieces || col >= p.d ? 0 : p.d - col < 8 ? (int)(p.d - col) : 8;
      out_at[u] = row * p.ld_out + col;
      if (OP != kExpand) {
        const T* from = static_cast<const T*>(p.in) + row * p.ld_in + col;
        if (!live[u]) in[u].zero();
        else if (ALIGNED) in[u].load(from);
        else load_any(in[u], from, live[u], span_in);
      }
      if (READS_CODES) {
        codes[u].zero();
        exps[u] = 0;
        if (live[u]) {
          codes[u].load(p.codes + i * 8);
          exps[u] = p.exps[i * 8 / kBlock];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = first + u * kThreads;
      float x[8], r[8];
      if (READS_CODES) {
        decode<KIND>(codes[u], x);
        const float s = scale_of(exps[u]);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= s;
      } else {
        in[u].get(x);
      }
      if (OP == kExpand) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = x[j];
      } else if (OP == kGelu) {
        gelu_values<T>(x, r);
      } else if (OP == kGeluBwd) {
        float g[8];
        in[u].get(g);
        gelu_slopes<T>(x, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] *= g[j];
      }
      if (OP != kPack) {
        Raw8<T> o;
        o.set(r);
        T* to = static_cast<T*>(p.out) + out_at[u];
        if (ALIGNED) {
          if (live[u]) o.store(to);
        } else {
          uint32_t prev[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) prev[j] = __shfl_up_sync(0xffffffffu, o.w[Raw8<T>::kWords - 4 + j], 1);
          const int lane = threadIdx.x & 31, next_live = __shfl_down_sync(0xffffffffu, live[u], 1), next_piece = __shfl_down_sync(0xffffffffu, piece[u], 1);
          if (live[u]) store_any(o, to, live[u], prev, lane > 0 && piece[u] > 0, lane < 31 && next_piece > 0 && next_live == 8);
        }
      }
      if (!READS_CODES) {
        float inv;
        const uint32_t e = block_exp<T, KIND>(block_max_bits(x), x, inv);
        Codes c;
        encode<KIND>(x, inv, c);
        if (i < p.pieces) {
          c.store(p.codes + i * 8);
          if ((i & 3) == 0) p.exps[i / 4] = (uint8_t)e;
        }
      }
    }
  }
}

template <int OP, typename T, int KIND, int MODE>
void launch(const ElemArgs& p, cudaStream_t stream) {
  constexpr int U = unroll_of<T>(MODE);
  const int64_t tiles = (p.pieces + kThreads * U - 1) / (kThreads * U), cap = (int64_t)sm_count() * 32;
  launch_kernel(elem8_kernel<OP, T, KIND, MODE>, (unsigned)(tiles < cap ? tiles : cap), kThreads, 0, stream, p);
}
template <int OP, typename T, int KIND>
void pick(const ElemArgs& p, int mode, cudaStream_t stream) {
  mode == kFlat ? launch<OP, T, KIND, kFlat>(p, stream) : mode == kAligned ? launch<OP, T, KIND, kAligned>(p, stream) : launch<OP, T, KIND, kAny>(p, stream);
}
template <int OP, typename T>
void pick(const ElemArgs& p, int kind, int mode, cudaStream_t stream) {
  kind == kInt8 ? pick<OP, T, kInt8>(p, mode, stream) : pick<OP, T, kE4m3>(p, mode, stream);
}
template <int OP>
int run(const void* in, int64_t ld_in, void* out, int64_t ld_out, int dtype, int64_t rows, int64_t d, int kind, uint8_t* codes,
        uint8_t* exps, cudaStream_t stream, const char* name) {
  const int size = dtype == BSRL_F32 ? 4 : 2;
  if (d % kBlock == 0 && (!in || ld_in == d) && (!out || ld_out == d)) {        // dense: one long row
    d *= rows;
    rows = 1;
    ld_in = ld_out = d;
  }
  const int unit = 8 * size;                       // bytes of a piece: 16, fp32 32
  auto on_units = [&](const void* base, int64_t ld) { return !base || (reinterpret_cast<uintptr_t>(base) % unit == 0 && (rows == 1 || (ld * size) % unit == 0)); };
  const bool aligned = d % 8 == 0 && on_units(in, ld_in) && on_units(out, ld_out);
  const int mode = !aligned ? kAny : rows == 1 && d % kBlock == 0 ? kFlat : kAligned;
  ElemArgs p{in, out, codes, exps, rows, d, ld_in, ld_out, rows * (pitch_of(d) / 8)};
  if (dtype == BSRL_F32) pick<OP, float>(p, kind, mode, stream);
  else if (dtype == BSRL_F16) pick<OP, __half>(p, kind, mode, stream);
  else pick<OP, __nv_bfloat16>(p, kind, mode, stream);
  BSRL_LAUNCH_OK(name);
  return BSRL_OK;
}
}  // namespace

int pack8(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t d, int kind, uint8_t* codes, uint8_t* exps, cudaStream_t stream) {
  return run<kPack>(x, ldx, nullptr, 0, dtype, rows, d, kind, codes, exps, stream, "pack8");
}
int expand8(const uint8_t* codes, const uint8_t* exps, int kind, int64_t rows, int64_t d, void* out, int dtype, int64_t ldo, cudaStream_t stream) {
  return run<kExpand>(nullptr, 0, out, ldo, dtype, rows, d, kind, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(exps), stream, "expand8");
}
int gelu8(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t d, void* y, int64_t ldy, int kind, uint8_t* codes, uint8_t* exps,
          cudaStream_t stream) {
  return run<kGelu>(x, ldx, y, ldy, dtype, rows, d, kind, codes, exps, stream, "gelu8");
}
int gelu8_bwd(const void* gy, int dtype, int64_t ldgy, const uint8_t* codes, const uint8_t* exps, int kind, int64_t rows, int64_t d, void* gx,
              int64_t ldgx, cudaStream_t stream) {
  return run<kGeluBwd>(gy, ldgy, gx, ldgx, dtype, rows, d, kind, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(exps), stream, "gelu8_bwd");
}

}  // namespace bsrl
