// Elementwise operators around activations kept in 8 bits (pack8.cuh): pack, expand, exact GELU forward (which keeps its input)
// and backward (which reads it).
//
// Pure streams: 16-bit elements cost 2 bytes read and 1 1/32 written (pack), the same the other way round (expand), 5 1/32 (GELU
// forward: x, y, codes; backward: gy, codes, gx).  The rows' codes are dense with a pitch of whole blocks, so a work item's
// place among the codes is its place among all items; only the rows of 16- or 32-bit elements have a pitch, and where those are
// dense too (and the width a multiple of 32) all rows are taken as one.
//
// Eight neighbouring elements per thread (16-byte accesses), four threads to a block, whose largest magnitude travels by two
// shuffles; kUnroll such pieces of a thread are requested before the first is used.  Rows that 16 bytes do not divide (odd widths or
// pitches, unaligned first elements) go one element per thread: a warp holds one block.
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
  int64_t pieces;        // pieces of V elements, padding included
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// log2 of Phi(-a) for two magnitudes at a time, and its power: the fits of common.cuh.  Results that are rounded to fp16 take the short
// one; bf16, whose range is fp32's, and fp32 the one that is exact in the tail too.
template <typename T, int V>
__device__ __forceinline__ void tails(const float (&a)[V], float (&p)[V]) {
  constexpr bool SHORT = top_binade<T>() == 15;
  constexpr int N = SHORT ? 9 : 13;
  auto c = [](int i) { return SHORT ? kGeluQ[i < 9 ? i : 0] : kGeluQ32[i]; };
  if constexpr (V == 1) {
    float q = c(N - 1);
#pragma unroll
    for (int i = N - 2; i >= 0; --i) q = fmaf(q, a[0], c(i));
    p[0] = gelu_ex2(q);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const uint64_t aa = f2_make(a[j], a[j + 1]);
      uint64_t q = f2_make(c(N - 1), c(N - 1));
#pragma unroll
      for (int i = N - 2; i >= 0; --i) q = f2_fma(q, aa, f2_make(c(i), c(i)));
      f2_split(q, p[j], p[j + 1]);
      p[j] = gelu_ex2(p[j]);
      p[j + 1] = gelu_ex2(p[j + 1]);
    }
  }
}
constexpr float kFar = 1e18f;      // past any finite tail; keeps infinity times zero out
// x Phi(x) = max(x, 0) - |x| Phi(-|x|)
template <typename T, int V>
__device__ __forceinline__ void gelu_values(const float (&x)[V], float (&y)[V]) {
  float a[V], p[V];
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = min_nan(fabsf(x[j]), kFar);
  tails<T, V>(a, p);
#pragma unroll
  for (int j = 0; j < V; ++j) y[j] = fmaf(-a[j], p[j], fmaxf(x[j], 0.f));
}
// the slope Phi(x) + x phi(x) = t for x < 0, 1 - t else, with t = Phi(-|x|) - |x| phi(|x|): no difference of near numbers
template <typename T, int V>
__device__ __forceinline__ void gelu_slopes(const float (&x)[V], float (&s)[V]) {
  float a[V], p[V];
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] = min_nan(fabsf(x[j]), kFar);
  tails<T, V>(a, p);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    // phi(a) = 2^(log2(1 / sqrt(2 pi)) - a^2 log2(e) / 2)
    const float phi = gelu_ex2(fmaf(a[j] * a[j], -0.72134752044448170368f, -1.32574806473616302f));
    const float t = fmaf(-a[j], phi, p[j]);
    s[j] = x[j] < 0.f ? t : 1.f - t;
  }
}

template <int OP, typename T, int KIND, int V>
__global__ void __launch_bounds__(kThreads) elem8_kernel(ElemArgs p) {
  constexpr int U = V == 8 ? (sizeof(T) == 4 ? 2 : 4) : 8;
  constexpr bool READS_CODES = OP == kExpand || OP == kGeluBwd;
  const int64_t per_row = pitch_of(p.d) / V;
  pdl_begin();
  for (int64_t tile = blockIdx.x; tile * (kThreads * U) < p.pieces; tile += gridDim.x) {
    const int64_t first = tile * (kThreads * U) + threadIdx.x;
    Raw<T, V> in[U];
    Codes<V> codes[U];
    uint32_t exps[U];
    int64_t out_at[U];
    bool live[U];                        // of the rows' own elements, not of the padding behind them
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = first + u * kThreads;
      int64_t row = 0, col = i * V;
      if (p.rows > 1) {
        int piece;
        row = div_index(i, (int)per_row, &piece);
        col = (int64_t)piece * V;
      }
      live[u] = i < p.pieces && col < p.d;
      out_at[u] = row * p.ld_out + col;
      if (OP != kExpand) {
        if (live[u]) in[u].load(static_cast<const T*>(p.in) + row * p.ld_in + col);
        else in[u].zero();
      }
      if (READS_CODES) {
        codes[u].zero();
        exps[u] = 0;
        if (live[u]) {
          codes[u].load(p.codes + i * V);
          exps[u] = p.exps[i * V / kBlock];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = first + u * kThreads;
      float x[V], r[V];
      if (READS_CODES) {
        decode<KIND>(codes[u], x);
        const float s = scale_of(exps[u]);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] *= s;
      } else {
        in[u].get(x);
      }
      if (OP == kExpand) {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = x[j];
      } else if (OP == kGelu) {
        gelu_values<T, V>(x, r);
      } else if (OP == kGeluBwd) {
        float g[V];
        in[u].get(g);
        gelu_slopes<T, V>(x, r);
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] *= g[j];
      }
      if (OP != kPack && live[u]) {
        Raw<T, V> o;
        o.set(r);
        o.store(static_cast<T*>(p.out) + out_at[u]);
      }
      if (!READS_CODES) {
        float inv;
        const uint32_t e = block_exp<T, KIND, V>(block_max_bits<V>(x), x, inv);
        Codes<V> c;
        encode<KIND>(x, inv, c);
        if (i < p.pieces) {
          c.store(p.codes + i * V);
          if ((i & (kBlock / V - 1)) == 0) p.exps[i * V / kBlock] = (uint8_t)e;
        }
      }
    }
  }
}

template <int OP, typename T, int KIND, int V>
void launch(const ElemArgs& p, cudaStream_t stream) {
  constexpr int U = V == 8 ? (sizeof(T) == 4 ? 2 : 4) : 8;
  const int64_t tiles = (p.pieces + kThreads * U - 1) / (kThreads * U), cap = (int64_t)sm_count() * 32;
  launch_kernel(elem8_kernel<OP, T, KIND, V>, (unsigned)(tiles < cap ? tiles : cap), kThreads, 0, stream, p);
}
template <int OP, typename T>
void pick(const ElemArgs& p, int kind, bool vec, cudaStream_t stream) {
  if (kind == kInt8) vec ? launch<OP, T, kInt8, 8>(p, stream) : launch<OP, T, kInt8, 1>(p, stream);
  else vec ? launch<OP, T, kE4m3, 8>(p, stream) : launch<OP, T, kE4m3, 1>(p, stream);
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
  auto by16 = [&](const void* base, int64_t ld) { return !base || (aligned16(base) && (rows == 1 || (ld * size) % 16 == 0)); };
  const bool vec = d % 8 == 0 && by16(in, ld_in) && by16(out, ld_out);
  ElemArgs p{in, out, codes, exps, rows, d, ld_in, ld_out, rows * (pitch_of(d) / (vec ? 8 : 1))};
  if (dtype == BSRL_F32) pick<OP, float>(p, kind, vec, stream);
  else if (dtype == BSRL_F16) pick<OP, __half>(p, kind, vec, stream);
  else pick<OP, __nv_bfloat16>(p, kind, vec, stream);
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
