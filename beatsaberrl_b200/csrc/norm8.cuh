// LayerNorm whose input is kept in 8 bits (pack8.cuh), forward and backward; instantiated per type in norm8_*.cu.
//
//   z = x + residual, rounded to the rows' type;  mean, rstd of z in fp32, two passes over rows held in registers
//   y = (z - mean) rstd gamma + beta;  kept: z in 8 bits, mean, rstd
//   h = (z8 - mean) rstd;  gh = gy gamma;  gx = rstd (gh - mean(gh) - h mean(gh h)) + g_residual
//   g_gamma = sum over rows of gy h,  g_beta = sum over rows of gy
//
// Streams: per element of fp32 rows with fp16 outputs 7 1/32 bytes forward and 7 1/32 backward.  A row belongs to a team of lanes -- 4, 8, 16 or 32
// of a warp up to 1024 columns, a whole block above -- which holds it in registers between its one read and its one write, eight
// neighbouring elements per lane and step (16-byte accesses).  Rows that 16 bytes do not divide go one element per lane.
//
// The parameter gradients are summed in one order: every lane adds the rows it meets into registers, a block's teams add up through
// shared memory one after the other, blocks write partial rows and a second kernel adds those in order.  No atomics, so a call gives the same
// bits every time.
#pragma once
#include <initializer_list>
#include <type_traits>

#include "kernels.cuh"
#include "pack8.cuh"

namespace bsrl {
namespace norm8 {
using namespace p8;

template <typename T, typename TY>
struct FwdArgs {
  const T* x;
  const T* res;
  T* z;
  TY* y;
  const float *gamma, *beta;
  uint8_t *codes, *exps;
  float *mean, *rstd;
  int64_t rows, ldx, ldr, ldz, ldy;
  int d, kind;
  float eps;
};
template <typename T, typename TY>
struct BwdArgs {
  const TY* gy;
  const T* gres;
  T* gx;
  const float* gamma;
  const uint8_t *codes, *exps;
  const float *mean, *rstd;
  float *g_gamma, *g_beta;       // of the only block; else
  float* parts;                  // (blocks, 2, d)
  int64_t rows, ldgy, ldgr, ldgx;
  int d, kind;
};

// Sums over a team's lanes.  TPR > 0: TPR lanes of a warp.  TPR = 0 (-1): a block of up to 512 (1024) threads; `turn` alternates between two sets of shared slots, so
// that one barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ void team_sum(float& a, float& b, float2 (*slots)[32], int& turn) {
  constexpr int W = TPR > 0 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (TPR <= 0) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slots[turn][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const float2 s = lane < warps ? slots[turn][lane] : make_float2(0.f, 0.f);
    a = s.x;
    b = s.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    turn ^= 1;
  }
}

template <int V>
__device__ __forceinline__ void load_f32(const float* p, float (&v)[V]) {
  Raw<float, V> r;
  r.load(p);
  r.get(v);
}

constexpr int kThreads = 256;
constexpr int block_threads(int tpr) { return tpr > 0 ? kThreads : tpr == 0 ? 512 : 1024; }
// blocks of kThreads per SM that the kernels are built for, by what a lane holds
constexpr int fwd_resident(int held) { return held <= 8 ? 5 : held <= 16 ? 3 : 2; }
constexpr int bwd_resident(int held) { return held <= 8 ? 4 : held <= 16 ? 2 : 1; }

// R: rows a team has in flight.  NV: steps of V elements that a lane takes of a row.
template <typename T, typename TY, int V, int TPR, int NV, int R>
__global__ void __launch_bounds__(block_threads(TPR), TPR > 0 ? fwd_resident(NV * V * R) : 1) norm8_fwd_kernel(FwdArgs<T, TY> p) {
  __shared__ float2 slots[2][32];
  int turn = 0;
  constexpr int W = TPR > 0 ? TPR : 32;
  const int lane = threadIdx.x & 31;
  const int at = TPR > 0 ? lane % W : threadIdx.x, stride = TPR > 0 ? W : blockDim.x;       // this lane's pieces of a row: at + i stride
  constexpr int TEAMS = TPR > 0 ? 32 / W : 1;
  const int team = TPR > 0 ? lane / W : 0;
  const int d = p.d, pitch = (int)pitch_of(d);
  const int64_t first = TPR > 0 ? ((int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * (TEAMS * R) : blockIdx.x;
  const int64_t step = TPR > 0 ? (int64_t)gridDim.x * (blockDim.x >> 5) * (TEAMS * R) : gridDim.x;
  pdl_begin();
  float g1[V], b1[V];
  if (NV == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) g1[j] = b1[j] = 0.f;
    if (at * V < d) {
      load_f32<V>(p.gamma + at * V, g1);
      if (p.beta) load_f32<V>(p.beta + at * V, b1);
    }
  }
  for (int64_t base = first; base < p.rows; base += step) {
    Raw<T, V> raw[R][NV], rres[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * TEAMS + team;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * V;
        if (row < p.rows && col < d) {
          raw[r][i].load(p.x + row * p.ldx + col);
          if (p.res) rres[r][i].load(p.res + row * p.ldr + col);
        } else {
          raw[r][i].zero();
          rres[r][i].zero();
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * TEAMS + team;
      const bool live = row < p.rows;
      float v[NV][V];
      float s = 0.f, q = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * V;
        raw[r][i].get(v[i]);
        if (p.res) {
          float w[V];
          rres[r][i].get(w);
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] += w[j];
          raw[r][i].set(v[i]);
          raw[r][i].get(v[i]);                     // as the stream has it: rounded to its type
          if (live && col < d && p.z) raw[r][i].store(p.z + row * p.ldz + col);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[i][j];
      }
      float none = 0.f;
      team_sum<TPR>(s, none, slots, turn);
      const float mean = s / d;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((at + i * stride) * V < d) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float c = v[i][j] - mean;
            q = fmaf(c, c, q);
          }
        }
      team_sum<TPR>(q, none, slots, turn);
      const float rstd = 1.f / sqrtf(q / d + p.eps);
      if (at == 0 && live) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * V;
        if (live && col < d) {
          float g[V], b[V], o[V];
          if (NV == 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = g1[j], b[j] = b1[j];
          } else {
            load_f32<V>(p.gamma + col, g);
            if (p.beta) load_f32<V>(p.beta + col, b);
            else
#pragma unroll
              for (int j = 0; j < V; ++j) b[j] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] = fmaf((v[i][j] - mean) * rstd, g[j], b[j]);
          Raw<TY, V> out;
          out.set(o);
          out.store(p.y + row * p.ldy + col);
        }
        float inv;
        const uint32_t bits = block_max_bits<V>(v[i]);
        Codes<V> c;
        uint32_t e;
        if (p.kind == kInt8) {
          e = block_exp<T, kInt8, V>(bits, v[i], inv);
          encode<kInt8>(v[i], inv, c);
        } else {
          e = block_exp<T, kE4m3, V>(bits, v[i], inv);
          encode<kE4m3>(v[i], inv, c);
        }
        if (live && col < pitch) {
          c.store(p.codes + row * pitch + col);
          if (col % kBlock == 0) p.exps[row * (pitch / kBlock) + col / kBlock] = (uint8_t)e;
        }
      }
    }
  }
}

template <typename T, typename TY, int V, int TPR, int NV, int R>
__global__ void __launch_bounds__(block_threads(TPR), TPR > 0 ? bwd_resident(NV * V * R) : 1) norm8_bwd_kernel(BwdArgs<T, TY> p) {
  __shared__ float2 slots[2][32];
  extern __shared__ float s_sums[];                  // [2][d], teams of lanes only
  int turn = 0;
  constexpr int W = TPR > 0 ? TPR : 32;
  const int lane = threadIdx.x & 31;
  const int at = TPR > 0 ? lane % W : threadIdx.x, stride = TPR > 0 ? W : blockDim.x;
  constexpr int TEAMS = TPR > 0 ? 32 / W : 1;
  const int team = TPR > 0 ? lane / W : 0;
  const int d = p.d, pitch = (int)pitch_of(d), blocks = pitch / kBlock;
  const int64_t first = TPR > 0 ? ((int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * (TEAMS * R) : blockIdx.x;
  const int64_t step = TPR > 0 ? (int64_t)gridDim.x * (blockDim.x >> 5) * (TEAMS * R) : gridDim.x;
  const float inv_d = 1.f / d;
  pdl_begin();
  float g1[V];
  if (NV == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) g1[j] = 0.f;
    if (at * V < d) load_f32<V>(p.gamma + at * V, g1);
  }
  float acc_g[NV][V], acc_b[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) acc_g[i][j] = acc_b[i][j] = 0.f;
  for (int64_t base = first; base < p.rows; base += step) {
    Raw<TY, V> rgy[R][NV];
    Raw<T, V> rres[R][NV];
    Codes<V> codes[R][NV];
    uint32_t exps[R][NV];
    float mean[R], rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * TEAMS + team;
      const bool live = row < p.rows;
      mean[r] = live ? p.mean[row] : 0.f;
      rstd[r] = live ? p.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * V;
        if (live && col < d) {
          rgy[r][i].load(p.gy + row * p.ldgy + col);
          codes[r][i].load(p.codes + row * pitch + col);
          exps[r][i] = p.exps[row * blocks + col / kBlock];
          if (p.gres) rres[r][i].load(p.gres + row * p.ldgr + col);
        } else {
          rgy[r][i].zero();
          codes[r][i].zero();
          exps[r][i] = 0;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * TEAMS + team;
      const bool live = row < p.rows;
      // h of one step: the codes' scale and the row's rstd in one factor
      const float shift = -mean[r] * rstd[r];
      auto hidden = [&](int i, float (&h)[V]) {
        if (p.kind == kInt8) decode<kInt8>(codes[r][i], h);
        else decode<kE4m3>(codes[r][i], h);
        const float s = scale_of(exps[r][i]);
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = fmaf(h[j] * s, rstd[r], shift);
      };
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * V;
        if (live && col < d) {
          float h[V], g[V], gm[V];
          hidden(i, h);
          rgy[r][i].get(g);
          if (NV == 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) gm[j] = g1[j];
          } else {
            load_f32<V>(p.gamma + col, gm);
          }
#pragma unroll
          for (int j = 0; j < V; ++j) {
            acc_g[i][j] = fmaf(g[j], h[j], acc_g[i][j]);
            acc_b[i][j] += g[j];
            const float gh = g[j] * gm[j];
            s1 += gh;
            s2 = fmaf(gh, h[j], s2);
          }
        }
      }
      team_sum<TPR>(s1, s2, slots, turn);
      s1 *= inv_d;
      s2 *= inv_d;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * V;
        if (live && col < d) {
          float h[V], g[V], gm[V], o[V];
          hidden(i, h);
          rgy[r][i].get(g);
          if (NV == 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) gm[j] = g1[j];
          } else {
            load_f32<V>(p.gamma + col, gm);
          }
          if (p.gres) rres[r][i].get(o);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float gx = rstd[r] * (fmaf(g[j], gm[j], -s1) - h[j] * s2);
            o[j] = p.gres ? o[j] + gx : gx;
          }
          Raw<T, V> out;
          out.set(o);
          out.store(p.gx + row * p.ldgx + col);
        }
      }
    }
  }
  pdl_trigger();
  float* to_g = p.parts ? p.parts + (int64_t)blockIdx.x * 2 * d : p.g_gamma;
  float* to_b = p.parts ? to_g + d : p.g_beta;
  if constexpr (TPR <= 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (at + i * stride) * V;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (col < d) {
          if (to_g) to_g[col + j] = acc_g[i][j];
          if (to_b) to_b[col + j] = acc_b[i][j];
        }
    }
  } else {
#pragma unroll
    for (int o = W; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          acc_g[i][j] += __shfl_xor_sync(0xffffffffu, acc_g[i][j], o);
          acc_b[i][j] += __shfl_xor_sync(0xffffffffu, acc_b[i][j], o);
        }
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int w = 0; w < warps; ++w) {
      if (warp == w && team == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (at + i * stride) * V;
          if (col < d) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              s_sums[col + j] = w ? s_sums[col + j] + acc_g[i][j] : acc_g[i][j];
              s_sums[d + col + j] = w ? s_sums[d + col + j] + acc_b[i][j] : acc_b[i][j];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
      if (to_g) to_g[c] = s_sums[c];
      if (to_b) to_b[c] = s_sums[d + c];
    }
  }
}

// How rows of d elements are shared out: lanes per team (TPR), steps per lane, rows in flight
struct Shape {
  int v, tpr, nv, r;
  int threads;             // per block
  int rows_per_block;
  int resident;            // blocks per SM
};
constexpr int kMaxWidth = 16384;
inline Shape shape_of(int d, bool vec, bool bwd) {
  const int pitch = (int)pitch_of(d);
  Shape s;
  s.v = vec ? 8 : 1;
  s.r = 1;
  if (vec) {
    const int pieces = pitch / 8;
    if (pieces <= 128) {
      s.tpr = pieces <= 4 ? 4 : pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32;
      s.nv = pieces <= 32 ? 1 : pieces <= 64 ? 2 : 4;
      s.r = s.nv == 1 ? 2 : 1;
    } else {
      s.nv = 2;
      s.tpr = pieces <= 1024 ? 0 : -1;
    }
  } else if (pitch <= 1024) {
    s.tpr = 32;
    s.nv = pitch <= 256 ? 8 : 32;
  } else {
    s.nv = 16;
    s.tpr = pitch <= 8192 ? 0 : -1;
  }
  if (s.tpr > 0) {
    s.threads = kThreads;
    s.rows_per_block = kThreads / s.tpr * s.r;
    s.resident = bwd ? bwd_resident(s.nv * s.v * s.r) : fwd_resident(s.nv * s.v * s.r);
  } else {
    s.threads = (int)round_up((pitch / s.v + s.nv - 1) / s.nv, 32);
    s.rows_per_block = 1;
    s.resident = (bwd ? 1024 : 2048) / s.threads;
    if (s.resident < 1) s.resident = 1;
  }
  return s;
}
inline int blocks_of(const Shape& s, int64_t rows, int waves) {
  const int64_t need = (rows + s.rows_per_block - 1) / s.rows_per_block, cap = (int64_t)sm_count() * s.resident * waves;
  return (int)(need < cap ? need : cap);
}

template <typename T, typename TY>
int fwd(const FwdArgs<T, TY>& p, bool vec, cudaStream_t stream);
template <typename T, typename TY>
int bwd(const BwdArgs<T, TY>& p, bool vec, cudaStream_t stream);      // p.parts: blocks_of(shape_of(d, vec, true), rows, 1) rows of 2 d floats if that is above 1

// calls fn(V, TPR, NV, R as integral constants) for the shape
template <typename Fn>
void with_shape(const Shape& s, Fn&& fn) {
#define BSRL_SHAPE(V_, TPR_, NV_, R_) \
  if (s.v == V_ && s.tpr == TPR_ && s.nv == NV_) return fn(std::integral_constant<int, V_>{}, std::integral_constant<int, TPR_>{}, std::integral_constant<int, NV_>{}, std::integral_constant<int, R_>{})
  BSRL_SHAPE(8, 4, 1, 2);
  BSRL_SHAPE(8, 8, 1, 2);
  BSRL_SHAPE(8, 16, 1, 2);
  BSRL_SHAPE(8, 32, 1, 2);
  BSRL_SHAPE(8, 32, 2, 1);
  BSRL_SHAPE(8, 32, 4, 1);
  BSRL_SHAPE(8, 0, 2, 1);
  BSRL_SHAPE(8, -1, 2, 1);
  BSRL_SHAPE(1, 32, 8, 1);
  BSRL_SHAPE(1, 32, 32, 1);
  BSRL_SHAPE(1, 0, 16, 1);
  BSRL_SHAPE(1, -1, 16, 1);
#undef BSRL_SHAPE
}
template <typename T, typename TY>
int launch_fwd(const FwdArgs<T, TY>& p, bool vec, cudaStream_t stream) {
  const Shape s = shape_of(p.d, vec, false);
  const int blocks = blocks_of(s, p.rows, 4);
  with_shape(s, [&](auto V, auto TPR, auto NV, auto R) { launch_kernel(norm8_fwd_kernel<T, TY, V(), TPR(), NV(), R()>, blocks, s.threads, 0, stream, p); });
  BSRL_LAUNCH_OK("norm8_fwd_kernel");
  return BSRL_OK;
}
template <typename T, typename TY>
int launch_bwd(const BwdArgs<T, TY>& p, bool vec, cudaStream_t stream) {
  const Shape s = shape_of(p.d, vec, true);
  const int blocks = blocks_of(s, p.rows, 1);
  const size_t smem = s.tpr > 0 ? 2 * p.d * sizeof(float) : 0;
  with_shape(s, [&](auto V, auto TPR, auto NV, auto R) { launch_kernel(norm8_bwd_kernel<T, TY, V(), TPR(), NV(), R()>, blocks, s.threads, smem, stream, p); });
  BSRL_LAUNCH_OK("norm8_bwd_kernel");
  return BSRL_OK;
}

}  // namespace norm8
}  // namespace bsrl
