// LayerNorm whose input is kept in 8 bits (pack8.cuh), forward and backward; instantiated per type in norm8_*.cu.
//
//   z = x + residual, rounded to the rows' type;  mean, rstd of z in fp32, two passes over rows held in registers
//   y = (z - mean) rstd gamma + beta;  kept: z in 8 bits, mean, rstd
//   h = (z8 - mean) rstd;  gh = gy gamma;  gx = rstd (gh - mean(gh) - h mean(gh h)) + g_residual
//   g_gamma = sum over rows of gy h,  g_beta = sum over rows of gy
//
// Streams: per element of fp32 rows with fp16 outputs 7 1/32 bytes forward and 7 1/32 backward.  A row belongs to a team of lanes -- 4, 8, 16 or 32
// of a warp up to 512 columns, a whole block above -- which holds it in registers between its one read and its one write, eight
// neighbouring elements per lane and step.  Rows that 16 bytes do not divide are read by the aligned 16 bytes around a lane's piece and shifted
// into place, and written the same way with the end of the neighbouring lane's piece.
// 475,136 fp32 rows of 256 with fp16 results: 140 us forward (94 % of the copy rate), 160 backward (83 %).  What bounds the backward is the
// instructions (220 per row and warp) and the 16 warps that its registers leave.  With twice the instructions (arithmetic one element at a
// time, IEEE divisions) both took over 200 us whatever was requested ahead, in registers or through a ring in shared memory.
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

// Sums of N numbers over a team's lanes.  TPR > 0: TPR lanes of a warp.  TPR = 0: the block; `turn` alternates between two sets of shared
// slots, so that one barrier per sum is enough.
// Among 32 lanes the first steps halve the numbers a lane goes on with (of two lanes one takes one half, one the other): as many shuffles less in
// every later step, and the same order as N separate trees (59,392 x 2,048: forward 191 -> 169 us, backward 189 -> 175).  Of fewer lanes the steps
// that are left do not make up for it (475,136 x 64 backward 54 -> 58).
template <int TPR, int N>
__device__ __forceinline__ void team_sum(float (&a)[N], float (*slots)[32][4], int& turn) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  if constexpr (TPR > 0 && TPR < 32) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
    return;
  }
  constexpr int L = 32 / N;                              // a number's lanes in the end
  const int lane = threadIdx.x & 31;
  float k = a[0];
  if constexpr (N == 4) {
    const bool up = lane & 16, up2 = lane & 8;
    const float k0 = (up ? a[2] : a[0]) + __shfl_xor_sync(0xffffffffu, up ? a[0] : a[2], 16);
    const float k1 = (up ? a[3] : a[1]) + __shfl_xor_sync(0xffffffffu, up ? a[1] : a[3], 16);
    k = (up2 ? k1 : k0) + __shfl_xor_sync(0xffffffffu, up2 ? k0 : k1, 8);
  } else if constexpr (N == 2) {
    const bool up = lane & 16;
    k = (up ? a[1] : a[0]) + __shfl_xor_sync(0xffffffffu, up ? a[0] : a[1], 16);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) k += __shfl_xor_sync(0xffffffffu, k, o);
  if constexpr (TPR == 0) {
    const int warps = blockDim.x >> 5, which = lane / L;
    if (lane % L == 0) slots[turn][threadIdx.x >> 5][which] = k;
    __syncthreads();
    k = 0.f;
#pragma unroll
    for (int w = 0; w < 16; w += L)                        // at most 16 warps
      if (w + lane % L < warps) k += slots[turn][w + lane % L][which];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) k += __shfl_xor_sync(0xffffffffu, k, o);
    turn ^= 1;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = N == 1 ? k : __shfl_sync(0xffffffffu, k, lane % L + i * L);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
template <bool ALIGNED, typename T>
__device__ __forceinline__ void load_piece(Raw8<T>& r, const T* p, int n, const Span& s) {
  if (ALIGNED) r.load(p);
  else load_any(r, p, n, s);
}
// eight of a parameter's d values
template <bool ALIGNED>
__device__ __forceinline__ Eight load_param(const float* p, int col, int d) {
  Raw8<float> r;
  load_piece<ALIGNED>(r, p + col, d - col, ALIGNED ? Span{} : span_of(p, 1, d, d));
  return Eight::of(r);
}
// Writes step i of a row.  `last`: the words of the step ahead, whose last lane's end lane 0 needs (a team of a warp's lanes; a block's warps
// write their edges element by element).  All lanes call it.
template <bool ALIGNED, int TPR, typename T>
__device__ __forceinline__ void store_piece(const Raw8<T>& r, T* row, int piece, int d, bool live, uint32_t (&last)[4]) {
  const int col = piece * 8;
  if (ALIGNED) {
    if (live && col < d) r.store(row + col);
    return;
  }
  constexpr int W = Raw8<T>::kWords, TEAM = TPR > 0 ? TPR : 32;
  const int lane = threadIdx.x & 31, in_team = lane % TEAM;
  uint32_t prev[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t mine = r.w[W - 4 + j];
    prev[j] = __shfl_sync(0xffffffffu, TPR > 0 && in_team == TEAM - 1 ? last[j] : mine, (lane - in_team) + (in_team + TEAM - 1) % TEAM);
    last[j] = mine;
  }
  const bool ahead = TPR > 0 ? piece > 0 : in_team > 0, behind = (TPR > 0 || in_team < TEAM - 1) && col + 16 <= d;
  if (live && col < d) store_any(r, row + col, d - col, prev, ahead, behind);
}

constexpr int kThreads = 256;                      // of blocks whose warps hold teams
// blocks of kThreads per SM: 128 registers each.  Three forward (80 registers, spills) 213 us where two are 176, of 475,136 rows of 256
constexpr int kResident = 2;
// Threads of blocks that hold a row, per SM, and blocks of kThreads: what registers are kept free for.  Unaligned rows run more warps than
// aligned ones and one row at a time: they wait for what follows from what a piece's place in memory is.  60,007 x 1,001 fp16 with a residual, 512 / 768
// threads: forward 240 / 201 us, backward 214 / 179; 100,003 x 509, two / three blocks: forward 197 / 170.  Aligned forward, 14,848 x 8,192 fp32, 512 / 1,024
// threads 191 / 162 us; its backward 231 / 245.  The unaligned backward above 4,096 columns, two steps per lane, pays for its 80 registers with about
// 450 to 510 bytes of spills; above 6,144 columns its one block would fit 128 (not measured).
constexpr int block_threads(int tpr, bool aligned, bool bwd) { return tpr > 0 ? kThreads : !aligned ? 768 : bwd ? 512 : 1024; }
constexpr int blocks_per_sm(int tpr, bool aligned, bool bwd) { return tpr == 0 ? 1 : aligned || bwd ? kResident : 3; }

// This thread's part of the rows.  TPR > 0: TPR lanes of a warp hold a row; TPR = 0: the block does.  A warp or block takes ROWS rows at a time.
template <int TPR, int R>
struct Place {
  static constexpr int TEAM = TPR > 0 ? TPR : 32, TEAMS = TPR > 0 ? 32 / TEAM : 1, ROWS = TEAMS * R;
  int at, stride, team;          // the lane's pieces of a row: at + i stride
  int64_t first, step;
  __device__ __forceinline__ Place() {
    const int lane = threadIdx.x & 31;
    at = TPR > 0 ? lane % TEAM : threadIdx.x;
    stride = TPR > 0 ? TEAM : blockDim.x;
    team = TPR > 0 ? lane / TEAM : 0;
    first = TPR > 0 ? ((int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * ROWS : (int64_t)blockIdx.x * ROWS;
    step = TPR > 0 ? (int64_t)gridDim.x * (blockDim.x >> 5) * ROWS : (int64_t)gridDim.x * ROWS;
  }
};

// R: rows a team works on together.  NV: steps of eight elements that a lane takes of a row.  RES: there is a residual.
template <typename T, typename TY, bool ALIGNED, bool RES, int TPR, int NV, int R>
__global__ void __launch_bounds__(block_threads(TPR, ALIGNED, false), blocks_per_sm(TPR, ALIGNED, false)) norm8_fwd_kernel(FwdArgs<T, TY> p) {
  __shared__ float slots[2][32][4];
  int turn = 0;
  const Place<TPR, R> pl;
  const int at = pl.at, stride = pl.stride, d = p.d, pitch = (int)pitch_of(d);
  const bool res = RES && (ALIGNED || p.res);      // the kernels of unaligned rows have one form
  const Span span_x = ALIGNED ? Span{} : span_of(p.x, p.rows, d, p.ldx), span_r = ALIGNED || !res ? Span{} : span_of(p.res, p.rows, d, p.ldr);
  const float inv_d = 1.f / d;
  pdl_begin();
  Eight g1 = Eight::all(0.f), b1 = g1;
  if (NV == 1 && at * 8 < d) {
    g1 = load_param<ALIGNED>(p.gamma, at * 8, d);
    if (p.beta) b1 = load_param<ALIGNED>(p.beta, at * 8, d);
  }
  for (int64_t base = pl.first; base < p.rows; base += pl.step) {
    Raw8<T> x[R][NV], r2[R][NV];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * pl.TEAMS + pl.team;
      live[r] = row < p.rows;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        x[r][i].zero();
        if (RES) r2[r][i].zero();
        if (live[r] && col < d) {
          load_piece<ALIGNED>(x[r][i], p.x + row * p.ldx + col, d - col, span_x);
          if (res) load_piece<ALIGNED>(r2[r][i], p.res + row * p.ldr + col, d - col, span_r);
        }
      }
    }
    // the next rows, into L2: no registers, and half of the latency (176 -> 141 us, backward 218 -> 167 of 475,136 rows of 256)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + pl.step + r * pl.TEAMS + pl.team;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        if (row < p.rows && col < d) {
          prefetch_l2(p.x + row * p.ldx + col);
          if (res) prefetch_l2(p.res + row * p.ldr + col);
        }
      }
    }
    float sum[R], var[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * pl.TEAMS + pl.team;
      sum[r] = var[r] = 0.f;
      uint32_t last[4] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Eight v = Eight::of(x[r][i]);
        if (RES) {
          const Eight w = Eight::of(r2[r][i]);
          float f[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) v.p[j] = f2_add(v.p[j], w.p[j]);
          v.split(f);
          x[r][i].set(f);
          v = Eight::of(x[r][i]);                  // as the stream has it: rounded to its type
          if (res) store_piece<ALIGNED, TPR>(x[r][i], p.z + row * p.ldz, at + i * stride, d, live[r], last);
        }
        sum[r] += v.sum();
      }
    }
    team_sum<TPR>(sum, slots, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[r] *= inv_d;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        Eight v = Eight::of(x[r][i]), q = Eight::all(0.f);
        const Eight m = Eight::all(-sum[r]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v.p[j] = f2_add(v.p[j], m.p[j]);
        if (!ALIGNED && col + 8 > d) {             // elements that the row does not have
          float f[8];
          v.split(f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = col + j < d ? f[j] : 0.f;
          v = Eight::of(f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) q.p[j] = f2_mul(v.p[j], v.p[j]);
        if (col < d) var[r] += q.sum();
      }
    }
    team_sum<TPR>(var, slots, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * pl.TEAMS + pl.team;
      const float rstd = rsqrtf(fmaf(var[r], inv_d, p.eps));
      if (at == 0 && live[r]) {
        p.mean[row] = sum[r];
        p.rstd[row] = rstd;
      }
      uint32_t last[4] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        Eight v = Eight::of(x[r][i]);
        Raw8<TY> out;
        out.zero();
        if (live[r] && col < d) {
          Eight g = g1, b = b1;
          if (NV > 1) {
            g = load_param<ALIGNED>(p.gamma, col, d);
            if (p.beta) b = load_param<ALIGNED>(p.beta, col, d);
          }
          const Eight m = Eight::all(-sum[r]), s = Eight::all(rstd);
          Eight o;
#pragma unroll
          for (int j = 0; j < 4; ++j) o.p[j] = f2_fma(f2_mul(f2_add(v.p[j], m.p[j]), s.p[j]), g.p[j], b.p[j]);
          float f[8];
          o.split(f);
          out.set(f);
        }
        store_piece<ALIGNED, TPR>(out, p.y + row * p.ldy, at + i * stride, d, live[r], last);
        float f[8], inv;
        v.split(f);
        const uint32_t bits = block_max_bits(f);
        Codes c;
        uint32_t e;
        if (p.kind == kInt8) {
          e = block_exp<T, kInt8>(bits, f, inv);
          encode<kInt8>(f, inv, c);
        } else {
          e = block_exp<T, kE4m3>(bits, f, inv);
          encode<kE4m3>(f, inv, c);
        }
        if (live[r] && col < pitch) {
          c.store(p.codes + row * pitch + col);
          if (col % kBlock == 0) p.exps[row * (pitch / kBlock) + col / kBlock] = (uint8_t)e;
        }
      }
    }
  }
}

template <typename T, typename TY, bool ALIGNED, bool RES, int TPR, int NV, int R>
__global__ void __launch_bounds__(block_threads(TPR, ALIGNED, true), blocks_per_sm(TPR, ALIGNED, true)) norm8_bwd_kernel(BwdArgs<T, TY> p) {
  __shared__ float slots[2][32][4];
  extern __shared__ float s_sums[];                  // [2][d], teams of lanes only
  int turn = 0;
  const Place<TPR, R> pl;
  const int at = pl.at, stride = pl.stride, d = p.d, pitch = (int)pitch_of(d), blocks = pitch / kBlock;
  const bool res = RES && (ALIGNED || p.gres);
  const Span span_g = ALIGNED ? Span{} : span_of(p.gy, p.rows, d, p.ldgy), span_r = ALIGNED || !res ? Span{} : span_of(p.gres, p.rows, d, p.ldgr);
  const float inv_d = 1.f / d;
  pdl_begin();
  Eight g1 = Eight::all(0.f);
  if (NV == 1 && at * 8 < d) g1 = load_param<ALIGNED>(p.gamma, at * 8, d);
  // steps ahead that rows are requested: with a residual two (fp16 rows of 256 208 -> 197 us; without one 159 -> 179)
  constexpr int kAhead = ALIGNED && RES ? 2 : 1;
  Eight acc_g[NV], acc_b[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc_g[i] = acc_b[i] = Eight::all(0.f);
  for (int64_t base = pl.first; base < p.rows; base += pl.step) {
    Raw8<TY> gy[R][NV];
    Raw8<T> r2[R][NV];
    Codes codes[R][NV];
    uint32_t exps[R][NV];
    float mean[R], rstd[R];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * pl.TEAMS + pl.team;
      live[r] = row < p.rows;
      mean[r] = rstd[r] = 0.f;
      if (live[r]) {
        mean[r] = p.mean[row];
        rstd[r] = p.rstd[row];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        gy[r][i].zero();
        codes[r][i].zero();
        exps[r][i] = 0;
        if (RES) r2[r][i].zero();
        if (live[r] && col < d) {
          load_piece<ALIGNED>(gy[r][i], p.gy + row * p.ldgy + col, d - col, span_g);
          codes[r][i].load(p.codes + row * pitch + col);
          exps[r][i] = p.exps[row * blocks + col / kBlock];
          if (res) load_piece<ALIGNED>(r2[r][i], p.gres + row * p.ldgr + col, d - col, span_r);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {                      // the next rows, into L2
      const int64_t row = base + kAhead * pl.step + r * pl.TEAMS + pl.team;
      if (at == 0 && row < p.rows) {
        prefetch_l2(p.mean + row);
        prefetch_l2(p.rstd + row);
        prefetch_l2(p.exps + row * blocks);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        if (row < p.rows && col < d) {
          prefetch_l2(p.gy + row * p.ldgy + col);
          prefetch_l2(p.codes + row * pitch + col);
          if (res) prefetch_l2(p.gres + row * p.ldgr + col);
        }
      }
    }
    // rows one after the other up to their sums; what is needed again is made again from what was loaded
    float sums[R][2];
    auto hidden = [&](int r, int i) {
      float f[8];
      if (p.kind == kInt8) decode<kInt8>(codes[r][i], f);
      else decode<kE4m3>(codes[r][i], f);
      Eight h = Eight::of(f);
      // the scale and rstd in one factor: one rounding of their product, a power of two times rstd is exact
      const Eight s = Eight::all(scale_of(exps[r][i]) * rstd[r]), m = Eight::all(-mean[r] * rstd[r]);
#pragma unroll
      for (int j = 0; j < 4; ++j) h.p[j] = f2_fma(h.p[j], s.p[j], m.p[j]);
      return h;
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Eight s1 = Eight::all(0.f), s2 = s1;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        if (live[r] && col < d) {
          const Eight h = hidden(r, i), g = Eight::of(gy[r][i]), gm = NV == 1 ? g1 : load_param<ALIGNED>(p.gamma, col, d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc_g[i].p[j] = f2_fma(g.p[j], h.p[j], acc_g[i].p[j]);
            acc_b[i].p[j] = f2_add(acc_b[i].p[j], g.p[j]);
            const uint64_t gh = f2_mul(g.p[j], gm.p[j]);
            s1.p[j] = f2_add(s1.p[j], gh);
            s2.p[j] = f2_fma(gh, h.p[j], s2.p[j]);
          }
        }
      }
      sums[r][0] = s1.sum();
      sums[r][1] = s2.sum();
    }
    team_sum<TPR>(reinterpret_cast<float(&)[2 * R]>(sums), slots, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * pl.TEAMS + pl.team;
      // gx = gh rstd - (rstd mean(gh) + h rstd mean(gh h))
      const Eight k0 = Eight::all(rstd[r]), k1 = Eight::all(-sums[r][0] * inv_d * rstd[r]), k2 = Eight::all(-sums[r][1] * inv_d * rstd[r]);
      uint32_t last[4] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (at + i * stride) * 8;
        Raw8<T> out;
        out.zero();
        if (live[r] && col < d) {
          const Eight h = hidden(r, i), g = Eight::of(gy[r][i]), gm = NV == 1 ? g1 : load_param<ALIGNED>(p.gamma, col, d);
          Eight o;
#pragma unroll
          for (int j = 0; j < 4; ++j) o.p[j] = f2_fma(h.p[j], k2.p[j], f2_fma(f2_mul(g.p[j], gm.p[j]), k0.p[j], k1.p[j]));
          if (RES) {
            const Eight w = Eight::of(r2[r][i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) o.p[j] = f2_add(o.p[j], w.p[j]);
          }
          float f[8];
          o.split(f);
          out.set(f);
        }
        store_piece<ALIGNED, TPR>(out, p.gx + row * p.ldgx, at + i * stride, d, live[r], last);
      }
    }
  }
  pdl_trigger();
  float* to_g = p.parts ? p.parts + (int64_t)blockIdx.x * 2 * d : p.g_gamma;
  float* to_b = p.parts ? to_g + d : p.g_beta;
  float sum_g[NV][8], sum_b[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    acc_g[i].split(sum_g[i]);
    acc_b[i].split(sum_b[i]);
  }
  if constexpr (TPR == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (at + i * stride) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < d) {
          if (to_g) to_g[col + j] = sum_g[i][j];
          if (to_b) to_b[col + j] = sum_b[i][j];
        }
    }
  } else {
#pragma unroll
    for (int o = pl.TEAM; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum_g[i][j] += __shfl_xor_sync(0xffffffffu, sum_g[i][j], o);
          sum_b[i][j] += __shfl_xor_sync(0xffffffffu, sum_b[i][j], o);
        }
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int w = 0; w < warps; ++w) {
      if (warp == w && pl.team == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (at + i * stride) * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < d) {
              s_sums[col + j] = w ? s_sums[col + j] + sum_g[i][j] : sum_g[i][j];
              s_sums[d + col + j] = w ? s_sums[d + col + j] + sum_b[i][j] : sum_b[i][j];
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

// rows a team works on together (backward of 475,136 x 256: one 224 us, two 160, three 191, four 173; of 237,568 x 512: one 167, two 157; unaligned, of
// 100,003 x 509: one 174, two 229).  All without a residual; with one, two rows of 257 to 512 spill 72 bytes (fp32 rows 216 to 268), not measured against one.
constexpr int rows_together(int tpr, int nv, bool aligned, bool bwd) { return aligned && (bwd ? nv == 1 || tpr > 0 : nv == 1 && tpr > 0) ? 2 : 1; }

// How rows of d elements are shared out: lanes per team (TPR), steps per lane, rows worked on together
struct Shape {
  int tpr, nv, r;
  int threads;             // per block
  int rows_per_block;
  int resident;            // blocks per SM
};
constexpr int kMaxWidth = 8192;
// Rows above 512: by blocks (65,536 x 1,024 bf16 with a residual: forward 104 us, a warp's lanes with four pieces each 110; backward 113 / 202).  fp32 rows of
// that width lose by it in the forward: 90 us, by a warp's lanes 84; the rule takes no note of the type.
inline Shape shape_of(int d, bool aligned, bool bwd) {
  const int pieces = (int)pitch_of(d) / 8;
  Shape s;
  if (pieces <= 64) {
    s.tpr = pieces <= 4 ? 4 : pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32;
    s.nv = pieces <= 32 ? 1 : 2;
    s.r = rows_together(s.tpr, s.nv, aligned, bwd);
    s.threads = kThreads;
    s.rows_per_block = kThreads / s.tpr * s.r;
    s.resident = blocks_per_sm(s.tpr, aligned, bwd);
  } else {
    s.tpr = 0;
    s.nv = pieces <= 512 ? 1 : 2;
    s.r = rows_together(s.tpr, s.nv, aligned, bwd);
    s.threads = (int)round_up((pieces + s.nv - 1) / s.nv, 32);
    s.rows_per_block = s.r;
    s.resident = block_threads(0, aligned, bwd) / s.threads;
  }
  return s;
}
inline int blocks_of(const Shape& s, int64_t rows, bool bwd) {
  if (bwd && rows <= 4 * s.rows_per_block) return 1;         // its sums need no second kernel: a launch costs more than three turns
  const int64_t need = (rows + s.rows_per_block - 1) / s.rows_per_block, cap = (int64_t)sm_count() * s.resident;
  return (int)(need < cap ? need : cap);
}

template <typename T, typename TY>
int fwd(const FwdArgs<T, TY>& p, bool aligned, cudaStream_t stream);
template <typename T, typename TY>
int bwd(const BwdArgs<T, TY>& p, bool aligned, cudaStream_t stream);      // p.parts: blocks_of(shape_of(d, aligned, true), rows, true) rows of 2 d floats if that is above 1

// calls fn(TPR, NV) for the shape
template <typename Fn>
void with_shape(const Shape& s, Fn&& fn) {
#define BSRL_SHAPE(TPR_, NV_) \
  if (s.tpr == TPR_ && s.nv == NV_) return fn(std::integral_constant<int, TPR_>{}, std::integral_constant<int, NV_>{})
  BSRL_SHAPE(4, 1);
  BSRL_SHAPE(8, 1);
  BSRL_SHAPE(16, 1);
  BSRL_SHAPE(32, 1);
  BSRL_SHAPE(32, 2);
  BSRL_SHAPE(0, 1);
  BSRL_SHAPE(0, 2);
#undef BSRL_SHAPE
}
template <typename T, typename TY>
int launch_fwd(const FwdArgs<T, TY>& p, bool aligned, cudaStream_t stream) {
  const Shape s = shape_of(p.d, aligned, false);
  const int blocks = blocks_of(s, p.rows, false);
  with_shape(s, [&](auto TPR, auto NV) {
    constexpr int R = rows_together(TPR(), NV(), true, false), R1 = rows_together(TPR(), NV(), false, false);
    if (!aligned) launch_kernel(norm8_fwd_kernel<T, TY, false, true, TPR(), NV(), R1>, blocks, s.threads, 0, stream, p);
    else if (p.res) launch_kernel(norm8_fwd_kernel<T, TY, true, true, TPR(), NV(), R>, blocks, s.threads, 0, stream, p);
    else launch_kernel(norm8_fwd_kernel<T, TY, true, false, TPR(), NV(), R>, blocks, s.threads, 0, stream, p);
  });
  BSRL_LAUNCH_OK("norm8_fwd_kernel");
  return BSRL_OK;
}
template <typename T, typename TY>
int launch_bwd(const BwdArgs<T, TY>& p, bool aligned, cudaStream_t stream) {
  const Shape s = shape_of(p.d, aligned, true);
  const int blocks = blocks_of(s, p.rows, true);
  const size_t smem = s.tpr > 0 ? 2 * p.d * sizeof(float) : 0;
  with_shape(s, [&](auto TPR, auto NV) {
    constexpr int R = rows_together(TPR(), NV(), true, true), R1 = rows_together(TPR(), NV(), false, true);
    if (!aligned) launch_kernel(norm8_bwd_kernel<T, TY, false, true, TPR(), NV(), R1>, blocks, s.threads, smem, stream, p);
    else if (p.gres) launch_kernel(norm8_bwd_kernel<T, TY, true, true, TPR(), NV(), R>, blocks, s.threads, smem, stream, p);
    else launch_kernel(norm8_bwd_kernel<T, TY, true, false, TPR(), NV(), R>, blocks, s.threads, smem, stream, p);
  });
  BSRL_LAUNCH_OK("norm8_bwd_kernel");
  return BSRL_OK;
}

}  // namespace norm8
}  // namespace bsrl
