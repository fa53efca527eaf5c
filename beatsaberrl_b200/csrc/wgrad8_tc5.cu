// Weight gradient of a linear layer from an input that was kept in 8 bits (pack8.cuh):
//   g_weight (n, k) = g^T x8,  g_bias (n) = column sums of g,  over `rows` rows; g 16-bit, results fp32.
//
// Persistent, warp-specialised tcgen05 kernel.  The contraction runs over rows, so both operands are MN-major tiles of 64 rows as they
// lie in memory:
//   warp 0       TMA producer: (64 rows x 128 MH columns) of g per stage, 128-byte swizzle, columns and rows past the ends as zeros;
//   warp 1       MMA issuer: per stage MH accumulators of 128 x BN in TMEM (MH = 2, BN = 256: all of it), the x tile read by both;
//   warps 2..9   converters: 16 codes per 16-byte load, requested a stage ahead, to the 16-bit type of g (exact: the scale is a power of
//                two) and into the swizzled tile; after a chain they drain the accumulators;
//   warps 10..13 column sums of g from the stage, for the first column tile's work items only (no second read of g).
// A work item is (tile, piece of the rows).  The pieces' partial tiles go to the workspace and a second kernel adds them in order: the
// same bits every time.  Inside an item the accumulators are drained every kChain stages and added in fp32, rounded to nearest: the tensor
// core's own running sum truncates, about 2e-8 of the sum per 16 rows (475,136 rows in one chain per CTA were 7.6e-6 off).
// All waits are bounded (tc5.cuh); a wait that runs out sets the device status word and every role falls through to the teardown.
#include <cmath>

#include "kernels.cuh"
#include "pack8.cuh"
#include "tc5.cuh"

namespace bsrl {
namespace {
using namespace tc5;
using namespace p8;

constexpr int KERNEL_ID = 14;
constexpr int BK = 64;                           // rows per stage
constexpr int BLOCK_BYTES = BK * 128;            // 64 columns x 64 rows of 16 bits
constexpr int CONV_WARPS = 8, SUM_WARPS = 4;
constexpr int THREADS = (2 + CONV_WARPS + SUM_WARPS) * 32;
constexpr int MAX_BN = 256;
constexpr int TMEM_COLS = 512;
constexpr int kChain = 64;                       // stages between drains: 4,096 rows
constexpr int stages_of(int mh) { return mh == 2 ? 3 : 4; }
constexpr int stage_bytes(int mh) { return (2 * mh + 4) * BLOCK_BYTES; }
constexpr int smem_bytes(int mh) { return stages_of(mh) * stage_bytes(mh) + 1024 /*alignment*/ + 256 /*barriers*/; }
constexpr int phases_of(int mh) { return SUM_WARPS * 32 / (16 * mh); }      // threads that share eight columns of g

struct Shared {
  uint64_t full_g[4], full_x[4], empty[4], acc_full, acc_empty, mma_done;
  uint32_t tmem_base;
  int abort;
};
__device__ __forceinline__ void give_up(Shared* sh, int* status, int role) {
  atomicCAS(status, 0, KERNEL_ID * 16 + role);
  sh->abort = 1;
}

struct Args {
  const uint8_t* codes;
  const uint8_t* exps;
  int64_t rows;
  int64_t pitch;                 // of the codes
  int n, bn;                     // bn: columns of a tile of x
  int k_tiles, tiles, splits;    // tiles = n tiles x k tiles
  int k_blocks;                  // stages of all rows
  float* parts;                  // (tiles, splits, 4 MH, bn, 32)
  float* bias_parts;             // (splits, phases, n tiles x 128 MH), nullptr: no column sums
};

// Item w -> (tile, split): the splits of a tile are neighbours, the k tiles of the same rows run at the same time
struct Item {
  int tile, split, nt, kt, kb0, kb1;
};
__device__ __forceinline__ Item item_of(int w, const Args& p) {
  Item it;
  it.split = w / p.tiles;
  it.tile = w - it.split * p.tiles;
  it.nt = it.tile / p.k_tiles;
  it.kt = it.tile - it.nt * p.k_tiles;
  it.kb0 = (int)((int64_t)p.k_blocks * it.split / p.splits);
  it.kb1 = (int)((int64_t)p.k_blocks * (it.split + 1) / p.splits);
  return it;
}

template <typename TG, int KIND, int MH>
__global__ void __launch_bounds__(THREADS, 1)
wgrad8_kernel(const __grid_constant__ CUtensorMap tm_g, Args p, int* status) {
  constexpr int STAGES = stages_of(MH), STAGE_BYTES = stage_bytes(MH), G_BYTES = 2 * MH * BLOCK_BYTES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* tiles_ptr = smem_raw + (base - raw);
  Shared* sh = reinterpret_cast<Shared*>(tiles_ptr + STAGES * STAGE_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &sh->abort;
  const int n_items = p.tiles * p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&sh->full_g[s]), 1);
      mbar_init(smem_u32(&sh->full_x[s]), CONV_WARPS);
      mbar_init(smem_u32(&sh->empty[s]), 1 + (p.bias_parts ? SUM_WARPS : 0));
    }
    mbar_init(smem_u32(&sh->acc_full), 1);
    mbar_init(smem_u32(&sh->acc_empty), CONV_WARPS);
    mbar_init(smem_u32(&sh->mma_done), 1);
    sh->abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_g);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sh->tmem_base), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;
  pdl_begin();

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
        const Item m = item_of(w, p);
        for (int kb = m.kb0; kb < m.kb1; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(smem_u32(&sh->empty[s]), ((it / STAGES) & 1) ^ 1, abort)) { give_up(sh, status, 1); ok = false; break; }
          const uint32_t bar = smem_u32(&sh->full_g[s]);
          mbar_expect_tx(bar, G_BYTES);
#pragma unroll
          for (int b = 0; b < 2 * MH; ++b) tma_load_2d(base + s * STAGE_BYTES + b * BLOCK_BYTES, &tm_g, m.nt * (128 * MH) + b * 64, kb * BK, bar);
        }
      }
      // what is in flight must land before this CTA may exit (bounded, ignoring abort)
      for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j) {
        uint32_t spins = 0;
        while (!mbar_try_wait(smem_u32(&sh->full_g[j % STAGES]), (j / STAGES) & 1) && ++spins < kSpinLimit) {}
        if (spins >= kSpinLimit) give_up(sh, status, 2);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      uint32_t it = 0, chains = 0;
      bool ok = true;
      uint32_t idesc = idesc_f16(128, p.bn, 1, 1);
      if (sizeof(TG) == 2 && top_binade<TG>() == 127) idesc |= (1u << 7) | (1u << 10);      // both operands bf16
      for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
        const Item m = item_of(w, p);
        for (int kb = m.kb0; kb < m.kb1; ++kb, ++it) {
          const int pos = (kb - m.kb0) % kChain;
          if (pos == 0) {
            if (!mbar_wait(smem_u32(&sh->acc_empty), (chains & 1) ^ 1, abort)) { give_up(sh, status, 3); ok = false; break; }
            ++chains;
          }
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(smem_u32(&sh->full_g[s]), ph, abort) || !mbar_wait(smem_u32(&sh->full_x[s]), ph, abort)) { give_up(sh, status, 4); ok = false; break; }
          tc_fence_after();
          const uint32_t g_addr = base + s * STAGE_BYTES;
          const uint64_t x_desc = smem_desc_mn_sw128(g_addr + G_BYTES, BLOCK_BYTES);
#pragma unroll
          for (int h = 0; h < MH; ++h) {
            const uint64_t g_desc = smem_desc_mn_sw128(g_addr + h * 2 * BLOCK_BYTES, BLOCK_BYTES);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) mma_f16_ss(tmem_base + h * MAX_BN, g_desc + 128 * k, x_desc + 128 * k, idesc, (pos || k) ? 1u : 0u);
          }
          tc_commit(smem_u32(&sh->empty[s]));
          if (pos == kChain - 1 || kb == m.kb1 - 1) tc_commit(smem_u32(&sh->acc_full));
        }
      }
      // every MMA issued must have retired before TMEM is freed (bounded, ignoring abort)
      tc_commit(smem_u32(&sh->mma_done));
      uint32_t spins = 0;
      while (!mbar_try_wait(smem_u32(&sh->mma_done), 0) && ++spins < kSpinLimit) {}
      if (spins >= kSpinLimit) give_up(sh, status, 5);
    }
  } else if (warp < 2 + CONV_WARPS) {
    // ---------------------------------------------------------------- converters, then the drain
    const int t = threadIdx.x - 64;                // 0 .. 255
    const int per_row = p.bn / 16, n_pieces = per_row * BK;
    constexpr int MAX_P = MAX_BN / 16 * BK / (CONV_WARPS * 32);       // pieces of 16 codes per thread and stage: 4
    int row[MAX_P], piece[MAX_P];
    uint32_t dst[MAX_P];
#pragma unroll
    for (int i = 0; i < MAX_P; ++i) {
      const int q = t + i * CONV_WARPS * 32;
      row[i] = q < n_pieces ? q / per_row : -1;
      piece[i] = q - (q / per_row) * per_row;
      dst[i] = (uint32_t)(G_BYTES + (piece[i] >> 2) * BLOCK_BYTES + row[i] * 128);
    }
    uint4 code[MAX_P];
    uint32_t ex[MAX_P];
    auto request = [&](const Item& m, int kb) {
#pragma unroll
      for (int i = 0; i < MAX_P; ++i) {
        const int64_t r = (int64_t)kb * BK + row[i];
        const int64_t col = (int64_t)m.kt * p.bn + piece[i] * 16;
        code[i] = make_uint4(0, 0, 0, 0);
        ex[i] = 0;
        if (row[i] >= 0 && r < p.rows && col < p.pitch) {
          code[i] = *reinterpret_cast<const uint4*>(p.codes + r * p.pitch + col);
          ex[i] = p.exps[r * (p.pitch / kBlock) + col / kBlock];
        }
      }
    };
    uint32_t it = 0, chains = 0;
    bool ok = true;
    const int quad = warp & 3, half = (warp - 2) >> 2;
    if ((int)blockIdx.x < n_items) {
      const Item m = item_of(blockIdx.x, p);
      request(m, m.kb0);
    }
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
      const Item m = item_of(w, p);
      for (int kb = m.kb0; kb < m.kb1; ++kb, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait_warp(smem_u32(&sh->empty[s]), ((it / STAGES) & 1) ^ 1, abort)) {
          if (lane == 0) give_up(sh, status, 6);
          ok = false;
          break;
        }
#pragma unroll
        for (int i = 0; i < MAX_P; ++i) {
          if (row[i] >= 0) {
            const float sc = scale_of(ex[i]);
            const uint32_t wd[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
            uint4 o[2];
            uint32_t* ow = reinterpret_cast<uint32_t*>(o);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float a, b, c, d;
              decode4<KIND>(wd[j], a, b, c, d);
              ow[2 * j] = pack2<TG>(a * sc, b * sc);
              ow[2 * j + 1] = pack2<TG>(c * sc, d * sc);
            }
            // the piece's two 16-byte chunks; every other four lanes the second one first, so that eight lanes cover all banks
            uint8_t* at = tiles_ptr + s * STAGE_BYTES + dst[i];
            const int c0 = (piece[i] & 3) * 2, flip = (piece[i] >> 2) & 1;
            *reinterpret_cast<uint4*>(at + (((c0 + flip) ^ (row[i] & 7)) << 4)) = flip ? o[1] : o[0];
            *reinterpret_cast<uint4*>(at + (((c0 + (flip ^ 1)) ^ (row[i] & 7)) << 4)) = flip ? o[0] : o[1];
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->full_x[s]));
        // the next stage's codes
        if (kb + 1 < m.kb1) {
          request(m, kb + 1);
        } else if (w + (int)gridDim.x < n_items) {
          const Item next = item_of(w + gridDim.x, p);
          request(next, next.kb0);
        }
        const int pos = (kb - m.kb0) % kChain;
        if (pos == kChain - 1 || kb == m.kb1 - 1) {
          if (!mbar_wait_warp(smem_u32(&sh->acc_full), chains & 1, abort)) {
            if (lane == 0) give_up(sh, status, 7);
            ok = false;
            break;
          }
          ++chains;
          tc_fence_after();
          const bool first = kb - m.kb0 < kChain;
          float* part = p.parts + ((int64_t)m.tile * p.splits + m.split) * (4 * MH * 32) * p.bn;
          // 32 rows x 32 columns at a time; a lane's row in every column's 128 bytes
          for (int c = MH == 2 ? 0 : half * 32; c < p.bn; c += MH == 2 ? 32 : 64) {
            uint32_t r[32];
            const int h = MH == 2 ? half : 0;
            tmem_ld32(tmem_base + ((uint32_t)(quad * 32) << 16) + h * MAX_BN + c, r);
            float* out = part + ((int64_t)(h * 4 + quad) * p.bn + c) * 32 + lane;
            const int cols = min(32, p.bn - c);
            float old[32];
            if (!first) {
#pragma unroll
              for (int j = 0; j < 32; ++j) old[j] = j < cols ? out[j * 32] : 0.f;
            }
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < cols) out[j * 32] = first ? __uint_as_float(r[j]) : old[j] + __uint_as_float(r[j]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->acc_empty));
        }
      }
    }
  } else if (p.bias_parts) {
    // ---------------------------------------------------------------- column sums of g
    const int t = threadIdx.x - (2 + CONV_WARPS) * 32;          // 0 .. 127
    constexpr int CHUNKS = 16 * MH, PHASES = phases_of(MH);
    const int chunk = t % CHUNKS, phase = t / CHUNKS;           // eight columns, every PHASES-th row; a partial sum each
    uint32_t it = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < n_items && ok; w += gridDim.x) {
      const Item m = item_of(w, p);
      float acc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      for (int kb = m.kb0; kb < m.kb1; ++kb, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait_warp(smem_u32(&sh->full_g[s]), (it / STAGES) & 1, abort)) {
          if (lane == 0) give_up(sh, status, 8);
          ok = false;
          break;
        }
        if (m.kt == 0) {
          const uint8_t* blk = tiles_ptr + s * STAGE_BYTES + (chunk >> 3) * BLOCK_BYTES;
#pragma unroll 8
          for (int r = phase; r < BK; r += PHASES) {
            const uint4 v = *reinterpret_cast<const uint4*>(blk + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
            float f[8];
            unpack2<TG>(v.x, f[0], f[1]);
            unpack2<TG>(v.y, f[2], f[3]);
            unpack2<TG>(v.z, f[4], f[5]);
            unpack2<TG>(v.w, f[6], f[7]);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += f[j];
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->empty[s]));
      }
      if (ok && m.kt == 0) {
        float4* out = reinterpret_cast<float4*>(p.bias_parts + (((int64_t)m.split * PHASES + phase) * (p.tiles / p.k_tiles) + m.nt) * (128 * MH) + chunk * 8);
        out[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        out[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Adds the partial tiles in the order of their rows: a block takes 32 x 32 of the weight (or, past those, 256 of the bias).
struct AddArgs {
  const float* parts;
  const float* bias_parts;
  float* gw;
  float* gb;
  int64_t ldw;
  int n, k, bn, k_tiles, tiles, splits, mh;
  int64_t patches;
};
__global__ void __launch_bounds__(256) wgrad8_add_kernel(AddArgs p) {
  pdl_begin();
  if (blockIdx.x >= p.patches) {
    const int c = (int)(blockIdx.x - p.patches) * 256 + threadIdx.x, width = p.tiles / p.k_tiles * 128 * p.mh;
    if (c < p.n) {
      float sum = 0.f;
#pragma unroll 8
      for (int s = 0; s < p.splits * phases_of(p.mh); ++s) sum += p.bias_parts[(int64_t)s * width + c];
      p.gb[c] = sum;
    }
    return;
  }
  __shared__ float patch[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (p.bn + 31) / 32, blocks = 4 * p.mh;
  int64_t i = blockIdx.x;
  const int chunk = (int)(i % chunks);
  i /= chunks;
  const int blk = (int)(i % blocks), tile = (int)(i / blocks);
  const int64_t slot = (int64_t)blocks * p.bn * 32;
  const float* from = p.parts + (int64_t)tile * p.splits * slot + ((int64_t)blk * p.bn + chunk * 32) * 32 + lane;
  const int cols = min(32, p.bn - chunk * 32);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (warp + 8 * j < cols) sum[j] += from[s * slot + (warp + 8 * j) * 32];
#pragma unroll
  for (int j = 0; j < 4; ++j) patch[warp + 8 * j][lane] = sum[j];
  __syncthreads();
  const int nt = tile / p.k_tiles, kt = tile % p.k_tiles;
  const int col = kt * p.bn + chunk * 32 + lane;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = nt * 128 * p.mh + blk * 32 + warp + 8 * j;
    if (row < p.n && col < p.k && lane < cols) p.gw[(int64_t)row * p.ldw + col] = patch[lane][warp + 8 * j];
  }
}

// A copy of g with rows that 16 bytes divide, for TMA (n or its pitch odd, or an unaligned first element)
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ g, int64_t ldg, int64_t rows, int n, uint16_t* __restrict__ out,
                                                         int ldo) {
  pdl_begin();
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += (int64_t)gridDim.x * 8)
    for (int c = threadIdx.x & 31; c < n; c += 32) out[row * ldo + c] = g[row * ldg + c];
}

// How a call is cut up
struct Plan {
  int mh, bn, k_tiles, tiles, splits, k_blocks;
  bool copy;
  int64_t copy_bytes, parts_bytes, bias_bytes;
};
Plan plan_of(int64_t rows, int n, int k, bool copy) {
  Plan best{};
  best.k_blocks = (int)((rows + BK - 1) / BK);
  best.copy = copy;
  const int sms = sm_count();
  double cost = 1e30;
  for (int mh = 1; mh <= 2; ++mh)
    for (int most = 64; most <= MAX_BN; most *= 2) {
      const int k_tiles = (k + most - 1) / most, bn = (int)round_up((k + k_tiles - 1) / k_tiles, 16);
      const int64_t tiles = (int64_t)((n + 128 * mh - 1) / (128 * mh)) * k_tiles;
      if (tiles > 1 << 20) continue;
      // cycles of a stage: conversions, MMAs with their operand reads; of a drain; of the partial tiles' way to memory and back, all SMs
      const double stage = fmax(2.2 * bn, fmax(4.0 * mh * 0.65 * bn, 140.0)), drain = 1500 + 24.0 * mh * bn;
      // pieces of the rows: as fill one or more waves of SMs, or stages of some length each
      for (int i = 0; i < 10; ++i) {
        int64_t splits = i < 4 ? (i + 1) * (int64_t)sms / tiles : best.k_blocks >> (i - 4);
        splits = splits < 1 ? 1 : splits > best.k_blocks ? best.k_blocks : splits;
        if (splits > 2 * sms) continue;
        const double waves = (double)((tiles * splits + sms - 1) / sms), per = (double)((best.k_blocks + splits - 1) / splits);
        const double c = waves * (per * stage + drain * ceil(per / kChain)) + (double)tiles * splits * 128 * mh * bn * 4 / 5000.0;
        if (c < cost) {
          cost = c;
          best.mh = mh; best.bn = bn; best.k_tiles = k_tiles; best.tiles = (int)tiles; best.splits = (int)splits;
        }
      }
    }
  best.copy_bytes = copy ? round_up(rows * round_up(n, 8) * 2, 256) : 0;
  best.parts_bytes = round_up((int64_t)best.tiles * best.splits * 128 * best.mh * best.bn * 4, 256);
  best.bias_bytes = round_up((int64_t)best.splits * phases_of(best.mh) * (best.tiles / best.k_tiles) * 128 * best.mh * 4, 256);
  return best;
}

template <typename TG, int KIND>
void launch(const Plan& pl, const CUtensorMap& tm, const Args& p, int* status, cudaStream_t stream) {
  const int items = p.tiles * p.splits, grid = items < sm_count() ? items : sm_count();
  if (pl.mh == 2) launch_kernel(wgrad8_kernel<TG, KIND, 2>, grid, THREADS, smem_bytes(2), stream, tm, p, status);
  else launch_kernel(wgrad8_kernel<TG, KIND, 1>, grid, THREADS, smem_bytes(1), stream, tm, p, status);
}
bool needs_copy(const void* g, int64_t ldg) { return !aligned16(g) || ldg % 8 != 0; }
}  // namespace

int64_t wgrad8_workspace(int64_t rows, int n, int k, bool aligned) {
  const Plan pl = plan_of(rows, n, k, !aligned);
  return pl.copy_bytes + pl.parts_bytes + pl.bias_bytes;
}

int wgrad8(const void* g, int g_dtype, int64_t ldg, const uint8_t* codes, const uint8_t* exps, int kind, int64_t rows, int n, int k, float* gw,
           int64_t ldw, float* gb, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  const Plan pl = plan_of(rows, n, k, needs_copy(g, ldg));
  if (workspace_bytes < pl.copy_bytes + pl.parts_bytes + pl.bias_bytes) {
    set_error("linear8_weight_grad: workspace %lld bytes < required %lld", (long long)workspace_bytes,
              (long long)(pl.copy_bytes + pl.parts_bytes + pl.bias_bytes));
    return BSRL_ERR_WORKSPACE;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (pl.copy) {
    const int64_t need = (rows + 7) / 8, cap = (int64_t)sm_count() * 8;
    launch_kernel(align_rows_kernel, (unsigned)(need < cap ? need : cap), 256, 0, stream, static_cast<const uint16_t*>(g), ldg, rows, n,
                  reinterpret_cast<uint16_t*>(ws), (int)round_up(n, 8));
    BSRL_LAUNCH_OK("align_rows_kernel");
    g = ws;
    ldg = round_up(n, 8);
  }
  float* parts = reinterpret_cast<float*>(ws + pl.copy_bytes);
  float* bias_parts = gb ? reinterpret_cast<float*>(ws + pl.copy_bytes + pl.parts_bytes) : nullptr;
  CUtensorMap tm;
  if (!make_tmap_f16(&tm, g, rows, n, ldg, BK)) return BSRL_ERR_CUDA;
  const Args p{codes, exps, rows, pitch_of(k), n, pl.bn, pl.k_tiles, pl.tiles, pl.splits, pl.k_blocks, parts, bias_parts};
  static DeviceOnce once;
  const int rc = once.run("wgrad8_kernel set-up", [] {
    cudaError_t e = cudaSuccess;
    for (auto* k : {wgrad8_kernel<__half, kInt8, 1>, wgrad8_kernel<__half, kE4m3, 1>, wgrad8_kernel<__nv_bfloat16, kInt8, 1>, wgrad8_kernel<__nv_bfloat16, kE4m3, 1>})
      if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(1));
    for (auto* k : {wgrad8_kernel<__half, kInt8, 2>, wgrad8_kernel<__half, kE4m3, 2>, wgrad8_kernel<__nv_bfloat16, kInt8, 2>, wgrad8_kernel<__nv_bfloat16, kE4m3, 2>})
      if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(2));
    return e;
  });
  if (rc != BSRL_OK) return rc;
  int* status = device_status_ptr();
  if (!status) return BSRL_ERR_CUDA;
  if (g_dtype == BSRL_F16) kind == kInt8 ? launch<__half, kInt8>(pl, tm, p, status, stream) : launch<__half, kE4m3>(pl, tm, p, status, stream);
  else kind == kInt8 ? launch<__nv_bfloat16, kInt8>(pl, tm, p, status, stream) : launch<__nv_bfloat16, kE4m3>(pl, tm, p, status, stream);
  BSRL_LAUNCH_OK("wgrad8_kernel");
  AddArgs a{parts, bias_parts, gw, gb, ldw, n, k, pl.bn, pl.k_tiles, pl.tiles, pl.splits, pl.mh, 0};
  a.patches = (int64_t)pl.tiles * 4 * pl.mh * ((pl.bn + 31) / 32);
  PdlScope overlap;
  pdl_enable();
  launch_kernel(wgrad8_add_kernel, (unsigned)(a.patches + (gb ? (n + 255) / 256 : 0)), 256, 0, stream, a);
  BSRL_LAUNCH_OK("wgrad8_add_kernel");
  return BSRL_OK;
}

}  // namespace bsrl
