// Weight gradient of a linear layer from an input that was kept in 8 bits (pack8.cuh):
//   g_weight (n, k) = g^T x8,  g_bias (n) = column sums of g,  over `rows` rows; g 16-bit, results fp32.
//
// Persistent, warp-specialised tcgen05 kernel, one CTA per SM or (CTAS = 2) pairs of CTAs on neighbouring SMs.  The contraction runs
// over rows, so both operands are MN-major tiles of 64 rows as they lie in memory; a tile of the result has 128 CTAS MH x BN elements:
//   warp 0        TMA producer of g: 64 rows x the CTA's own 128 MH columns per stage, columns and rows past the ends as zeros;
//   warp 1        MMA issuer (a pair's leader's), into one of two sets of accumulators of BN columns in TMEM;
//   converters    16 codes per 16-byte load to the 16-bit type of g (exact: the scale is a power of two), into the swizzled tile that the
//                 MMAs (of both CTAs) read.  Groups of warps take stages in turn and request a stage's codes before they wait for its slot, so several
//                 stages' loads are under way;
//   drain         accumulators to the workspace while the next chain runs into the other set (one set where a CTA has two accumulators
//                 beside each other: the MMAs wait);
//   column sums   of g from the stage, for the first column tile's work items only (no second read of g).
// Why groups: the proxy fence ahead of a converter's arrival waits for all loads its thread has in flight, so a thread cannot hold the
// next stages' codes in registers (that took 2,150 cycles a stage, a load's latency each).  Codes through a TMA ring instead cost the shared
// memory 16 KB a stage, which is what bounds the kernel together with the issue slots: 1,310 cycles a stage with column sums, 1,030 without.
// A work item is (tile, piece of the rows).  The pieces' partial tiles go to the workspace and a second kernel adds them in order: the
// same bits every time.  Inside an item the accumulators are drained every kChain stages and added in fp32, rounded to nearest: the tensor
// core's own running sum truncates, about 2e-8 of the sum per 16 rows (475,136 rows in chains of 6,420 were 7.6e-6 off, of 2,048 2e-6).
// A pair halves what a CTA converts and what its MMAs read of shared memory; two accumulators per CTA halve the conversions per MMA again.
// 475,136 x 1,024 x 256 with chains of 2,560 rows (floor 170 us by bytes, 149 by FLOPs): one CTA 607 us, pairs 288, pairs with two accumulators 263 (282 with all
// CTAs' drains at once, 232 with no drains but the last: the additions into L2 are what is left); 100,003 x 2,048 x 2,048: 1,860 / 898 / 734.
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
constexpr int MAX_BN = 256;
constexpr int TMEM_COLS = 2 * MAX_BN;
// Stages between drains: 2,560 rows of bf16, 1,152 of fp16, whose longer products lose more to the tensor cores' truncation.  Norm of the error against
// 64 bits over that of the sums, normal numbers, int8 / e4m3: 22,725 x 200 x 671 fp16 1.2e-6 / 1.3e-6 with 40 stages, 7.1e-7 / 7.6e-7 with 18; in longer pieces 2.2e-6 and 9.1e-7;
// bf16 with 40 up to 5.7e-7 / 7.9e-7.  bf16 gains by blocks that share an exponent from row to row: with rows whose sizes differ by a factor of e 1.6e-6 (fp16 1.3e-6), of
// e^2 3.7e-6; with k = 1 1.5e-6 to 2e-6.  An fp32 product of 100,003 x 1,000 x 513: 1.9e-6 to 4.6e-6, rows by e^2 6.4e-6.  475,136 x 1,024 x 256 fp16 takes 288 us
// instead of 261 for its chains.
constexpr int kChain = 40, kChainF16 = 18;
template <typename TG>
__host__ __device__ constexpr int chain_of() { return top_binade<TG>() == 15 ? kChainF16 : kChain; }
// An item's first chain: of another length for neighbouring items, so that the CTAs do not all drain at once (they add into L2 at its rate
// for atomics, 4.8 TB/s, and the MMAs of two accumulators wait)
template <typename TG>
__device__ __forceinline__ int first_chain(int item) { return chain_of<TG>() - (item % 8) * chain_of<TG>() / 8; }

// CTAS: 1, or 2: a pair.  MH: accumulators of 128 columns of g beside each other per CTA.
template <int CTAS, int MH>
struct Form {
  static constexpr int G_BYTES = 2 * MH * BLOCK_BYTES, STAGE_BYTES = G_BYTES + 4 / CTAS * BLOCK_BYTES;
  static constexpr int STAGES = CTAS == 1 ? 4 : MH == 1 ? 6 : 4;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 /*alignment*/ + 512 /*barriers*/;
  static constexpr int BUFS = 2 / MH;                                          // sets of accumulators in TMEM
  // Converters take stages in turn, a group each; sum warps likewise.  A group always has the same slots of the ring: its waits, by parity, are
  // for consecutive phases of their barriers.  (Groups that do not divide the stages meet a slot every other time, and slots are freed out of
  // order where the sums lag: a wait could then take the phase before the last one for the last one.)
  static constexpr int CONV_WARPS = CTAS == 1 ? 16 : MH == 1 ? 12 : 8, GROUPS = CTAS == 1 ? 2 : CONV_WARPS / 4;
  static constexpr int SUM_WARPS = MH == 1 && CTAS == 2 ? 6 : 4, SUM_GROUPS = CTAS == 1 ? 2 : SUM_WARPS;
  static_assert(STAGES % GROUPS == 0 && STAGES % SUM_GROUPS == 0, "phases");
  static constexpr int CHUNKS = 16 * MH, PHASES = SUM_WARPS * 32 / CHUNKS;     // pieces of eight columns of g; threads that share one
  static constexpr int CONV0 = 2, DRAIN0 = CONV0 + CONV_WARPS, SUM0 = DRAIN0 + 4 * MH, THREADS = (SUM0 + SUM_WARPS) * 32;      // first warp of each role
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct Shared {
  uint64_t full_g[6], full_x[6], empty[6], acc_full[2], acc_empty[2], mma_done;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Shared) <= 512, "barrier space");
__device__ __forceinline__ void give_up(Shared* sh, int* status, int role) {
  atomicCAS(status, 0, KERNEL_ID * 16 + role);
  sh->abort = 1;
}

struct Args {
  const uint8_t* codes;
  const uint8_t* exps;
  int64_t rows;
  int64_t pitch;                 // of the codes
  int bn;                        // columns of a tile of x
  int n_tiles, k_tiles, splits;    // n tiles of 128 CTAS MH columns of g
  int k_blocks;                  // stages of all rows
  float* parts;                  // (tiles, splits, 4 CTAS MH, bn / 4, 32 rows, 4 columns)
  float* bias_parts;             // (splits, PHASES, n_tiles x 128 CTAS MH), nullptr: no column sums
};

// Item w -> (split, n tile, k tile), split-major: the tiles of the same rows run at the same time
struct Item {
  int split, nt, kt, kb0, kb1;
};
__device__ __forceinline__ Item item_of(int w, const Args& p) {
  Item it;
  const int tiles = p.n_tiles * p.k_tiles;
  it.split = w / tiles;
  const int tile = w - it.split * tiles;
  it.nt = tile / p.k_tiles;
  it.kt = tile - it.nt * p.k_tiles;
  it.kb0 = (int)((int64_t)p.k_blocks * it.split / p.splits);
  it.kb1 = (int)((int64_t)p.k_blocks * (it.split + 1) / p.splits);
  return it;
}

// With one k tile g is read once and should not displace the partial tiles from the L2 (475,136 x 1,024 x 256, chains of 2,560 rows, 265 -> 259 us, back to back 325 -> 316;
// with more of them each reads g, and the hint costs 8 %)
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void tma_load_2d_once(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}

// a, b += the two 16-bit numbers of w, in fp32
template <typename TG>
__device__ __forceinline__ void add_pair(uint32_t w, float& a, float& b) {
  if (top_binade<TG>() == 15)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.f32.f16 %0, l, %0;\n\tadd.f32.f16 %1, h, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.f32.bf16 %0, l, %0;\n\tadd.f32.bf16 %1, h, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(w));
}

// 16 codes and their exponent -> 16 numbers of 16 bits, two at a time where the scale allows it
template <typename TG, int KIND>
__device__ __forceinline__ void convert16(const uint4& code, uint32_t e, uint32_t (&o)[8]) {
  const uint32_t w[4] = {code.x, code.y, code.z, code.w};
  constexpr bool F16 = top_binade<TG>() == 15;
  if (F16 && e - 113u < 19u) {               // 2^-14 .. 2^4: the scale, and 1152 times it, are normal fp16 numbers
    const uint32_t sc = ((e - 112u) << 10) * 0x10001u;
    const __half2 s2 = *reinterpret_cast<const __half2*>(&sc);
    const __half2 off = __hmul2(s2, __floats2half2_rn(-1152.f, -1152.f));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo, hi;
      __half2 a, b;
      if (KIND == kInt8) {
        const uint32_t u = w[j] ^ 0x80808080u;                                // 1152 + code = 1024 + (code + 128)
        lo = __byte_perm(u, 0x64646464u, 0x4140);
        hi = __byte_perm(u, 0x64646464u, 0x4342);
        a = __hfma2(*reinterpret_cast<__half2*>(&lo), s2, off);               // code x scale, exactly
        b = __hfma2(*reinterpret_cast<__half2*>(&hi), s2, off);
      } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w[j]));
        a = __hmul2(*reinterpret_cast<__half2*>(&lo), s2);
        b = __hmul2(*reinterpret_cast<__half2*>(&hi), s2);
      }
      o[2 * j] = *reinterpret_cast<uint32_t*>(&a);
      o[2 * j + 1] = *reinterpret_cast<uint32_t*>(&b);
    }
    return;
  }
  const float s = scale_of(e);
  if (!F16 && KIND == kInt8 && e - 1u < 200u) {           // 2^23 times the scale is finite
    const uint64_t s2 = f2_make(s, s), off = f2_make(-8388736.f * s, -8388736.f * s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = w[j] ^ 0x80808080u;
      float a, b, c, d;
      f2_split(f2_fma(f2_make(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7651))), s2, off), a, b);
      f2_split(f2_fma(f2_make(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7652)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7653))), s2, off), c, d);
      o[2 * j] = pack2<TG>(a, b);
      o[2 * j + 1] = pack2<TG>(c, d);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b, c, d;
    decode4<KIND>(w[j], a, b, c, d);
    o[2 * j] = pack2<TG>(a * s, b * s);
    o[2 * j + 1] = pack2<TG>(c * s, d * s);
  }
}

template <typename TG, int KIND, int CTAS, int MH>
__global__ void __launch_bounds__(Form<CTAS, MH>::THREADS, 1)
wgrad8_kernel(const __grid_constant__ CUtensorMap tm_g, Args p, int* status) {
  using F = Form<CTAS, MH>;
  constexpr bool PAIR = CTAS == 2;
  constexpr int STAGES = F::STAGES, STAGE_BYTES = F::STAGE_BYTES, G_BYTES = F::G_BYTES;
  constexpr int GROUPS = F::GROUPS, GROUP_WARPS = F::CONV_WARPS / GROUPS, CONV0 = F::CONV0, DRAIN0 = F::DRAIN0, SUM0 = F::SUM0;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* tiles_ptr = smem_raw + (base - raw);
  Shared* sh = reinterpret_cast<Shared*>(tiles_ptr + STAGES * STAGE_BYTES);
  const int own = p.bn / CTAS;                // columns of the x tile that this CTA converts
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  volatile int* abort = &sh->abort;
  const int n_items = p.n_tiles * p.k_tiles * p.splits;
  const int w_first = (int)blockIdx.x / CTAS, w_step = (int)gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&sh->full_g[s]), 1);
      mbar_init(smem_u32(&sh->full_x[s]), CTAS * GROUP_WARPS);       // the leader's: both CTAs' converters
      mbar_init(smem_u32(&sh->empty[s]), 1 + (p.bias_parts ? F::SUM_WARPS / F::SUM_GROUPS : 0));
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sh->acc_full[b]), 1);
      mbar_init(smem_u32(&sh->acc_empty[b]), CTAS * 4 * MH);   // the leader's: both CTAs' drain warps
    }
    mbar_init(smem_u32(&sh->mma_done), 1);
    sh->abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_g);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(&sh->tmem_base), TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&sh->tmem_base), TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();          // the peer's barriers exist before anything is signalled across
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;
  pdl_begin();
  // an arrival at the leader's barrier; its MMA issuer waits for it at cluster scope
  auto arrive_leader = [&](uint64_t* bar) {
    const uint32_t at = PAIR ? map_to_cta(smem_u32(bar), 0) : smem_u32(bar);
    if (PAIR) mbar_arrive_cluster(at);
    else mbar_arrive(at);
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      uint32_t it = 0, s = 0, phase = 0;
      const uint64_t once = evict_first();
      bool ok = true;
      for (int w = w_first; w < n_items && ok; w += w_step) {
        const Item m = item_of(w, p);
        const int x = (m.nt * CTAS + rank) * (128 * MH);
        for (int kb = m.kb0; kb < m.kb1; ++kb, ++it) {
          if (!mbar_wait(smem_u32(&sh->empty[s]), phase ^ 1, abort)) { give_up(sh, status, 1); ok = false; break; }
          const uint32_t bar = smem_u32(&sh->full_g[s]), dst = base + s * STAGE_BYTES;
          mbar_expect_tx(bar, G_BYTES);
#pragma unroll
          for (int b = 0; b < 2 * MH; ++b) {
            if (p.k_tiles == 1) tma_load_2d_once(dst + b * BLOCK_BYTES, &tm_g, x + b * 64, kb * BK, bar, once);
            else tma_load_2d(dst + b * BLOCK_BYTES, &tm_g, x + b * 64, kb * BK, bar);
          }
          if (++s == STAGES) { s = 0; phase ^= 1; }
        }
      }
      // what is in flight must land before this CTA may exit (bounded, ignoring abort)
      uint32_t spins = 0;
      for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j)
        while (!mbar_try_wait(smem_u32(&sh->full_g[j % STAGES]), (j / STAGES) & 1) && ++spins < kSpinLimit) {}
      if (spins >= kSpinLimit) give_up(sh, status, 2);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0 && rank == 0) {
      // One thread issues everything: slots, phases and descriptors by counters, nothing derived per stage
      uint32_t slot = 0, phase = 0, buf = 0, acc_phase = 1;
      bool ok = true;
      uint32_t idesc = idesc_f16(128 * CTAS, p.bn, 1, 1);
      if (top_binade<TG>() == 127) idesc |= (1u << 7) | (1u << 10);      // both operands bf16
      const uint64_t g0 = smem_desc_mn_sw128(base, BLOCK_BYTES), x0 = smem_desc_mn_sw128(base + G_BYTES, BLOCK_BYTES);
      for (int w = w_first; w < n_items && ok; w += w_step) {
        const Item m = item_of(w, p);
        int n = 0;
        for (int left = m.kb1 - m.kb0; left > 0 && ok; left -= n) {
          if (!mbar_wait<PAIR>(smem_u32(&sh->acc_empty[buf]), acc_phase, abort)) { give_up(sh, status, 3); ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + buf * MAX_BN;
          n = min(left, n == 0 ? first_chain<TG>(w) : chain_of<TG>());
          for (int i = 0; i < n; ++i) {
            // the converters' arrivals stand for g too
            if (!mbar_wait<PAIR>(smem_u32(&sh->full_x[slot]), phase, abort)) { give_up(sh, status, 4); ok = false; break; }
            tc_fence_after();
            const uint64_t g_desc = g0 + slot * (STAGE_BYTES >> 4), x_desc = x0 + slot * (STAGE_BYTES >> 4);
#pragma unroll
            for (int h = 0; h < MH; ++h)
#pragma unroll
              for (int k = 0; k < BK / 16; ++k) {
                const uint64_t g_at = g_desc + h * (2 * BLOCK_BYTES >> 4) + 128 * k;
                if (PAIR) mma_f16_ss_pair(d + h * MAX_BN, g_at, x_desc + 128 * k, idesc, (i || k) ? 1u : 0u);
                else mma_f16_ss(d + h * MAX_BN, g_at, x_desc + 128 * k, idesc, (i || k) ? 1u : 0u);
              }
            PAIR ? tc_commit_pair(smem_u32(&sh->empty[slot])) : tc_commit(smem_u32(&sh->empty[slot]));
            if (++slot == STAGES) { slot = 0; phase ^= 1; }
          }
          if (ok) PAIR ? tc_commit_pair(smem_u32(&sh->acc_full[buf])) : tc_commit(smem_u32(&sh->acc_full[buf]));
          if (F::BUFS == 2) {
            acc_phase ^= buf;
            buf ^= 1;
          } else {
            acc_phase ^= 1;
          }
        }
      }
      // every MMA issued must have retired before TMEM is freed (bounded, ignoring abort)
      PAIR ? tc_commit_pair(smem_u32(&sh->mma_done)) : tc_commit(smem_u32(&sh->mma_done));
      uint32_t spins = 0;
      while (!mbar_try_wait(smem_u32(&sh->mma_done), 0) && ++spins < kSpinLimit) {}
      if (spins >= kSpinLimit) give_up(sh, status, 5);
    }
  } else if (warp < DRAIN0) {
    // ---------------------------------------------------------------- converters
    // A piece: 16 codes, two 16-byte chunks of the swizzled tile.  Eight lanes take four pieces of rows r and r ^ 1, whose chunks meet all
    // banks once; a thread takes every ROWS-th row of its piece's columns.
    constexpr int LANES = GROUP_WARPS * 32, MAX_PIECES = MAX_BN / CTAS / 16, ROWS = LANES / MAX_PIECES, P = BK / ROWS;
    const int group = (warp - CONV0) / GROUP_WARPS, t = threadIdx.x - (CONV0 + group * GROUP_WARPS) * 32;
    const int high = t >> 3, piece = (t & 3) | (high % (MAX_PIECES / 4)) * 4, row = high / (MAX_PIECES / 4) * 2 + ((t >> 2) & 1);
    const uint32_t dst0 = G_BYTES + (piece >> 2) * BLOCK_BYTES + row * 128 + ((((piece & 3) * 2) ^ (row & 7)) << 4);
    const bool mine = piece * 16 < own;
    const int blocks = (int)(p.pitch >> 5);
    const int64_t code_step = ROWS * p.pitch, code_stage = GROUPS * BK * p.pitch;
    const int exp_step = ROWS * blocks;
    const int64_t exp_stage = (int64_t)GROUPS * BK * blocks;
    uint32_t slot = group, phase = 0;
    int before = 0;                                  // stages of earlier items, modulo the groups
    bool ok = true;
    for (int w = w_first; w < n_items && ok; w += w_step) {
      const Item m = item_of(w, p);
      const int col = m.kt * p.bn + rank * own + piece * 16;
      const bool there = mine && col < p.pitch;
      int kb = m.kb0 + (group + GROUPS - before) % GROUPS;
      before = (before + m.kb1 - m.kb0) % GROUPS;
      const int64_t r0 = (int64_t)kb * BK + row;
      const uint8_t* codes = p.codes + r0 * p.pitch + col;
      const uint8_t* exps = p.exps + r0 * blocks + (col >> 5);
      for (; kb < m.kb1; kb += GROUPS) {
        uint4 code[P];
        uint32_t ex[P];
        if (there && (kb + 1) * (int64_t)BK <= p.rows) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            code[i] = *reinterpret_cast<const uint4*>(codes + i * code_step);
            ex[i] = exps[i * exp_step];
          }
        } else {                                     // the last stage's rows end, or columns past the codes
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const bool live = there && (int64_t)kb * BK + row + i * ROWS < p.rows;
            code[i] = live ? *reinterpret_cast<const uint4*>(codes + i * code_step) : make_uint4(0, 0, 0, 0);
            ex[i] = live ? exps[i * exp_step] : 0;
          }
        }
        codes += code_stage;
        exps += exp_stage;
        if (!mbar_wait_warp(smem_u32(&sh->empty[slot]), phase ^ 1, abort)) {
          if (lane == 0) give_up(sh, status, 6);
          ok = false;
          break;
        }
        if (mine) {
          uint8_t* to = tiles_ptr + slot * STAGE_BYTES + dst0;
          uint8_t* to2 = tiles_ptr + slot * STAGE_BYTES + (dst0 ^ 16u);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            uint32_t o[8];
            convert16<TG, KIND>(code[i], ex[i], o);
            *reinterpret_cast<uint4*>(to + i * (ROWS * 128)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(to2 + i * (ROWS * 128)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        // one warp's arrival also says that the CTA's part of g has landed
        if ((warp - CONV0) % GROUP_WARPS == 0 && !mbar_wait_warp(smem_u32(&sh->full_g[slot]), phase, abort)) {
          if (lane == 0) give_up(sh, status, 7);
          ok = false;
          break;
        }
        if (lane == 0) arrive_leader(&sh->full_x[slot]);
        if ((slot += GROUPS) >= STAGES) { slot -= STAGES; phase ^= 1; }
      }
    }
  } else if (warp < SUM0) {
    // ---------------------------------------------------------------- drain
    const int quad = warp & 3, half = (warp - DRAIN0) >> 2;      // TMEM lane quadrant this warp may read; which accumulator
    uint32_t chains = 0;
    bool ok = true;
    for (int w = w_first; w < n_items && ok; w += w_step) {
      const Item m = item_of(w, p);
      float* part = p.parts + (((int64_t)(m.nt * p.k_tiles + m.kt) * p.splits + m.split) * (4 * CTAS * MH) + (rank * MH + half) * 4 + quad) * (p.bn * 32) + lane * 4;
      for (int kb = m.kb0; kb < m.kb1; kb += kb == m.kb0 ? first_chain<TG>(w) : chain_of<TG>(), ++chains) {
        const int buf = F::BUFS == 2 ? chains & 1 : 0;
        if (!mbar_wait_warp(smem_u32(&sh->acc_full[buf]), (F::BUFS == 2 ? chains >> 1 : chains) & 1, abort)) {
          if (lane == 0) give_up(sh, status, 8);
          ok = false;
          break;
        }
        tc_fence_after();
        const bool first = kb == m.kb0;
        // Four columns of 32 rows are 512 bytes of the workspace.  Later chains are added where they lie: the only additions to an element come
        // from this thread, in order, so their sum is the same every time, and nothing waits for them (loaded, added and stored the drain took
        // longer than a chain).
        for (int c = 0; c < p.bn; c += 32) {
          uint32_t r[32];
          tmem_ld32(tmem_base + ((uint32_t)(quad * 32) << 16) + (buf + half) * MAX_BN + c, r);
          tmem_wait_ld();
          float* out = part + c * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            if (first) *reinterpret_cast<uint4*>(out + j * 32) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            else
              asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(out + j * 32), "f"(__uint_as_float(r[j])),
                           "f"(__uint_as_float(r[j + 1])), "f"(__uint_as_float(r[j + 2])), "f"(__uint_as_float(r[j + 3]))
                           : "memory");
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader(&sh->acc_empty[buf]);
      }
    }
  } else if (p.bias_parts) {
    // ---------------------------------------------------------------- column sums of g
    constexpr int SG = F::SUM_GROUPS, LANES = F::SUM_WARPS * 32 / SG, CHUNKS = F::CHUNKS;      // a group takes every SG-th stage
    const int t = threadIdx.x - SUM0 * 32, group = t / LANES;
    const int chunk = t % CHUNKS, first = (t % LANES) / CHUNKS;        // eight columns, every (LANES / CHUNKS)-th row: a partial sum of its own
    uint32_t s = 0, phase = 0, turn = 0;
    bool ok = true;
    for (int w = w_first; w < n_items && ok; w += w_step) {
      const Item m = item_of(w, p);
      float acc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      for (int kb = m.kb0; kb < m.kb1; ++kb) {
        if (turn == group) {
          if (!mbar_wait_warp(smem_u32(&sh->full_g[s]), phase, abort)) {
            if (lane == 0) give_up(sh, status, 9);
            ok = false;
            break;
          }
          if (m.kt == 0) {
            const uint8_t* blk = tiles_ptr + s * STAGE_BYTES + (chunk >> 3) * BLOCK_BYTES;
#pragma unroll 8
            for (int r = first; r < BK; r += LANES / CHUNKS) {
              const uint4 v = *reinterpret_cast<const uint4*>(blk + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
              add_pair<TG>(v.x, acc[0], acc[1]);
              add_pair<TG>(v.y, acc[2], acc[3]);
              add_pair<TG>(v.z, acc[4], acc[5]);
              add_pair<TG>(v.w, acc[6], acc[7]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->empty[s]));
        }
        if (++turn == SG) turn = 0;
        if (++s == STAGES) { s = 0; phase ^= 1; }
      }
      if (ok && m.kt == 0) {
        float4* out = reinterpret_cast<float4*>(p.bias_parts + (((int64_t)m.split * F::PHASES + t / CHUNKS) * p.n_tiles + m.nt) * (128 * CTAS * MH) + rank * (128 * MH) + chunk * 8);
        out[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        out[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();          // nothing is signalled to, or read from, a CTA that has left
  if (warp == 1) {
    tc_fence_after();
    PAIR ? tmem_dealloc_pair(tmem_base, TMEM_COLS) : tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Adds the partial tiles in the order of their rows: a block takes 32 x 32 of the weight (or, past those, 32 of the bias).
struct AddArgs {
  const float* parts;
  const float* bias_parts;
  float* gw;
  float* gb;
  int64_t ldw;
  int n, k, bn, n_tiles, k_tiles, splits, tile_n, phases;      // tile_n: columns of g of a tile; phases: partial column sums of a split
  int64_t patches;
};
__global__ void __launch_bounds__(256) wgrad8_add_kernel(AddArgs p) {
  pdl_begin();
  __shared__ float patch[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= p.patches) {             // 32 columns of g: a warp takes every eighth partial sum, then the warps' sums in order
    const int c = (int)(blockIdx.x - p.patches) * 32 + lane, width = p.n_tiles * p.tile_n;
    float sum = 0.f;
    if (c < p.n) {
#pragma unroll 8
      for (int s = warp; s < p.splits * p.phases; s += 8) sum += p.bias_parts[(int64_t)s * width + c];
    }
    patch[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.n) {
#pragma unroll
      for (int w = 1; w < 8; ++w) sum += patch[w][lane];
      p.gb[c] = sum;
    }
    return;
  }
  const int chunks = p.bn / 32, blocks = p.tile_n / 32;
  int64_t i = blockIdx.x;
  const int chunk = (int)(i % chunks);
  i /= chunks;
  const int blk = (int)(i % blocks), tile = (int)(i / blocks);
  const int64_t slot = (int64_t)blocks * p.bn * 32;
  // thread: row `lane` of four columns (bn is a multiple of 32)
  const float4* from = reinterpret_cast<const float4*>(p.parts + (int64_t)tile * p.splits * slot + ((int64_t)blk * p.bn + chunk * 32) * 32 + warp * 128) + lane;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < p.splits; ++s) {
    const float4 v = from[s * (slot / 4)];
    sum.x += v.x;
    sum.y += v.y;
    sum.z += v.z;
    sum.w += v.w;
  }
  patch[warp * 4][lane] = sum.x;
  patch[warp * 4 + 1][lane] = sum.y;
  patch[warp * 4 + 2][lane] = sum.z;
  patch[warp * 4 + 3][lane] = sum.w;
  __syncthreads();
  const int nt = tile / p.k_tiles, kt = tile % p.k_tiles;
  const int col = kt * p.bn + chunk * 32 + lane;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = nt * p.tile_n + blk * 32 + warp + 8 * j;
    if (row < p.n && col < p.k) p.gw[(int64_t)row * p.ldw + col] = patch[lane][warp + 8 * j];
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
  int ctas, mh, bn, n_tiles, k_tiles, splits, k_blocks, phases;
  bool copy;
  int tile_n() const { return 128 * ctas * mh; }
  int64_t copy_bytes, parts_bytes, bias_bytes;
};
Plan plan_of(int64_t rows, int n, int k, bool copy) {
  Plan best{};
  best.k_blocks = (int)((rows + BK - 1) / BK);
  best.copy = copy;
  const int sms = sm_count();
  double cost = 1e30;
  for (int form = 0; form < 3; ++form)
    for (int most = 64; most <= MAX_BN; most *= 2) {
      const int ctas = form == 0 ? 1 : 2, mh = form == 2 ? 2 : 1;
      const int k_tiles = (k + most - 1) / most, bn = (int)round_up((k + k_tiles - 1) / k_tiles, 32 * ctas);
      const int n_tiles = (n + 128 * ctas * mh - 1) / (128 * ctas * mh), units = sms / ctas;
      const int64_t tiles = (int64_t)n_tiles * k_tiles;
      if (tiles > 1 << 20) continue;
      // cycles of a stage and of a drain that nothing hides (an item's last one; with one set of accumulators every one); bytes of partial tiles, all SMs.
      // It ranks forms and splits and does not foretell times: 100,003 x 1,000 x 513 comes out at 77 us (measured 181), 475,136 x 1,024 x 256 at 150 (259 to 288).  Drains
      // are counted by bf16's chains for either type, fewer than fp16 has: with fp16's own 44 of 2,000 drawn sizes take another form, and of 20 of those 5 were 2 to 13 % faster
      // for it and 12 slower (73,077 x 280 x 1,711: 163 -> 290 us), since the stages' costs are off by more than the drains.
      const double stage = fmax((form == 0 ? 4.0 : form == 1 ? 3.1 : 4.6) * bn, form == 2 ? 700.0 : 450.0), drain = 2000 + 8.0 * mh * bn;
      // pieces of the rows: as fill one or more waves of SMs, or stages of some length each
      for (int i = 0; i < 10; ++i) {
        int64_t splits = i < 4 ? (i + 1) * (int64_t)units / tiles : best.k_blocks >> (i - 4);
        splits = splits < 1 ? 1 : splits > best.k_blocks ? best.k_blocks : splits;
        if (splits > 2 * sms) continue;
        const double waves = (double)((tiles * splits + units - 1) / units), per = (double)((best.k_blocks + splits - 1) / splits);
        const double c = waves * (per * stage + (mh == 2 ? drain * ceil(per / kChain) : 0.0)) + drain + (double)tiles * splits * 128 * ctas * mh * bn * 4 / 5000.0;
        if (c < cost) {
          cost = c;
          best.ctas = ctas; best.mh = mh; best.bn = bn; best.n_tiles = n_tiles; best.k_tiles = k_tiles; best.splits = (int)splits;
        }
      }
    }
  best.phases = best.ctas == 1 ? Form<1, 1>::PHASES : best.mh == 1 ? Form<2, 1>::PHASES : Form<2, 2>::PHASES;
  best.copy_bytes = copy ? round_up(rows * round_up(n, 8) * 2, 256) : 0;
  best.parts_bytes = round_up((int64_t)best.n_tiles * best.k_tiles * best.splits * best.tile_n() * best.bn * 4, 256);
  best.bias_bytes = round_up((int64_t)best.splits * best.phases * best.n_tiles * best.tile_n() * 4, 256);
  return best;
}

template <typename TG, int KIND, int CTAS, int MH>
int launch(const CUtensorMap& tm, const Args& p, int* status, cudaStream_t stream) {
  using F = Form<CTAS, MH>;
  static DeviceOnce once;
  const int rc = once.run("wgrad8_kernel set-up", [] {
    return cudaFuncSetAttribute(wgrad8_kernel<TG, KIND, CTAS, MH>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
  });
  if (rc != BSRL_OK) return rc;
  const int items = p.n_tiles * p.k_tiles * p.splits, units = sm_count() / CTAS, grid = (items < units ? items : units) * CTAS;
  launch_kernel<CTAS>(wgrad8_kernel<TG, KIND, CTAS, MH>, grid, F::THREADS, F::SMEM, stream, tm, p, status);
  BSRL_LAUNCH_OK("wgrad8_kernel");
  return BSRL_OK;
}
template <typename TG, int KIND>
int launch(const Plan& pl, const CUtensorMap& tm, const Args& p, int* status, cudaStream_t stream) {
  return pl.ctas == 1 ? launch<TG, KIND, 1, 1>(tm, p, status, stream)
         : pl.mh == 1 ? launch<TG, KIND, 2, 1>(tm, p, status, stream) : launch<TG, KIND, 2, 2>(tm, p, status, stream);
}
bool needs_copy(const void* g, int64_t ldg) { return !aligned16(g) || ldg % 8 != 0; }
}  // namespace

int64_t wgrad8_workspace(int64_t rows, int n, int k, bool aligned) {
  const Plan pl = plan_of(rows, n, k, !aligned);
  return pl.copy_bytes + pl.parts_bytes + pl.bias_bytes;
}

void wgrad8_plan(int64_t rows, int n, int k, int32_t (&plan)[3]) {
  const Plan pl = plan_of(rows, n, k, false);
  plan[0] = pl.tile_n();
  plan[1] = pl.bn;
  plan[2] = pl.splits;
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
  const Args p{codes, exps, rows, pitch_of(k), pl.bn, pl.n_tiles, pl.k_tiles, pl.splits, pl.k_blocks, parts, bias_parts};
  int* status = device_status_ptr();
  if (!status) return BSRL_ERR_CUDA;
  const int rc = g_dtype == BSRL_F16 ? (kind == kInt8 ? launch<__half, kInt8>(pl, tm, p, status, stream) : launch<__half, kE4m3>(pl, tm, p, status, stream))
                                     : (kind == kInt8 ? launch<__nv_bfloat16, kInt8>(pl, tm, p, status, stream)
                                                      : launch<__nv_bfloat16, kE4m3>(pl, tm, p, status, stream));
  if (rc != BSRL_OK) return rc;
  AddArgs a{parts, bias_parts, gw, gb, ldw, n, k, pl.bn, pl.n_tiles, pl.k_tiles, pl.splits, pl.tile_n(), pl.phases, 0};
  a.patches = (int64_t)pl.n_tiles * pl.k_tiles * (pl.tile_n() / 32) * (pl.bn / 32);
  PdlScope overlap;
  pdl_enable();
  launch_kernel(wgrad8_add_kernel, (unsigned)(a.patches + (gb ? (n + 31) / 32 : 0)), 256, 0, stream, a);
  BSRL_LAUNCH_OK("wgrad8_add_kernel");
  return BSRL_OK;
}

}  // namespace bsrl
