// The 8-bit product where the MMAs are what bounds it (prompts): CTA pairs on tiles of 256 tokens x up to 256 output channels.
//
//   D[256 tokens, N channels] += C[256, 128 k] . Q[N, 128 k]^T      int8 operands, int32 sums, cta_group::2 MMAs
//
// Each CTA of a pair brings 128 tokens' codes and half of the tile's channels a step (TMA, 128-byte swizzle); the MMAs, which one CTA
// issues, read both CTAs' shared memory.  The accumulator's lanes are the tokens; two accumulators take turns, so the epilogue of a tile
// runs under the next tile's MMAs.
//   The correction alpha r L^T cannot join a sum of integers.  So a corrected tile's sums are turned into fp32 where they lie: the
// epilogue reads them, scales them (by s_t w_o / alpha, and bias / alpha) and puts them back into tensor memory, fp16 MMAs add r L^T to
// them, and the epilogue reads the result once more and multiplies by alpha.  That detour takes no time from the MMAs: the correction's steps
// of a tile are put into the middle of the NEXT tile's steps, when its sums have long been converted, and its accumulator is free again
// before the tile after that begins.
//   warps 0 and 3  copies (a thread each)     warp 1  MMAs (CTA 0's)     warp 2  tensor memory     warps 4-11  epilogue, two for each 32 lanes
//   What bounds it: 256 channels, the MMAs (512 clocks a step) and over longer runs the 1 kW limit - 4096 tokens, 5120 -> 13824: 173 us
// (3350 TOP/s) in runs of milliseconds, 203 (2860) back to back; 2048 tokens, 5120 -> 27648: 180, with a correction of rank 128 195.
// Narrower tiles: the copies, 0.21 to 0.24 us a step whatever the width; a chain of 5.5 us around all steps.
// Every wait is bounded; on expiry a status word is set and the CTAs drain.
#include <cuda_bf16.h>

#include <algorithm>

#include "tcgen05.cuh"
#include "w8a8.h"

namespace glowq {

namespace {

__device__ uint32_t g_w8a8_pair_status;   // nonzero once a wait of this file's kernel has run out on the device

constexpr int kRows = 128;                 // tokens of a CTA
constexpr int kAStage = kRows * 128;
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kTmemCols = 512;
constexpr int kMaxStages = 8;
constexpr int kOStage = 2048;              // output stage of an epilogue warp: 32 tokens x 64 bytes
constexpr int kSmemMax = 227 * 1024 - 512;
constexpr unsigned kDrainSpin = 1u << 18;

struct PairParams {
  const float *scales, *weight_scales, *bias;
  void* out;
  long long out_stride;
  int M, OC, N, nk, nr, insert;     // insert: steps of a tile in front of the correction's steps of the tile before
  int n_x, n_y, band, tiles, stages;
  int out_dtype, out_tma;
  float alpha, inv_alpha;
};
struct alignas(64) PairMaps {
  CUtensorMap a, b, r, l, out;
};

// Barriers in the first KB of shared memory.
constexpr uint32_t kFull = 0;               // [kMaxStages] CTA 0: both CTAs' copies have landed
constexpr uint32_t kEmpty = 64;             // [kMaxStages] each CTA: the step's MMAs are done
constexpr uint32_t kAccFull = 128;          // [2] each CTA: a tile's sums
constexpr uint32_t kAccEmpty = 144;         // [2] CTA 0: the epilogue warps of both CTAs have read the result
constexpr uint32_t kConverted = 160;        // [2] CTA 0: they have put fp32 sums in the place of the integers
constexpr uint32_t kCorrected = 176;        // [2] each CTA: the correction is added
constexpr uint32_t kFin = 192;              // CTA 0: all MMAs are done

#define GLOWQ_PAIR_STEP(KIND)                                                                                                       \
  asm volatile(                                                                                                                     \
      "{\n\t.reg .pred e, p, t;\n\t.reg .b32 x<4>, y<4>;\n\t.reg .b64 a<4>, b<4>;\n\t.reg .b16 m;\n\t"                              \
      "setp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"                                            \
      "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\tadd.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\t"              \
      "add.u32 y3, %2, 6;\n\tmov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"  \
      "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\tmov.b16 m, 3;\n\t"       \
      "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a0, b0, %4, p;\n\t"                                                         \
      "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a1, b1, %4, t;\n\t"                                                         \
      "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a2, b2, %4, t;\n\t"                                                         \
      "@e tcgen05.mma.cta_group::2.kind::" KIND " [%0], a3, b3, %4, t;\n\t"                                                         \
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], m;\n\t}" ::"r"(d),         \
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(bar)                                                          \
      : "memory")
__device__ __forceinline__ void step_i8(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate,
                                        uint32_t bar) {
  GLOWQ_PAIR_STEP("i8");
}
__device__ __forceinline__ void step_f16(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate,
                                         uint32_t bar) {
  GLOWQ_PAIR_STEP("f16");
}
__device__ __forceinline__ void commit_both(uint32_t bar) {   // both CTAs' barriers, once all MMAs issued so far are done
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar)
      : "memory");
}
// A copy into this CTA whose bytes count on a barrier of CTA 0.
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(cluster_bar)
      : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
// The epilogue warps of a CTA go on together or leave together.
__device__ __forceinline__ bool epi_vote(bool ok) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"(static_cast<uint32_t>(ok))
               : "memory");
  return r != 0;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    w8a8_pair_kernel(const __grid_constant__ PairParams p, const __grid_constant__ PairMaps tm) {
  extern __shared__ unsigned char smem[];
  __shared__ int s_abort;
  __shared__ uint32_t s_tmem;
  __shared__ __align__(16) float2 s_cols[256];   // a tile's channels: scale and bias; read two at a time
  uint32_t* const status = &g_w8a8_pair_status;
  const int N = p.N, stages = p.stages;
  const uint32_t stage_bytes = kAStage + static_cast<uint32_t>(N) * 64;
  const uint32_t smem0 = (sm_u32(smem) + 1023u) & ~1023u, ring = smem0 + 1024, ostage = ring + stages * stage_bytes;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
  volatile int* const abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < stages; ++i) {
      g_mbar_init(smem0 + kFull + 8 * i, 1);
      g_mbar_init(smem0 + kEmpty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      g_mbar_init(smem0 + kAccFull + 8 * i, 1);
      g_mbar_init(smem0 + kCorrected + 8 * i, 1);
      g_mbar_init(smem0 + kAccEmpty + 8 * i, 2 * kEpiWarps);
      g_mbar_init(smem0 + kConverted + 8 * i, 2 * kEpiWarps);
    }
    g_mbar_init(smem0 + kFin, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  cluster_sync_all();

  // token tiles in bands; within a band, channel tile by channel tile
  const auto place = [&](int tile, int& m0, int& n0) {
    const int per = p.n_x * p.band, b = tile / per, rem = tile - b * per, rows = min(p.band, p.n_y - b * p.band);
    const int x = rem / rows, y = b * p.band + rem - x * rows;
    m0 = y * (2 * kRows);
    n0 = x * N;
  };
  const uint32_t full0 = map_to_cta(smem0 + kFull, 0);
  const int prologue = min(stages, p.nk);   // steps whose weights are asked for before the dependency wait
  if (threadIdx.x == 0) {
    int m0, n0;
    place(pair, m0, n0);
    for (int i = 0; i < prologue; ++i) {
      if (rank == 0) g_mbar_expect_tx(smem0 + kFull + 8 * i, 2 * stage_bytes);
      tma_pair(ring + i * stage_bytes + kAStage, &tm.b, i * 128, n0 + rank * (N >> 1), full0 + 8 * i);
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_u32(&s_tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync_all();   // both CTAs' tensor memory
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;

  if (warp == 0 || warp == 3) {
    // Copies: warp 0 the tokens' operand (codes, r) and the announcement of a step's bytes, warp 3 the channels' (weights, L).  One thread
    // for both took 955 clocks a step, whatever the tile's width; the MMAs of 256 channels take 512.
    if (lane == 0) {
      const bool tokens = warp == 0;
      const CUtensorMap *const main_map = tokens ? &tm.a : &tm.b, *const corr_map = tokens ? &tm.r : &tm.l;
      const int mine = rank * (tokens ? kRows : N >> 1), ahead = tokens ? 0 : prologue;   // (of the weights' first steps are under way)
      const bool announce = tokens && rank == 0;
      uint32_t st = 0, ph = 1, bar = smem0 + kEmpty, full = full0, dst = ring + (tokens ? 0 : kAStage);
      const uint32_t first = dst;
      int issued = 0, before_at = 0;
      bool ok = true;
      for (int tile = pair, i = 0; ok; tile += pairs, ++i) {
        const bool valid = tile < p.tiles, before = i > 0 && p.nr > 0 && tile - pairs < p.tiles;
        if (!valid && !before) break;
        int m0 = 0, n0 = 0;
        if (valid) place(tile, m0, n0);
        const int at = (tokens ? m0 : n0) + mine;
        const int nk = valid ? p.nk : 0, ins = valid ? p.insert : 0, nr = before ? p.nr : 0;
        for (int s = 0; s < nk + nr; ++s, ++issued) {
          const bool corr = s >= ins && s < ins + nr;
          if (issued >= ahead) {
            if (!(ok = g_mbar_wait(bar, ph, abort_flag, status))) break;
            if (announce && issued >= prologue) g_mbar_expect_tx(smem0 + kFull + 8 * st, 2 * stage_bytes);
            tma_pair(dst, corr ? corr_map : main_map, corr ? (s - ins) * 64 : (s < ins ? s : s - nr) * 128, corr ? before_at : at, full);
          }
          dst += stage_bytes;
          bar += 8;
          full += 8;
          if (++st == static_cast<uint32_t>(stages)) {
            st = 0;
            ph ^= 1;
            dst = first;
            bar = smem0 + kEmpty;
            full = full0;
          }
        }
        before_at = at;
      }
      // the steps that were issued are consumed before the CTA leaves (or the wait for that runs out)
      for (int j = max(0, issued - stages); j < issued; ++j) {
        uint32_t spins = 0;
        while (!g_mbar_try_once(smem0 + kEmpty + 8 * (j % stages), (j / stages) & 1) && ++spins < kDrainSpin) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      // instruction descriptors: s32 sums of signed bytes, fp32 sums of fp16; K-major operands; 256 x N
      const uint32_t shape = (static_cast<uint32_t>(N) >> 3) << 17 | (2 * kRows >> 4) << 24;
      const uint32_t i8 = (2u << 4) | (1u << 7) | (1u << 10) | shape, f16 = (1u << 4) | shape;
      const uint64_t desc = smem_desc_sw128(ring);
      const uint32_t hi = static_cast<uint32_t>(desc >> 32), lo0 = static_cast<uint32_t>(desc), step16 = stage_bytes >> 4;
      uint32_t st = 0, ph = 0;
      bool ok = true;
      uint32_t ready = 0;
      for (int tile = pair, i = 0; ok; tile += pairs, ++i) {
        const bool valid = tile < p.tiles, before = i > 0 && p.nr > 0 && tile - pairs < p.tiles;
        if (!valid && !before) break;
        const uint32_t buf = i & 1, use = static_cast<uint32_t>(i) >> 1;
        const uint32_t pbuf = buf ^ 1, puse = static_cast<uint32_t>(i - 1) >> 1;
        const int nk = valid ? p.nk : 0, ins = valid ? p.insert : 0, nr = before ? p.nr : 0;
        if (valid) {
          if (!(ok = g_mbar_wait_warp<false>(smem0 + kAccEmpty + 8 * buf, (use & 1) ^ 1, abort_flag, status))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        const uint32_t d = tmem + buf * 256, dp = tmem + pbuf * 256;
        uint32_t acc = 0;
        for (int s = 0; s < nk + nr; ++s) {
          const bool corr = s >= ins && s < ins + nr;
          if (corr && s == ins) {
            if (!(ok = g_mbar_wait_warp<true>(smem0 + kConverted + 8 * pbuf, puse & 1, abort_flag, status))) break;
          }
          if (!__any_sync(0xffffffffu, ready) &&
              !(ok = g_mbar_wait_warp<true>(smem0 + kFull + 8 * st, ph, abort_flag, status)))
            break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a_lo = lo0 + st * step16, b_lo = a_lo + (kAStage >> 4), bar = smem0 + kEmpty + 8 * st;
          if (corr) {
            step_f16(dp, a_lo, b_lo, hi, f16, 1u, bar);
            if (s == ins + nr - 1) commit_both(smem0 + kCorrected + 8 * pbuf);
          } else {
            step_i8(d, a_lo, b_lo, hi, i8, acc, bar);
            acc = 1;
          }
          if (++st == static_cast<uint32_t>(stages)) {
            st = 0;
            ph ^= 1;
          }
          ready = g_mbar_test_elected(smem0 + kFull + 8 * st, ph);
        }
        if (ok && valid) commit_both(smem0 + kAccFull + 8 * buf);
      }
      asm volatile(
          "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
          "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem0 + kFin)
          : "memory");
      if (lane == 0) {
        uint32_t spins = 0;
        while (!g_mbar_try_once(smem0 + kFin, 0) && ++spins < kDrainSpin) {
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q = warp & 3, half = (warp - 4) >> 2;   // the 32 lanes that this warp reaches; its half of the columns
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t stage = ostage + (warp - 4) * kOStage, srow = stage + lane * 64, swz = (static_cast<uint32_t>(lane) >> 1) & 3u;
    const uint32_t empty0 = map_to_cta(smem0 + kAccEmpty, 0), converted0 = map_to_cta(smem0 + kConverted, 0);
    const int c0 = half * (N >> 1), c1 = c0 + (N >> 1);
    const bool corrected = p.nr > 0;
    const uint32_t cols0 = sm_u32(s_cols);
    bool ok = true;
    for (int tile = pair, i = 0; tile < p.tiles; tile += pairs, ++i) {
      int m0, n0;
      place(tile, m0, n0);
      const uint32_t buf = i & 1, use = static_cast<uint32_t>(i) >> 1, acc = tmem + lanes + buf * 256;
      const int row = m0 + rank * kRows + q * 32 + lane;
      const float s = row < p.M ? p.scales[row] : 0.f;
      // (all warps are through with the tile before: the vote after it was read for the last time)
      if (!epi_vote(ok)) break;
      {
        const int c = threadIdx.x - 128;
        if (c < N) {
          const bool in = n0 + c < p.OC;
          float w = in ? p.weight_scales[n0 + c] : 0.f, b = in && p.bias ? p.bias[n0 + c] : 0.f;
          s_cols[c] = corrected ? make_float2(w, b * p.inv_alpha) : make_float2(w, b);
        }
      }
      ok = __all_sync(0xffffffffu, g_mbar_wait(smem0 + kAccFull + 8 * buf, use & 1, abort_flag, status));
      if (!epi_vote(ok)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const auto scaled = [&](uint32_t (&v)[32], int c) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float4 w;
          asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w) : "r"(cols0 + (c + j) * 8));
          float a = static_cast<float>(static_cast<int>(v[j])) * s, b = static_cast<float>(static_cast<int>(v[j + 1])) * s;
          if (corrected) {
            a *= p.inv_alpha;
            b *= p.inv_alpha;
          }
          v[j] = __float_as_uint(fmaf(a, w.x, w.y));
          v[j + 1] = __float_as_uint(fmaf(b, w.z, w.w));
        }
      };
      if (corrected) {
        for (int c = c0; c < c1; c += 32) {
          uint32_t v[32];
          tmem_ld32(acc + c, v);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          scaled(v, c);
          tmem_st32(acc + c, v);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_cluster(converted0 + 8 * buf);
        ok = __all_sync(0xffffffffu, g_mbar_wait(smem0 + kCorrected + 8 * buf, use & 1, abort_flag, status));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (!ok) continue;   // (to the vote)
      }
      for (int c = c0; c < c1; c += 32) {
        uint32_t v[32];
        tmem_ld32(acc + c, v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (c + 32 >= c1) {   // the last of this warp's columns are in registers
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_cluster(empty0 + 8 * buf);
        }
        if (corrected) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * p.alpha);
        } else {
          scaled(v, c);
        }
        const int col = n0 + c;
        if (col >= p.OC) continue;
        if (p.out_dtype != GLOWQ_F32) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (p.out_dtype == GLOWQ_F16) {
              const __half2 h = __floats2half2_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
              v[j] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
              const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
              v[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
        }
        const int parts = p.out_dtype == GLOWQ_F32 ? 2 : 1, per = 32 / parts;   // 64 bytes of a row at a time
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (part >= parts) break;
          if (p.out_tma) {   // the copy that read this stage before is through with it
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(srow + ((static_cast<uint32_t>(j) ^ swz) << 4)),
                         "r"(v[16 * part + 4 * j]), "r"(v[16 * part + 4 * j + 1]), "r"(v[16 * part + 4 * j + 2]), "r"(v[16 * part + 4 * j + 3])
                         : "memory");
          const int pc = col + part * per;
          if (p.out_tma) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (pc < p.OC && m0 + rank * kRows + q * 32 < p.M)
                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&tm.out), "r"(pc),
                             "r"(m0 + rank * kRows + q * 32), "r"(stage)
                             : "memory");
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            // rows that the copy engine cannot write: a warp writes one row after the other
            __syncwarp();
            const int first = m0 + rank * kRows + q * 32, rows = min(32, p.M - first);
            for (int t = 0; t < rows; ++t) {
              const long long at = static_cast<long long>(first + t) * p.out_stride + pc;
              const uint32_t sw = (static_cast<uint32_t>(t) >> 1) & 3u;
              if (parts == 2) {
                if (lane < 16 && pc + lane < p.OC) {
                  uint32_t w;
                  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(stage + t * 64 + (((lane >> 2) ^ sw) << 4) + (lane & 3) * 4) : "memory");
                  static_cast<uint32_t*>(p.out)[at + lane] = w;
                }
              } else if (pc + lane < p.OC) {
                uint16_t w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(stage + t * 64 + (((lane >> 3) ^ sw) << 4) + (lane & 7) * 2) : "memory");
                static_cast<uint16_t*>(p.out)[at + lane] = w;
              }
            }
            __syncwarp();
          }
        }
      }
    }
    if (p.out_tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  cluster_sync_all();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

}  // namespace

cudaError_t w8a8_pair_status(uint32_t* out, cudaStream_t stream) { return take_status(g_w8a8_pair_status, out, stream); }

int w8a8_pair_forward(const glowq_w8a8_linear_t& g, int n, bool ahead, int sms, cudaStream_t stream) {
  const bool corrected = g.r_mode != GLOWQ_R_NONE;
  PairParams p{};
  p.scales = g.scales;
  p.weight_scales = g.weight_scales;
  p.bias = g.bias;
  p.out = g.out;
  p.out_stride = g.out_stride;
  p.out_dtype = g.out_dtype;
  p.M = g.M;
  p.OC = g.OC;
  p.N = n;
  p.nk = (g.K + 127) / 128;
  p.nr = corrected ? (g.rank + 63) / 64 : 0;
  p.insert = p.nk / 2;
  p.n_x = (g.OC + n - 1) / n;
  p.n_y = (g.M + 2 * kRows - 1) / (2 * kRows);
  p.band = std::min(p.n_y, 16);
  p.tiles = p.n_x * p.n_y;
  p.alpha = g.alpha;
  p.inv_alpha = corrected ? 1.f / g.alpha : 0.f;
  const int e = static_cast<int>(dtype_bytes(g.out_dtype));
  // (the copy engine writes whole 16-byte pieces, past the last channel too where that does not end one)
  p.out_tma = (static_cast<int64_t>(g.OC) * e) % 16 == 0 && (g.out_stride * e) % 16 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15u) == 0;
  const int stage = kAStage + n * 64, room = kSmemMax - 2048 - kEpiWarps * kOStage - 2048;
  p.stages = std::min(kMaxStages, room / stage);
  PairMaps tm;
  int rc = tensor_map_2d_ex(&tm.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.codes, g.K, g.M, g.code_stride, 128, kRows, 1);
  if (!rc) rc = tensor_map_2d_ex(&tm.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.weight, g.K, g.OC, g.weight_stride, 128, n / 2, 1);
  if (!rc && corrected) {
    rc = tensor_map_2d_ex(&tm.r, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, g.r, g.rank, g.M, 2 * g.r_stride, 64, kRows, 1);
    if (!rc) rc = tensor_map_2d_ex(&tm.l, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, g.L, g.rank, g.OC, 2 * g.L_stride, 64, n / 2, 1);
  }
  if (!rc && p.out_tma)
    rc = tensor_map_2d_ex(&tm.out,
                          g.out_dtype == GLOWQ_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : g.out_dtype == GLOWQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          g.out, g.OC, g.M, g.out_stride * e, 64 / e, 32, 3);
  if (rc) return rc;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(w8a8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - 3072);
    if (err != cudaSuccess) return note_cuda_error(err);
    attr_done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(p.tiles, sms / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 2048 + p.stages * stage + kEpiWarps * kOStage;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ahead && use_pdl() ? 1 : 0;
  return note_cuda_error(cudaLaunchKernelEx(&cfg, w8a8_pair_kernel, p, tm));
}

}  // namespace glowq
