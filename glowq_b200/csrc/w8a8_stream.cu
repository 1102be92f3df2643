// The 8-bit product where the weights are what is read: few tokens, one CTA or one cluster of CTAs per 128 output channels.
//
//   D[128 channels, N tokens] += Q[128, 128 k] . C[N, 128 k]^T          int8 operands, int32 sums (tcgen05.mma kind::i8)
//   F[128 channels, N tokens] += L[128, 64 j] . r[N, 64 j]^T            the correction's steps, fp16 operands, fp32 sums
//   y = s_t w_o D + alpha F + bias
//
// and, with fp16 operands in the first place, r = x . R^T (channels: the rows of R).
//   Bound by HBM: every weight is read once.  TMA brings 128 rows x 128 bytes of weights and N tokens' 128 bytes a step into a ring
// of 200 KB (or two CTAs to an SM, of 100 KB each), and tcgen05.mma reads both from there: no weight passes through registers.  The weights do not hang
// on the kernels before, so the ring is filled before the dependency wait: a launch's first 30 MB of weights arrive while the codes are
// still being made.  The steps of a tile are shared out over the CTAs of a cluster (up to 8) so that all SMs are
// at work whatever the number of channels; their sums meet in shared memory (each CTA reads its share of the others' blocks),
// integers in any order, the correction's fp32 sums in the order of the CTAs: no workspace, no counters, the same bits every time.
//   warps 0 and 6  copies (a thread each)    warp 1  tensor memory, MMAs    warps 2-5  sums to shared memory; all: scales, bias, output
//   One token, 2048 -> 2048 4.5 us, 5120 -> 5120 6.8 (3.9 TB/s), 5120 -> 13824 13.1 (5.4); 16 tokens, 5120 -> 27648 25.2 (5.6); 77 tokens,
// 18944 -> 3584 14.1 (4.9): a chain of some 4 us - launch, first weights, a cluster's sum - and the copy rate.
// Tensor memory is taken after the dependency wait: a CTA that held it while it waits could keep a kernel in front from taking its own.
#include <cuda_bf16.h>

#include <algorithm>

#include "tcgen05.cuh"
#include "w8a8.h"

namespace glowq {

namespace {

__device__ uint32_t g_w8a8_status;   // nonzero once a wait of one of this file's kernels has run out on the device

constexpr int kRows = 128;
constexpr int kAStage = kRows * 128;
constexpr int kThreads = 224;
// Dynamic shared memory at most: of a launch whose CTAs have an SM each, and of one that has more of them, two to an SM.
constexpr int kSmemOne = 220 * 1024, kSmemTwo = 113 * 1024;
constexpr int kMaxStages = 12;
constexpr int kMaxSplit = 16;          // CTAs of a cluster (above 8 for r alone)
constexpr unsigned kDrainSpin = 1u << 18;

struct StreamParams {
  const float *scales, *weight_scales, *bias;
  void* out;
  long long out_stride;
  int M, OC, out_dtype, vec;     // vec: four outputs are stored together
  int nk, nr, split;             // steps of the product and of the correction; CTAs of a cluster
  int early;                     // the launch behind this one may begin at once
  int beside;                    // this launch may run beside the one in front, and ends after it
  float alpha;
};
struct alignas(64) StreamMaps {
  CUtensorMap a, b, l, r;
};

template <int N, bool TWO> constexpr int stages_of() { return std::min(kMaxStages, ((TWO ? kSmemTwo : kSmemOne) - 2048) / (kAStage + N * 128)); }
template <int N, bool TWO> constexpr int smem_of() { return 2048 + stages_of<N, TWO>() * (kAStage + N * 128); }

// The four MMAs of a step (32 bytes of K each) and the commit that gives its stage back, by one elected lane of a converged warp.
#define GLOWQ_STREAM_STEP(KIND)                                                                                                     \
  asm volatile(                                                                                                                     \
      "{\n\t.reg .pred e, p, t;\n\t.reg .b32 x<4>, y<4>;\n\t.reg .b64 a<4>, b<4>;\n\t"                                              \
      "setp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"                                            \
      "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\tadd.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\t"              \
      "add.u32 y3, %2, 6;\n\tmov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"  \
      "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\t"                        \
      "@e tcgen05.mma.cta_group::1.kind::" KIND " [%0], a0, b0, %4, p;\n\t"                                                         \
      "@e tcgen05.mma.cta_group::1.kind::" KIND " [%0], a1, b1, %4, t;\n\t"                                                         \
      "@e tcgen05.mma.cta_group::1.kind::" KIND " [%0], a2, b2, %4, t;\n\t"                                                         \
      "@e tcgen05.mma.cta_group::1.kind::" KIND " [%0], a3, b3, %4, t;\n\t"                                                         \
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}" ::"r"(d),                               \
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(bar)                                                          \
      : "memory")
__device__ __forceinline__ void step_i8(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate,
                                        uint32_t bar) {
  GLOWQ_STREAM_STEP("i8");
}
__device__ __forceinline__ void step_f16(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate,
                                         uint32_t bar) {
  GLOWQ_STREAM_STEP("f16");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ uint4 lds_cluster_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Four outputs of one token.
__device__ __forceinline__ void store4(const StreamParams& p, int token, int col, const float (&v)[4]) {
  const long long at = static_cast<long long>(token) * p.out_stride + col;
  if (p.out_dtype == GLOWQ_F32) {
    float* const o = static_cast<float*>(p.out) + at;
    if (p.vec && col + 4 <= p.OC) {
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.OC) o[j] = v[j];
    }
    return;
  }
  uint16_t h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    h[j] = p.out_dtype == GLOWQ_F16 ? __half_as_ushort(__float2half_rn(v[j])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[j]));
  uint16_t* const o = static_cast<uint16_t*>(p.out) + at;
  if (p.vec && col + 4 <= p.OC) {
    *reinterpret_cast<uint2*>(o) = make_uint2(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < p.OC) o[j] = h[j];
  }
}

// N tokens a tile; F16: fp16 operands and fp32 sums (r = x . R^T, which has neither scales nor a correction).
template <int N, bool F16, bool TWO>
__global__ void __launch_bounds__(kThreads, TWO ? 2 : 1) stream_kernel(const __grid_constant__ StreamParams p, const __grid_constant__ StreamMaps tm) {
  constexpr int kStages = stages_of<N, TWO>(), kStage = kAStage + N * 128;
  constexpr uint32_t kFull = 0, kEmpty = 8 * kMaxStages, kAcc = 16 * kMaxStages;
  static_assert(kAcc + 8 <= 1024, "barriers");
  extern __shared__ unsigned char smem[];
  __shared__ int s_abort;
  __shared__ uint32_t s_tmem;
  const uint32_t smem0 = (sm_u32(smem) + 1023u) & ~1023u, ring = smem0 + 1024;
  uint32_t* const status = &g_w8a8_status;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int split = p.split, z = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / split * kRows, m0 = static_cast<int>(blockIdx.y) * N;
  const int total = p.nk + p.nr;
  const auto first_step = [&](int c) { return total * c / split; };   // (steps of a CTA of the cluster)
  const int it0 = first_step(z), it1 = first_step(z + 1);
  volatile int* const abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) {
      g_mbar_init(smem0 + kFull + 8 * i, 1);
      g_mbar_init(smem0 + kEmpty + 8 * i, 1);
    }
    g_mbar_init(smem0 + kAcc, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (p.early && threadIdx.x == 64) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // The first steps' weights are asked for before the dependency wait.
  const int ahead = min(kStages, it1 - it0);
  const auto load_a = [&](int it, uint32_t bar, uint32_t dst) {
    g_mbar_expect_tx(bar, kStage);
    if (it < p.nk)
      g_tma_2d(dst, &tm.a, it * (F16 ? 64 : 128), n0, bar);
    else
      g_tma_2d(dst, &tm.l, (it - p.nk) * 64, n0, bar);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < ahead; ++i) load_a(it0 + i, smem0 + kFull + 8 * i, ring + i * kStage);
  if (!p.beside) asm volatile("griddepcontrol.wait;" ::: "memory");
  // (a constant: with a number of columns that the launch chose, an SM held one CTA instead of two)
  constexpr uint32_t columns = F16 ? (N < 32 ? 32 : N) : 2 * N;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_u32(&s_tmem)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (threadIdx.x == 64) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;

  // this thread's first four outputs: what they are scaled by is on its way while the sums are made
  const int tokens = min(N, p.M - m0), quads = tokens * (kRows / 4);
  const int q0 = quads * z / split, q1 = quads * (z + 1) / split;
  struct Scales {
    float s, w[4], b[4];
  };
  const auto scales_of = [&](int q) {
    Scales c;
    const int col = n0 + 4 * (q % (kRows / 4));
    c.s = p.scales[m0 + q / (kRows / 4)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c.w[j] = col + j < p.OC ? p.weight_scales[col + j] : 0.f;
      c.b[j] = p.bias && col + j < p.OC ? p.bias[col + j] : 0.f;
    }
    return c;
  };
  const int q_mine = q0 + static_cast<int>(threadIdx.x);
  Scales mine{};
  if (!F16 && q_mine < q1) mine = scales_of(q_mine);

  if (warp == 0 || warp == 6) {
    // Copies: warp 0 the weights (and L) and the announcement of a step's bytes, warp 6 the tokens (and r).  One thread for both took a
    // thousand clocks a step: 43 GB/s of weights.
    if (lane == 0) {
      const bool weights = warp == 0;
      uint32_t stage = weights && ahead == kStages ? 0u : weights ? static_cast<uint32_t>(ahead) : 0u, ph = weights && ahead == kStages ? 0u : 1u;
      for (int it = it0 + (weights ? ahead : 0); it < it1; ++it) {
        const uint32_t bar = smem0 + kFull + 8 * stage, dst = ring + stage * kStage;
        if (!g_mbar_wait(smem0 + kEmpty + 8 * stage, ph, abort_flag, status)) break;
        if (weights)
          load_a(it, bar, dst);
        else
          g_tma_2d(dst + kAStage, it < p.nk ? &tm.b : &tm.r, it < p.nk ? it * (F16 ? 64 : 128) : (it - p.nk) * 64, m0, bar);
        if (++stage == kStages) {
          stage = 0;
          ph ^= 1;
        }
      }
      // the copies have landed before the CTA goes on (or the wait for them runs out)
      if (weights)
        for (int j = max(0, it1 - it0 - kStages); j < it1 - it0; ++j) {
          uint32_t spins = 0;
          while (!g_mbar_try_once(smem0 + kFull + 8 * (j % kStages), (j / kStages) & 1) && ++spins < kDrainSpin) {
          }
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    // instruction descriptors: sums s32 of signed bytes, or fp32 of fp16; K-major operands; 128 x N
    constexpr uint32_t shape = (static_cast<uint32_t>(N) >> 3) << 17 | (kRows >> 4) << 24;
    constexpr uint32_t i8 = (2u << 4) | (1u << 7) | (1u << 10) | shape, f16 = (1u << 4) | shape;
    const uint64_t desc = smem_desc_sw128(ring);
    const uint32_t hi = static_cast<uint32_t>(desc >> 32), lo = static_cast<uint32_t>(desc);
    bool ok = true;
    for (int it = it0; it < it1 && ok; ++it) {
      const int j = it - it0, stage = j % kStages;
      if (!(ok = g_mbar_wait_warp<false>(smem0 + kFull + 8 * stage, (j / kStages) & 1, abort_flag, status))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t a_lo = lo + stage * (kStage >> 4), b_lo = a_lo + (kAStage >> 4), bar = smem0 + kEmpty + 8 * stage;
      if (F16)
        step_f16(tmem, a_lo, b_lo, hi, f16, it > it0, bar);
      else if (it < p.nk)
        step_i8(tmem, a_lo, b_lo, hi, i8, it > it0, bar);
      else
        step_f16(tmem + N, a_lo, b_lo, hi, f16, it > max(it0, p.nk), bar);
    }
    commit(smem0 + kAcc);
    __syncwarp();
  }
  // sums of a CTA: [tokens][128] of the product, then of the correction, where the ring was
  const uint32_t sums = ring;
  if (warp >= 2 && warp < 6) {
    const bool ok = __all_sync(0xffffffffu, g_mbar_wait(smem0 + kAcc, 0, abort_flag, status));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (ok) {
      const int q = warp & 3;   // the tensor-memory lanes that this warp reaches
      const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16, row = static_cast<uint32_t>(q * 32 + lane);
#pragma unroll
      for (int part = 0; part < (F16 ? 1 : 2); ++part) {
        if (part == 0 ? it0 >= p.nk : it1 <= p.nk) continue;
        for (int t = 0; t < tokens; t += 16) {
          uint32_t v[16];
          tmem_ld16(tmem + lanes + part * N + t, v);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 16; ++j)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(sums + ((part * N + t + j) * kRows + row) * 4), "r"(v[j]) : "memory");
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  if (split > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
  }
  for (int q = q_mine; q < q1; q += kThreads) {
    const int t = q / (kRows / 4), col = 4 * (q % (kRows / 4));
    const uint32_t at = sums + (t * kRows + col) * 4;
    int d[4] = {0, 0, 0, 0};
    float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < kMaxSplit; ++c) {
      if (c >= split) break;
      const int a = first_step(c), b = first_step(c + 1);
      const uint32_t there = split > 1 ? map_to_cta(at, c) : at;
      if (a < p.nk) {
        const uint4 v = lds_cluster_v4(there);
        if (F16) {
          f[0] += __uint_as_float(v.x);
          f[1] += __uint_as_float(v.y);
          f[2] += __uint_as_float(v.z);
          f[3] += __uint_as_float(v.w);
        } else {
          d[0] += static_cast<int>(v.x);
          d[1] += static_cast<int>(v.y);
          d[2] += static_cast<int>(v.z);
          d[3] += static_cast<int>(v.w);
        }
      }
      if (!F16 && b > p.nk) {
        const uint4 v = lds_cluster_v4(there + N * kRows * 4);
        f[0] += __uint_as_float(v.x);
        f[1] += __uint_as_float(v.y);
        f[2] += __uint_as_float(v.z);
        f[3] += __uint_as_float(v.w);
      }
    }
    float y[4];
    if (F16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = f[j];
    } else {
      const Scales c = q == q_mine ? mine : scales_of(q);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = static_cast<float>(d[j]) * c.s * c.w[j];
        if (p.nr > 0) y[j] = fmaf(p.alpha, f[j], y[j]);
        y[j] += c.b[j];
      }
    }
    store4(p, m0 + t, n0 + col, y);
  }
  if (split > 1) cluster_sync_all();   // the others' reads of this CTA's sums
  if (p.beside) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// CTAs of a cluster: as many as leave all tiles in one round with an SM for each CTA (clusters of some sizes fill the SMs less well), each
// with two steps at least.  us, one token, 5120 -> 5120 (40 tiles) in clusters of 1, 2, 3, 4: 10.1, 8.4, 7.4, 11.8; 77 tokens,
// 18944 -> 3584 (28 tiles) in 1 to 5: 37.5, 23.3, 19.3, 17.2, 28.9.
int plan_split(long long tiles, int steps, int sms, int most) {
  constexpr int kHeld[kMaxSplit + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120, 0, 0, 0, 0, 0, 0, 0, 112};   // CTAs in clusters of so many on 148 SMs
  int best = 1;
  for (int s = 2; s <= std::min(most, steps / 2); ++s)
    if (tiles * s <= static_cast<long long>(kHeld[s]) * sms / 148) best = s;
  return best;
}

// (sixteen, of an SM each, where r's rows are long: 77 tokens, 18944 columns (296 steps), rank 128: 13.0 us in eight, 9.7; 7 tokens, 5120
// columns (80 steps): 5.5, so 6.1.  Nothing between was measured: 160 is twice the one and half the other.)
int most_split(bool f16, int steps) { return f16 && steps >= 160 ? kMaxSplit : 8; }

template <int N, bool F16, bool TWO>
int launch_stream(StreamParams p, const StreamMaps& tm, bool ahead, int sms, cudaStream_t stream) {
  constexpr int smem = smem_of<N, TWO>();
  const int x = (p.OC + kRows - 1) / kRows, y = (p.M + N - 1) / N;
  p.split = TWO ? 1 : plan_split(static_cast<long long>(x) * y, p.nk + p.nr, sms, most_split(F16, p.nk));
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(stream_kernel<N, F16, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return note_cuda_error(e);
    if (F16) {   // clusters of more than eight
      const cudaError_t c = cudaFuncSetAttribute(stream_kernel<N, F16, TWO>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (c != cudaSuccess) return note_cuda_error(c);
    }
    attr_done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(x * p.split, y);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (ahead && use_pdl()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = p.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return note_cuda_error(cudaLaunchKernelEx(&cfg, stream_kernel<N, F16, TWO>, p, tm));
}
template <int N, bool F16> int launch_ring(const StreamParams& p, const StreamMaps& tm, bool ahead, int sms, cudaStream_t stream) {
  static_assert((F16 ? 1 : 2) * N * kRows * 4 <= smem_of<N, false>() - 2048, "the sums fit the ring");
  // Two CTAs to an SM where one each would leave a second round: 16 tokens, 5120 -> 27648 (216 tiles) 25.5 us, so 29.3; with one round
  // the deeper ring: 5120 -> 13824 (108 tiles) 13.1 us, so 14.7.  (Their rings do not hold the two blocks of sums of 128 tokens.)
  if constexpr (N <= 64) {
    static_assert((F16 ? 1 : 2) * N * kRows * 4 <= smem_of<N, true>() - 2048, "the sums fit the ring");
    if (static_cast<long long>((p.OC + kRows - 1) / kRows) * ((p.M + N - 1) / N) > sms) return launch_stream<N, F16, true>(p, tm, ahead, sms, stream);
  }
  return launch_stream<N, F16, false>(p, tm, ahead, sms, stream);
}
template <bool F16> int launch_tokens(const StreamParams& p, const StreamMaps& tm, int n, bool ahead, int sms, cudaStream_t stream) {
  if (n == 16) return launch_ring<16, F16>(p, tm, ahead, sms, stream);
  if (n == 32) return launch_ring<32, F16>(p, tm, ahead, sms, stream);
  if (n == 64) return launch_ring<64, F16>(p, tm, ahead, sms, stream);
  return launch_ring<128, F16>(p, tm, ahead, sms, stream);
}

}  // namespace

cudaError_t w8a8_stream_status(uint32_t* out, cudaStream_t stream) { return take_status(g_w8a8_status, out, stream); }

int w8a8_stream_split(long long tiles, int steps, int sms) { return plan_split(tiles, steps, sms, 8); }

int w8a8_stream_forward(const glowq_w8a8_linear_t& g, bool ahead, int sms, cudaStream_t stream) {
  const bool corrected = g.r_mode != GLOWQ_R_NONE;
  const int n = g.M <= 16 ? 16 : g.M <= 32 ? 32 : g.M <= 64 ? 64 : 128;
  StreamParams p{};
  p.scales = g.scales;
  p.weight_scales = g.weight_scales;
  p.bias = g.bias;
  p.out = g.out;
  p.out_stride = g.out_stride;
  p.out_dtype = g.out_dtype;
  p.M = g.M;
  p.OC = g.OC;
  p.nk = (g.K + 127) / 128;
  p.nr = corrected ? (g.rank + 63) / 64 : 0;
  p.alpha = g.alpha;
  const size_t e = dtype_bytes(g.out_dtype);
  p.vec = g.out_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(g.out) & (4 * e - 1)) == 0;
  StreamMaps tm;
  int rc = tensor_map_2d_ex(&tm.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.weight, g.K, g.OC, g.weight_stride, 128, kRows, 1);
  if (!rc) rc = tensor_map_2d_ex(&tm.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.codes, g.K, g.M, g.code_stride, 128, n, 1);
  if (!rc && corrected) {
    rc = tensor_map_2d_ex(&tm.l, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, g.L, g.rank, g.OC, 2 * g.L_stride, 64, kRows, 1);
    if (!rc) rc = tensor_map_2d_ex(&tm.r, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, g.r, g.rank, g.M, 2 * g.r_stride, 64, n, 1);
  }
  return rc ? rc : launch_tokens<false>(p, tm, n, ahead, sms, stream);
}

int w8a8_right_factor(const glowq_w8a8_linear_t& g, bool beside, bool ahead, int sms, cudaStream_t stream) {
  // Tokens of a tile: those with which a CTA reads least (narrow tiles read R once more each, but there are more CTAs).  77 tokens, 18944
  // columns, rank 128: one tile of 128 tokens in 8 CTAs 13.0 us, five of 16 in 16 each 9.7.
  int n = 128;
  double least = 0.0;
  for (int t = 16; t <= 128; t *= 2) {
    if (g.M > 65535 * t) continue;   // (a grid's second dimension)
    const long long tiles = static_cast<long long>((g.rank + kRows - 1) / kRows) * ((g.M + t - 1) / t);
    const int steps = (g.K + 63) / 64, split = plan_split(tiles, steps, sms, most_split(true, steps));
    const double rounds = static_cast<double>((tiles * split + sms - 1) / sms);
    const double cost = rounds * ((steps + split - 1) / split) * (kAStage + t * 128);
    if (least == 0.0 || cost < least) {
      n = t;
      least = cost;
    }
  }
  StreamParams p{};
  p.out = g.r;
  p.out_stride = g.r_stride;
  p.out_dtype = GLOWQ_F16;
  p.M = g.M;
  p.OC = g.rank;
  p.nk = (g.K + 63) / 64;
  p.vec = g.r_stride % 4 == 0;
  p.early = p.beside = beside;   // (in front of the product, behind the codes of the same x)
  StreamMaps tm;
  int rc = tensor_map_2d_ex(&tm.a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, g.R, g.K, g.rank, 2 * g.R_stride, 64, kRows, 1);
  if (!rc) rc = tensor_map_2d_ex(&tm.b, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, g.r_x, g.K, g.M, 2 * g.r_x_stride, 64, n, 1);
  return rc ? rc : launch_tokens<true>(p, tm, n, ahead, sms, stream);
}

}  // namespace glowq
