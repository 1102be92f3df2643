// The row kernels' entry points by type, and what a few tokens in front of a corrected linear take.
#include "w8a8_rows.cuh"

namespace glowq {

// One file for each type of rows: together they take the compiler minutes.
cudaError_t launch_rows_f16(const RowsParams& params, int norm, int sms, cudaStream_t stream);
cudaError_t launch_rows_bf16(const RowsParams& params, int norm, int sms, cudaStream_t stream);
cudaError_t launch_rows_f32(const RowsParams& params, int norm, int sms, cudaStream_t stream);
cudaError_t launch_norm_grad_f16(const GradParams& params, cudaStream_t stream);
cudaError_t launch_norm_grad_bf16(const GradParams& params, cudaStream_t stream);
cudaError_t launch_norm_grad_f32(const GradParams& params, cudaStream_t stream);

namespace {

// A few tokens in front of a corrected linear: their codes, and r = x . R^T, in one launch.  CTAs 0 .. M - 1 take a token each, as above;
// each of the others one row of R, whose pieces it holds while it goes through the tokens (R does not hang on the kernels before and is
// read before the wait for them).  For so few tokens the product of the streaming form is a launch of its own that takes 5.3 us
// (5120 columns, rank 128) for 1.3 MB, as a tile of it goes to eight CTAs at most: a whole linear 5120 -> 5120 12.6 us, so 8.9.
constexpr int kFewTokens = 4;
struct FewParams {
  RowsParams rows;
  const __half* R;
  __half* r;
  long long R_stride, r_stride;
};
template <int THREADS> __global__ void __launch_bounds__(THREADS) few_tokens_kernel(const __grid_constant__ FewParams p) {
  constexpr int V = 8;
  __shared__ uint32_t s_max[32];
  __shared__ float s_dot[THREADS / 32][kFewTokens];
  const int t = threadIdx.x, step = blockDim.x * V, K = p.rows.K, M = p.rows.M;
  const auto column = [&](int i) { return min(t * V + i * step, K - V); };
  const __half* const x0 = static_cast<const __half*>(p.rows.x);
  if (static_cast<int>(blockIdx.x) < M) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int row = blockIdx.x;
    Vec h[kNV];
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kNV; ++i) h[i] = load_row<__half, kWhole>(x0 + row * p.rows.xs, column(i), K);
#pragma unroll
    for (int i = 0; i < kNV; ++i) top = Num<__half>::top(top, h[i]);
    const Scale sc = make_scale(row_max<false>(Num<__half>::top_bits(top), s_max));
    if (t == 0) p.rows.scales[row] = sc.s;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      float f[V];
      uint32_t c4[V / 4];
      Num<__half>::unpack(h[i], f);
      codes_of<V>(f, sc, c4);
      store_codes<V, kWhole>(p.rows.codes + row * p.rows.cs, column(i), K, true, 0, c4);
    }
    return;
  }
  const int j = blockIdx.x - M, lane = t & 31, warp = t >> 5;
  F2 w[kNV][V / 2];
#pragma unroll
  for (int i = 0; i < kNV; ++i)
    unpack2<__half>(t * V + i * step < K ? ld16(p.R + j * p.R_stride + t * V + i * step) : Vec{}, w[i]);   // (zeros past the end)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Vec x[kFewTokens][kNV];
#pragma unroll
  for (int m = 0; m < kFewTokens; ++m)
#pragma unroll
    for (int i = 0; i < kNV; ++i)
      x[m][i] = m < M && t * V + i * step < K ? ld16(x0 + m * p.rows.xs + t * V + i * step) : Vec{};
  float dot = 0.f;   // lane m: token m's sum over this warp's columns
#pragma unroll
  for (int m = 0; m < kFewTokens; ++m) {
    if (m >= M) break;
    F2 s = 0ull;
#pragma unroll
    for (int i = 0; i < kNV; ++i) {
      F2 f[V / 2];
      unpack2<__half>(x[m][i], f);
#pragma unroll
      for (int q = 0; q < V / 2; ++q) s = fma2(w[i][q], f[q], s);
    }
    float sum = parts(s).x + parts(s).y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == m) dot = sum;
  }
  if (lane < M) s_dot[warp][lane] = dot;
  __syncthreads();
  if (warp == 0 && lane < M) {
    const int nw = blockDim.x >> 5;
    for (int i = 1; i < nw; ++i) dot += s_dot[i][lane];
    p.r[lane * p.r_stride + j] = __float2half_rn(dot);
  }
}

}  // namespace

cudaError_t launch_rows(const glowq_w8a8_rows_t& r, int sms, cudaStream_t stream) {
  const RowsParams p{r.x,        r.residual,        r.weight,        r.bias,     r.hidden,      r.y, r.codes, r.scales, r.mean, r.rstd, r.eps, 1.0 / r.K,
                     r.x_stride, r.residual_stride, r.hidden_stride, r.y_stride, r.code_stride, r.M, r.K};
  if (r.dtype == GLOWQ_F16) return launch_rows_f16(p, r.norm, sms, stream);
  if (r.dtype == GLOWQ_BF16) return launch_rows_bf16(p, r.norm, sms, stream);
  return launch_rows_f32(p, r.norm, sms, stream);
}

bool few_tokens(const glowq_w8a8_linear_t& g) {
  const auto whole = [](const void* q, long long stride) { return on16(q) && stride % 8 == 0; };
  return g.M <= kFewTokens && g.x == g.r_x && g.x_dtype == GLOWQ_F16 && (g.M == 1 || g.x_stride == g.r_x_stride) && g.K % 8 == 0 &&
         g.K <= 8 * kNV * kRowThreads && whole(g.x, g.M > 1 ? g.x_stride : 0);
}
cudaError_t launch_few_tokens(const glowq_w8a8_linear_t& g, bool ahead, cudaStream_t stream) {
  FewParams p{};
  p.rows.x = g.x;
  p.rows.xs = g.x_stride;
  p.rows.codes = g.codes;
  p.rows.cs = g.code_stride;
  p.rows.scales = g.scales;
  p.rows.M = g.M;
  p.rows.K = g.K;
  p.R = static_cast<const __half*>(g.R);
  p.R_stride = g.R_stride;
  p.r = static_cast<__half*>(g.r);
  p.r_stride = g.r_stride;
  const int threads = ((g.K / 8 + kNV - 1) / kNV + 31) / 32 * 32;
  if (threads <= 256) return launch(few_tokens_kernel<256>, dim3(g.M + g.rank), threads, stream, p, ahead);
  return launch(few_tokens_kernel<kRowThreads>, dim3(g.M + g.rank), threads, stream, p, ahead);
}

__global__ void settle_kernel() {}
cudaError_t launch_settle(cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = cfg.blockDim = dim3(1);
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, settle_kernel);
}

size_t layer_norm_grad_bytes(int M, int K) {
  // every plan's parts (of at most kGradParts CTAs, a multiple of eight), and the row sums of the plan for long rows
  return (2ull * K * std::min(kGradParts, (std::max(M, 1) + 7) / 8 * 8) + 2ull * std::max(M, 1)) * 4;
}

cudaError_t launch_layer_norm_grad(const glowq_layer_norm_grad_t& g, cudaStream_t stream) {
  const GradParams p{g.h,        g.dy,        g.dh,        g.weight,    g.mean, g.rstd, g.dx, g.dweight, g.dbias, static_cast<float*>(g.workspace),
                     g.h_stride, g.dy_stride, g.dh_stride, g.dx_stride, g.M,    g.K,    1,    32};
  if (g.dtype == GLOWQ_F16) return launch_norm_grad_f16(p, stream);
  if (g.dtype == GLOWQ_BF16) return launch_norm_grad_bf16(p, stream);
  return launch_norm_grad_f32(p, stream);
}

}  // namespace glowq
