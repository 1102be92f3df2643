// Entry points declared in include/glowq_w8a8.h: checks of the arguments and dispatch.
#include <algorithm>
#include <cmath>

#include "w8a8.h"

using namespace glowq;

namespace {

constexpr int kMaxExactK = 131071;     // 128 * 128 * K stays below 2^31: the sums of products are exact
constexpr int kMaxRank = 1024;
constexpr int kMaxTokens = 1 << 22;    // tiles of 128 tokens (above 64 there are no narrower ones) are numbered by 16 bits of a grid
// Rows and columns of the kernels that count them in 32 bits: a row and all rows, a column and a CTA's columns, both halves of the
// gradients' sums stay below 2^31.
constexpr int kMaxRows = 1 << 30, kMaxColumns = 1 << 29;

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool known(int dtype) { return dtype == GLOWQ_F16 || dtype == GLOWQ_F32 || dtype == GLOWQ_BF16; }
bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// a row stride that is used: of a single row it may be anything
bool strided(int64_t stride, int rows, int cols) { return rows <= 1 || stride >= cols; }

int check_rows(const glowq_w8a8_rows_t& r, bool codes) {
  if (r.M < 0 || r.K <= 0 || r.reserved != 0 || !known(r.dtype)) return GLOWQ_ERR_BAD_ARGUMENT;
  if (r.norm != GLOWQ_NORM_NONE && r.norm != GLOWQ_NORM_LAYER && r.norm != GLOWQ_NORM_RMS) return GLOWQ_ERR_BAD_ARGUMENT;
  if (codes ? r.y != nullptr : r.norm != GLOWQ_NORM_LAYER || r.codes || r.scales) return GLOWQ_ERR_BAD_ARGUMENT;
  if (r.norm == GLOWQ_NORM_NONE ? r.weight || r.residual || r.mean || r.rstd : !r.weight || !(r.eps >= 0.0)) return GLOWQ_ERR_BAD_ARGUMENT;
  if ((r.bias && r.norm != GLOWQ_NORM_LAYER) || (r.hidden && !r.residual) || (r.constant && r.norm != GLOWQ_NORM_NONE))
    return GLOWQ_ERR_BAD_ARGUMENT;
  if (r.M > kMaxRows || r.K > kMaxColumns) return GLOWQ_ERR_TOO_LARGE;
  if (r.M == 0) return GLOWQ_OK;
  if (!r.x || (codes ? !r.codes || !r.scales : !r.y)) return GLOWQ_ERR_BAD_ARGUMENT;
  const size_t e = dtype_bytes(r.dtype);
  for (const void* p : {r.x, r.residual, r.weight, r.bias, static_cast<const void*>(r.hidden), static_cast<const void*>(r.y)})
    if (!aligned(p, e)) return GLOWQ_ERR_BAD_ARGUMENT;
  if (!strided(r.x_stride, r.M, r.K) || (r.residual && !strided(r.residual_stride, r.M, r.K)) ||
      (r.hidden && !strided(r.hidden_stride, r.M, r.K)) || (codes ? !strided(r.code_stride, r.M, r.K) : !strided(r.y_stride, r.M, r.K)))
    return GLOWQ_ERR_BAD_STRIDE;
  return GLOWQ_OK;
}

int run_rows(const glowq_w8a8_rows_t* rows, bool codes) {
  if (!rows) return GLOWQ_ERR_BAD_ARGUMENT;
  int rc = check_rows(*rows, codes), sms = 0;
  if (rc == GLOWQ_OK) rc = current_device_sms(&sms);
  if (rc != GLOWQ_OK || rows->M == 0) return rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(rows->stream);
  cudaError_t e = launch_rows(*rows, sms, stream);
  if (e == cudaSuccess && rows->constant) e = launch_settle(stream);
  return note_cuda_error(e);
}

// operands that the copy engine reads: they begin on 16 bytes, and so does every row
int check_operand(const void* p, int64_t stride, size_t e, int rows, int cols) {
  if (!p || !on16(p)) return GLOWQ_ERR_BAD_ARGUMENT;
  if (stride < cols || (stride * static_cast<int64_t>(e)) % 16 != 0 || stride > (int64_t{1} << 35)) return GLOWQ_ERR_BAD_STRIDE;
  (void)rows;
  return GLOWQ_OK;
}

int check_right_factor(const glowq_w8a8_linear_t& g) {
  if (g.M < 0 || g.K <= 0 || g.rank <= 0 || g.reserved != 0) return GLOWQ_ERR_BAD_ARGUMENT;
  if (g.M > kMaxTokens || g.K > kMaxColumns || g.rank > kMaxRank) return GLOWQ_ERR_TOO_LARGE;
  if (g.M == 0) return GLOWQ_OK;
  int rc = check_operand(g.r_x, g.r_x_stride, 2, g.M, g.K);
  if (!rc) rc = check_operand(g.R, g.R_stride, 2, g.rank, g.K);
  if (!rc) rc = check_operand(g.r, g.r_stride, 2, g.M, g.rank);
  return rc;
}

int check_linear(const glowq_w8a8_linear_t& g) {
  if (g.M < 0 || g.K <= 0 || g.OC <= 0 || g.rank < 0 || g.reserved != 0 || !known(g.out_dtype)) return GLOWQ_ERR_BAD_ARGUMENT;
  if (g.r_mode != GLOWQ_R_NONE && g.r_mode != GLOWQ_R_COMPUTE && g.r_mode != GLOWQ_R_LOAD) return GLOWQ_ERR_BAD_ARGUMENT;
  if (g.K > kMaxExactK || g.M > kMaxTokens || g.OC > kMaxColumns) return GLOWQ_ERR_TOO_LARGE;
  if (g.M == 0) return GLOWQ_OK;
  if (!g.scales || !g.weight_scales || !g.out || !aligned(g.out, dtype_bytes(g.out_dtype)) || !aligned(g.scales, 4) ||
      !aligned(g.weight_scales, 4) || !aligned(g.bias, 4))
    return GLOWQ_ERR_BAD_ARGUMENT;
  if (!strided(g.out_stride, g.M, g.OC)) return GLOWQ_ERR_BAD_STRIDE;
  int rc = check_operand(g.codes, g.code_stride, 1, g.M, g.K);
  if (!rc) rc = check_operand(g.weight, g.weight_stride, 1, g.OC, g.K);
  if (!rc && g.x && !(known(g.x_dtype) && aligned(g.x, dtype_bytes(g.x_dtype)))) rc = GLOWQ_ERR_BAD_ARGUMENT;
  if (!rc && g.x && !strided(g.x_stride, g.M, g.K)) rc = GLOWQ_ERR_BAD_STRIDE;
  if (rc || g.r_mode == GLOWQ_R_NONE) return rc;
  if (g.rank <= 0) return GLOWQ_ERR_BAD_ARGUMENT;
  if (g.rank > kMaxRank) return GLOWQ_ERR_TOO_LARGE;
  rc = check_operand(g.L, g.L_stride, 2, g.OC, g.rank);
  if (!rc) rc = g.r_mode == GLOWQ_R_COMPUTE ? check_right_factor(g) : check_operand(g.r, g.r_stride, 2, g.M, g.rank);
  return rc;
}

// Microseconds of a call of more than 64 tokens in either form (for choosing between them), on B200: fitted to eight weights from
// 3584 x 1024 to 5120 x 27648 at 65 to 1024 tokens; within some 10 %.  (us, streaming / pairs of the width taken: 96 tokens 18944 -> 3584
// 19.4 / 36.9, 5120 -> 27648 42.5 / 33.0; 200 tokens 18944 -> 3584 27.0 / 37.7, 5120 -> 13824 38.6 / 20.9.)
// Streaming: rounds of CTAs, each a chain of about 6 to 8 us and its steps, which take 0.25 us or what HBM needs for all CTAs' weights.
double stream_us(int M, long long steps, int OC, int sms) {
  const long long x = (OC + 127) / 128, y = (M + 127) / 128, tiles = x * y;
  const int split = w8a8_stream_split(tiles, static_cast<int>(steps), sms);
  const double chain = 6.0 + 0.015 * std::min(M, 128), each = static_cast<double>((steps + split - 1) / split);
  const auto round = [&](double ctas) { return chain + each * std::max(0.25, ctas * 16384.0 / 5.4e6); };
  const long long ctas = tiles * split, whole = ctas / sms, rest = ctas % sms;
  return static_cast<double>(whole) * round(sms) + (rest ? round(static_cast<double>(rest)) : 0.0);
}
// Pairs: a chain of 5.5 us, and rounds of tiles whose steps take what the narrow ones' copies or the wide ones' MMAs do.
double pair_us(int M, long long steps, int OC, int n, int sms) {
  const double step = n == 64 ? 0.211 : n == 128 ? 0.224 : n == 192 ? 0.228 : 0.292;
  const long long tiles = static_cast<long long>((OC + n - 1) / n) * ((M + 255) / 256), pairs = sms / 2;
  return 5.5 + static_cast<double>((tiles + pairs - 1) / pairs) * (static_cast<double>(steps) * step + 0.4);
}
// Channels of a pair's tile, or 0: the streaming form.
int pair_columns(const glowq_w8a8_linear_t& g, int sms) {
  if (g.M <= 64) return 0;
  const bool corrected = g.r_mode != GLOWQ_R_NONE;
  // (a converted tile is held as sums / alpha: a factor near nothing would leave the range of fp32)
  if (corrected && !(std::fabs(g.alpha) >= 0x1p-60f && std::fabs(g.alpha) <= 0x1p60f)) return 0;
  const long long steps = (g.K + 127) / 128 + (corrected ? (g.rank + 63) / 64 : 0);
  int best = 0;
  double least = stream_us(g.M, steps, g.OC, sms);
  for (int n = 64; n <= 256; n += 64) {
    const double us = pair_us(g.M, steps, g.OC, n, sms);
    if (us < least) {
      best = n;
      least = us;
    }
  }
  return best;
}

}  // namespace

extern "C" {

int glowq_w8a8_quantize(const glowq_w8a8_rows_t* rows) { return run_rows(rows, true); }
int glowq_layer_norm_forward(const glowq_w8a8_rows_t* rows) { return run_rows(rows, false); }

size_t glowq_layer_norm_workspace_bytes(int M, int K) { return M <= 0 || K <= 0 ? 0 : layer_norm_grad_bytes(M, K); }

int glowq_layer_norm_backward(const glowq_layer_norm_grad_t* grad) {
  if (!grad) return GLOWQ_ERR_BAD_ARGUMENT;
  const glowq_layer_norm_grad_t& g = *grad;
  if (g.M <= 0 || g.K <= 0 || g.reserved != 0 || !known(g.dtype)) return GLOWQ_ERR_BAD_ARGUMENT;
  if (!g.h || !g.dy || !g.weight || !g.mean || !g.rstd || (!g.dweight) != (!g.dbias) || (!g.dx && !g.dweight) || (g.dh && !g.dx))
    return GLOWQ_ERR_BAD_ARGUMENT;
  if (g.M > kMaxRows || g.K > kMaxColumns) return GLOWQ_ERR_TOO_LARGE;
  const size_t e = dtype_bytes(g.dtype);
  for (const void* p : {g.h, g.dy, g.dh, g.weight, static_cast<const void*>(g.dx), static_cast<const void*>(g.dweight),
                        static_cast<const void*>(g.dbias)})
    if (!aligned(p, e)) return GLOWQ_ERR_BAD_ARGUMENT;
  if (!strided(g.h_stride, g.M, g.K) || !strided(g.dy_stride, g.M, g.K) || (g.dh && !strided(g.dh_stride, g.M, g.K)) ||
      (g.dx && !strided(g.dx_stride, g.M, g.K)))
    return GLOWQ_ERR_BAD_STRIDE;
  if (!g.workspace || !aligned(g.workspace, 16) || g.workspace_bytes < layer_norm_grad_bytes(g.M, g.K)) return GLOWQ_ERR_WORKSPACE_TOO_SMALL;
  int sms = 0;
  const int rc = current_device_sms(&sms);
  if (rc != GLOWQ_OK) return rc;
  return note_cuda_error(launch_layer_norm_grad(g, static_cast<cudaStream_t>(g.stream)));
}

int glowq_w8a8_right_factor(const glowq_w8a8_linear_t* linear) {
  if (!linear) return GLOWQ_ERR_BAD_ARGUMENT;
  int rc = check_right_factor(*linear), sms = 0;
  if (rc == GLOWQ_OK) rc = current_device_sms(&sms);
  if (rc != GLOWQ_OK || linear->M == 0) return rc;
  return w8a8_right_factor(*linear, false, (linear->r_mode & GLOWQ_W8A8_FRESH) == 0, sms, static_cast<cudaStream_t>(linear->stream));
}

int glowq_w8a8_linear(const glowq_w8a8_linear_t* linear) {
  if (!linear) return GLOWQ_ERR_BAD_ARGUMENT;
  glowq_w8a8_linear_t g = *linear;
  // Operands that were made right in front: the call's first launch waits for that as any kernel does.  (Codes' launch reads none of them,
  // and those behind it begin when it is past its own wait.)
  const bool ahead = (g.r_mode & GLOWQ_W8A8_FRESH) == 0;
  g.r_mode &= ~GLOWQ_W8A8_FRESH;
  int rc = check_linear(g), sms = 0;
  if (rc == GLOWQ_OK) rc = current_device_sms(&sms);
  if (rc != GLOWQ_OK || g.M == 0) return rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(g.stream);
  if (g.alpha == 0.f) g.r_mode = GLOWQ_R_NONE;   // nothing to add
  if (g.x && g.r_mode == GLOWQ_R_COMPUTE && few_tokens(g)) {
    if ((rc = note_cuda_error(launch_few_tokens(g, ahead, stream))) != GLOWQ_OK) return rc;
  } else {
    if (g.x) {
      glowq_w8a8_rows_t r{};
      r.x = g.x;
      r.x_stride = g.x_stride;
      r.codes = g.codes;
      r.code_stride = g.code_stride;
      r.scales = g.scales;
      r.M = g.M;
      r.K = g.K;
      r.dtype = g.x_dtype;
      if ((rc = note_cuda_error(launch_rows(r, sms, stream))) != GLOWQ_OK) return rc;
    }
    if (g.r_mode == GLOWQ_R_COMPUTE && (rc = w8a8_right_factor(g, g.x != nullptr, ahead || g.x, sms, stream)) != GLOWQ_OK) return rc;
  }
  const int n = pair_columns(g, sms);
  // (behind another launch of this call, that one was waited for)
  const bool first = !g.x && g.r_mode != GLOWQ_R_COMPUTE;
  return n > 0 ? w8a8_pair_forward(g, n, ahead || !first, sms, stream) : w8a8_stream_forward(g, ahead || !first, sms, stream);
}

int glowq_w8a8_read_status(void* stream) {
  uint32_t words[2] = {0, 0};
  int rc = note_cuda_error(w8a8_stream_status(&words[0], static_cast<cudaStream_t>(stream)));
  if (rc == GLOWQ_OK) rc = note_cuda_error(w8a8_pair_status(&words[1], static_cast<cudaStream_t>(stream)));
  return rc != GLOWQ_OK ? rc : words[0] | words[1] ? GLOWQ_ERR_DEVICE_TIMEOUT : GLOWQ_OK;
}

}  // extern "C"
