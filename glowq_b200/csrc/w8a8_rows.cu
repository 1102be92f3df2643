// Rows in front of a linear: residual add, layer norm or RMSNorm, int8 codes; and the layer norm's gradients.
//
//   h = x + residual;  v = norm(h);  scale = max |v| / 127;  code = nearest integer of v / scale
//
// All of it is bound by memory: a row is read once, stays in registers through the norm, the maximum and the codes, and every output is
// written once.  A row belongs to one CTA of as many threads as it has pieces of 4 x 16 bytes (to one warp up to 1024 16-bit columns,
// several rows to a CTA then), so that a row's loads are all in flight at once and the SM holds many rows.
//   A code is the nearest integer of the EXACT quotient, ties to even: it does not hang on how a division rounds.  n = rint(v * (1 / s))
// is off only where the quotient lies within 2^-16 of a border; there the remainder v - n s, which one FMA gives exactly, decides.
//   The statistics of a norm are sums in 64 bits, rounded to fp32 once, so that they - and with them every code - do not depend on the
// order of the sums.  They are taken in one pass of the differences to the row's first element c:  var = S2/K - (S1/K)^2.  The
// cancellation in it is at most K-fold, because c is an element of the row: var >= (c - mean)^2 / K.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "w8a8.h"

namespace glowq {
namespace {

constexpr int kNV = 4;             // 16-byte pieces per thread
constexpr int kNS = 16;            // single elements per thread where a row cannot be read in pieces
constexpr int kRowThreads = 1024;  // threads of a row at most
constexpr int kWarpRows = 4;       // rows of a CTA where a warp takes one

struct RowsParams {
  const void *x, *residual, *weight, *bias;
  void *hidden, *y;
  int8_t* codes;
  float *scales, *mean, *rstd;
  double eps;
  long long xs, rs, hs, ys, cs;
  int M, K;
};

template <typename T> struct Num;
template <> struct Num<float> {
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Num<__half> {
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <> struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};
template <typename T> __device__ __forceinline__ float rounded(float v) { return Num<T>::up(Num<T>::down(v)); }

// VEC elements that are read and written together.
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Piece {
  T e[VEC];
};
template <typename T, int VEC> __device__ __forceinline__ Piece<T, VEC> load(const T* p) {
  return *reinterpret_cast<const Piece<T, VEC>*>(p);
}
template <typename T, int VEC> __device__ __forceinline__ void store(T* p, const float (&v)[VEC]) {
  Piece<T, VEC> o;
#pragma unroll
  for (int i = 0; i < VEC; ++i) o.e[i] = Num<T>::down(v[i]);
  *reinterpret_cast<Piece<T, VEC>*>(p) = o;
}

// ---------------------------------------------------------------- codes
struct Scale {
  float s, inv;
  bool plain;   // neither zero, tiny nor NaN
};
// `bits`: the row's largest absolute value, as an integer (so that a NaN is above all numbers)
__device__ __forceinline__ Scale make_scale(uint32_t bits) {
  Scale r;
  const float a = __uint_as_float(bits);
  r.s = bits >= 0x7F800000u ? CUDART_NAN_F : __fdiv_rn(a, 127.f);
  r.plain = bits < 0x7F800000u && a >= 0x1p-100f;
  r.inv = r.plain ? __fdiv_rn(1.f, r.s) : 0.f;
  return r;
}
// The quotient v inv, its nearest integer n and whether a border is near.  (Up to 127 the quotient is off by less than 2^-16.)
__device__ __forceinline__ int code_plain(float v, float s, float inv) {
  const float q = v * inv;
  const float m = q + 12582912.f;   // 1.5 * 2^23: the sum rounds to an integer
  float n = m - 12582912.f;
  if (fabsf(fabsf(q - n) - 0.5f) < 0x1p-14f) {
    const float rem = fmaf(-n, s, v), half = 0.5f * s;   // exact: a multiple of both ulps, and no larger than s
    const bool odd = (__float_as_uint(m) & 1u) != 0u;
    if (fabsf(rem) > half || (fabsf(rem) == half && odd)) n += copysignf(1.f, rem);
  }
  return static_cast<int>(n);
}
// Rows of values below 2^-100, where the scale may be a subnormal number: both are scaled up first, which is exact.
__device__ __noinline__ int code_tiny(float v, float s) {
  if (!(s > 0.f)) return 0;   // zero, NaN
  const float sv = v * 0x1p64f, ss = s * 0x1p64f;
  const int n = code_plain(sv, ss, __fdiv_rn(1.f, ss));
  return max(-127, min(127, n));
}
template <int VEC> __device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[VEC], const Scale& sc) {
  int c[VEC];
  if (sc.plain) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = code_plain(v[i], sc.s, sc.inv);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = code_tiny(v[i], sc.s);
  }
  if constexpr (VEC == 1) {
    *p = static_cast<int8_t>(c[0]);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
    if constexpr (VEC == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// ---------------------------------------------------------------- sums over a row's threads
// (butterflies: every lane ends with the same bits)
__device__ __forceinline__ double2 warp_sum(double2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}
template <bool WARP> __device__ __forceinline__ double2 row_sum(double2 v, double2* room) {
  v = warp_sum(v);
  if (WARP) return v;
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < nw ? room[lane] : make_double2(0.0, 0.0));
}
template <bool WARP> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* room) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (WARP) return v;
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < nw ? room[lane] : 0u);
}

struct Stats {
  float mean, rstd;
};
template <int NORM> __device__ __forceinline__ Stats make_stats(double2 sum, double c, double eps, int K) {
  const double n = static_cast<double>(K), s1 = sum.x / n, s2 = sum.y / n;
  Stats st;
  st.mean = NORM == GLOWQ_NORM_LAYER ? static_cast<float>(c + s1) : 0.f;
  double var = NORM == GLOWQ_NORM_LAYER ? s2 - s1 * s1 : s2;
  if (var < 0.0) var = 0.0;   // (a NaN stays)
  st.rstd = static_cast<float>(1.0 / sqrt(var + eps));
  return st;
}
template <typename T, int NORM> __device__ __forceinline__ float normed(float h, const Stats& st, float w, float b) {
  if (NORM == GLOWQ_NORM_LAYER) return rounded<T>(fmaf((h - st.mean) * st.rstd, w, b));
  return rounded<T>(w * rounded<T>(h * st.rstd));
}

// One row per CTA, or per warp.
template <typename T, int VEC, int NV, int NORM, bool CODES, bool WARP>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const __grid_constant__ RowsParams p, const int constant) {
  __shared__ double2 s_sum[32];
  __shared__ uint32_t s_max[32];
  if (!constant) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row = WARP ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, step = (WARP ? 32 : blockDim.x) * VEC, K = p.K;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= p.M) return;   // (whole warps)
  const T* const x = static_cast<const T*>(p.x) + row * p.xs;
  const T* const res = p.residual ? static_cast<const T*>(p.residual) + row * p.rs : nullptr;

  Piece<T, VEC> raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (t * VEC + i * step < K) raw[i] = load<T, VEC>(x + t * VEC + i * step);
  float v[NV][VEC];
  if (res) {
    Piece<T, VEC> add[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t * VEC + i * step < K) add[i] = load<T, VEC>(res + t * VEC + i * step);
    T* const hid = p.hidden ? static_cast<T*>(p.hidden) + row * p.hs : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t * VEC + i * step;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = k < K ? rounded<T>(Num<T>::up(raw[i].e[j]) + Num<T>::up(add[i].e[j])) : 0.f;
      if (hid && k < K) store<T, VEC>(hid + k, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = t * VEC + i * step < K ? Num<T>::up(raw[i].e[j]) : 0.f;
  }

  if (NORM != GLOWQ_NORM_NONE) {
    double c = 0.0;
    if (NORM == GLOWQ_NORM_LAYER) {
      float first = Num<T>::up(x[0]);
      if (res) first = rounded<T>(first + Num<T>::up(res[0]));
      c = first;
    }
    double2 sum = make_double2(0.0, 0.0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t * VEC + i * step < K) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const double d = static_cast<double>(v[i][j]) - c;
          if (NORM == GLOWQ_NORM_LAYER) sum.x += d;
          sum.y = fma(d, d, sum.y);
        }
      }
    sum = row_sum<WARP>(sum, s_sum);
    const Stats st = make_stats<NORM>(sum, c, p.eps, K);
    if (t == 0) {
      if (p.mean) p.mean[row] = st.mean;
      if (p.rstd) p.rstd[row] = st.rstd;
    }
    const T *const w = static_cast<const T*>(p.weight), *const b = static_cast<const T*>(p.bias);
    T* const y = CODES ? nullptr : static_cast<T*>(p.y) + row * p.ys;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t * VEC + i * step;
      if (k >= K) continue;
      const Piece<T, VEC> wv = load<T, VEC>(w + k);
      Piece<T, VEC> bv;
      if (NORM == GLOWQ_NORM_LAYER && b) bv = load<T, VEC>(b + k);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        v[i][j] = normed<T, NORM>(v[i][j], st, Num<T>::up(wv.e[j]), NORM == GLOWQ_NORM_LAYER && b ? Num<T>::up(bv.e[j]) : 0.f);
      if (!CODES) store<T, VEC>(y + k, v[i]);
    }
  }

  if (CODES) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);   // (zeros past the end)
    const Scale sc = make_scale(row_max<WARP>(top, s_max));
    if (t == 0) p.scales[row] = sc.s;
    int8_t* const out = p.codes + row * p.cs;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t * VEC + i * step < K) store_codes<VEC>(out + t * VEC + i * step, v[i], sc);
  }
}

// Rows that do not fit a CTA's registers: the same in passes over the row, which stays in L2.
template <typename T, int NORM, bool CODES>
__global__ void __launch_bounds__(kRowThreads) long_rows_kernel(const __grid_constant__ RowsParams p, const int constant) {
  __shared__ double2 s_sum[32];
  __shared__ uint32_t s_max[32];
  if (!constant) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = blockIdx.x, K = p.K;
  const T* const x = static_cast<const T*>(p.x) + row * p.xs;
  const T* const res = p.residual ? static_cast<const T*>(p.residual) + row * p.rs : nullptr;
  const auto value = [&](int k) {
    const float v = Num<T>::up(x[k]);
    return res ? rounded<T>(v + Num<T>::up(res[k])) : v;
  };
  Stats st{0.f, 1.f};
  if (NORM != GLOWQ_NORM_NONE) {
    const double c = NORM == GLOWQ_NORM_LAYER ? value(0) : 0.0;
    double2 sum = make_double2(0.0, 0.0);
    for (int k = threadIdx.x; k < K; k += blockDim.x) {
      const double d = static_cast<double>(value(k)) - c;
      sum.x += d;
      sum.y = fma(d, d, sum.y);
    }
    st = make_stats<NORM>(row_sum<false>(sum, s_sum), c, p.eps, K);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[row] = st.mean;
      if (p.rstd) p.rstd[row] = st.rstd;
    }
  }
  const T *const w = static_cast<const T*>(p.weight), *const b = static_cast<const T*>(p.bias);
  const auto result = [&](int k) {
    const float h = value(k);
    if (NORM == GLOWQ_NORM_NONE) return h;
    return normed<T, NORM>(h, st, Num<T>::up(w[k]), NORM == GLOWQ_NORM_LAYER && b ? Num<T>::up(b[k]) : 0.f);
  };
  // (hidden may not overlap x or the residual: the passes read them again)
  T* const hid = p.hidden ? static_cast<T*>(p.hidden) + row * p.hs : nullptr;
  uint32_t top = 0u;
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    if (hid) hid[k] = Num<T>::down(value(k));
    const float v = result(k);
    if (CODES)
      top = max(top, __float_as_uint(v) & 0x7FFFFFFFu);
    else
      (static_cast<T*>(p.y) + row * p.ys)[k] = Num<T>::down(v);
  }
  if (CODES) {
    const Scale sc = make_scale(row_max<false>(top, s_max));
    if (threadIdx.x == 0) p.scales[row] = sc.s;
    for (int k = threadIdx.x; k < K; k += blockDim.x) {
      const float v[1] = {result(k)};
      store_codes<1>(p.codes + row * p.cs + k, v, sc);
    }
  }
}

template <typename Kernel, typename Params, typename... More>
cudaError_t launch(Kernel kernel, int grid, int threads, cudaStream_t stream, const Params& p, More... more) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = use_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p, more...);
}

bool on(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T, int NORM, bool CODES> cudaError_t launch_rows_of(const RowsParams& p, int constant, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const auto whole = [](const void* q, long long stride) { return !q || (on(q, 16) && stride % V == 0); };
  const bool pieces = p.K % V == 0 && whole(p.x, p.xs) && whole(p.residual, p.rs) && whole(p.hidden, p.hs) && whole(p.y, p.ys) &&
                      whole(p.weight, 0) && whole(p.bias, 0) && (!p.codes || (on(p.codes, V) && p.cs % V == 0));
  const auto warps = [](int n) { return (n + 31) / 32 * 32; };
  if (pieces) {
    const int threads = warps((p.K / V + kNV - 1) / kNV);
    if (threads == 32)
      return launch(rows_kernel<T, V, kNV, NORM, CODES, true>, (p.M + kWarpRows - 1) / kWarpRows, 32 * kWarpRows, stream, p, constant);
    if (threads <= kRowThreads) return launch(rows_kernel<T, V, kNV, NORM, CODES, false>, p.M, threads, stream, p, constant);
  } else {
    const int threads = warps((p.K + kNS - 1) / kNS);
    if (threads == 32)
      return launch(rows_kernel<T, 1, kNS, NORM, CODES, true>, (p.M + kWarpRows - 1) / kWarpRows, 32 * kWarpRows, stream, p, constant);
    if (threads <= kRowThreads) return launch(rows_kernel<T, 1, kNS, NORM, CODES, false>, p.M, threads, stream, p, constant);
  }
  return launch(long_rows_kernel<T, NORM, CODES>, p.M, kRowThreads, stream, p, constant);
}
template <typename T> cudaError_t launch_rows_typed(const RowsParams& p, int norm, int constant, cudaStream_t stream) {
  if (norm == GLOWQ_NORM_NONE) return launch_rows_of<T, GLOWQ_NORM_NONE, true>(p, constant, stream);
  if (norm == GLOWQ_NORM_RMS) return launch_rows_of<T, GLOWQ_NORM_RMS, true>(p, constant, stream);
  if (p.codes) return launch_rows_of<T, GLOWQ_NORM_LAYER, true>(p, constant, stream);
  return launch_rows_of<T, GLOWQ_NORM_LAYER, false>(p, constant, stream);
}

// ---------------------------------------------------------------- gradients of the layer norm
// A CTA takes rows r, r + grid, ... ROWS at a time, a thread the same columns of all of them: the sums of dweight and dbias stay in its
// registers until the end.  Reads h, dy (dh) and writes dx once: bound by memory.
struct GradParams {
  const void *h, *dy, *dh, *weight;
  const float *mean, *rstd;
  void *dx, *dweight, *dbias;
  float* partial;     // [grid][2][K], then (long rows) [M][2] sums
  long long hs, ys, ds, xs;
  int M, K, parts;
};

template <typename T, int VEC, int NV, int ROWS, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_grad_kernel(const __grid_constant__ GradParams p) {
  __shared__ float s_part[2][2 * ROWS][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x, step = blockDim.x * VEC, K = p.K, nw = blockDim.x >> 5, lane = t & 31, warp = t >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float dw[NV][VEC], db[NV][VEC];
  Piece<T, VEC> w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (t * VEC + i * step < K) w[i] = load<T, VEC>(static_cast<const T*>(p.weight) + t * VEC + i * step);
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  const float inv_k = 1.f / static_cast<float>(K);
  int buf = 0;
  for (int r0 = blockIdx.x * ROWS; r0 < p.M; r0 += gridDim.x * ROWS, buf ^= 1) {
    Piece<T, VEC> h[ROWS][NV], g[ROWS][NV];
    float mean[ROWS], rstd[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int row = r0 + r;
      const bool in = row < p.M;
      mean[r] = in ? p.mean[row] : 0.f;
      rstd[r] = in ? p.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = t * VEC + i * step;
        if (in && k < K) {
          h[r][i] = load<T, VEC>(static_cast<const T*>(p.h) + row * p.hs + k);
          g[r][i] = load<T, VEC>(static_cast<const T*>(p.dy) + row * p.ys + k);
        }
      }
    }
    // sums of g = dy w and g xh over the columns
    float c[2 * ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      c[2 * r] = c[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (r0 + r < p.M && t * VEC + i * step < K) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float d = Num<T>::up(g[r][i].e[j]), xh = (Num<T>::up(h[r][i].e[j]) - mean[r]) * rstd[r], gw = d * Num<T>::up(w[i].e[j]);
            c[2 * r] += gw;
            c[2 * r + 1] = fmaf(gw, xh, c[2 * r + 1]);
            dw[i][j] = fmaf(d, xh, dw[i][j]);
            db[i][j] += d;
          }
        }
    }
#pragma unroll
    for (int q = 0; q < 2 * ROWS; ++q) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) c[q] += __shfl_xor_sync(0xffffffffu, c[q], o);
      if (lane == 0) s_part[buf][q][warp] = c[q];
    }
    __syncthreads();   // (two buffers: the next round's parts do not meet this one's readers)
#pragma unroll
    for (int q = 0; q < 2 * ROWS; ++q) {
      c[q] = lane < nw ? s_part[buf][q][lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) c[q] += __shfl_xor_sync(0xffffffffu, c[q], o);
      c[q] *= inv_k;
    }
    if (p.dx == nullptr) continue;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int row = r0 + r, k = t * VEC + i * step;
        if (row >= p.M || k >= K) continue;
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = (Num<T>::up(h[r][i].e[j]) - mean[r]) * rstd[r], gw = Num<T>::up(g[r][i].e[j]) * Num<T>::up(w[i].e[j]);
          o[j] = rstd[r] * (gw - c[2 * r] - xh * c[2 * r + 1]);
        }
        if (p.dh) {
          const Piece<T, VEC> a = load<T, VEC>(static_cast<const T*>(p.dh) + row * p.ds + k);
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] += Num<T>::up(a.e[j]);
        }
        store<T, VEC>(static_cast<T*>(p.dx) + row * p.xs + k, o);
      }
  }
  if (p.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = t * VEC + i * step;
    if (k >= K) continue;
    float* const at = p.partial + static_cast<size_t>(blockIdx.x) * 2 * K + k;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      at[j] = dw[i][j];
      at[K + j] = db[i][j];
    }
  }
}

// dweight and dbias: the CTAs' parts, added in their order.
template <typename T> __global__ void __launch_bounds__(256) norm_grad_sum_kernel(const __grid_constant__ GradParams p) {
  __shared__ float s_sum[8][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const long long col = static_cast<long long>(blockIdx.x) * 32 + lane, cols = 2ll * p.K;   // dweight's columns, then dbias's
  float s = 0.f;
  if (col < cols) {
    for (int i = part; i < p.parts; i += 8) s += p.partial[i * cols + col];
  }
  s_sum[part][lane] = s;
  __syncthreads();
  if (part != 0 || col >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += s_sum[i][lane];
  if (col < p.K)
    static_cast<T*>(p.dweight)[col] = Num<T>::down(s);
  else
    static_cast<T*>(p.dbias)[col - p.K] = Num<T>::down(s);
}

// Rows that do not fit a CTA: the sums over the columns first, then dx and the column sums of 256 columns x a share of the rows.
template <typename T> __global__ void __launch_bounds__(kRowThreads) long_grad_sums_kernel(const __grid_constant__ GradParams p) {
  __shared__ double2 s_sum[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = blockIdx.x;
  const T *const h = static_cast<const T*>(p.h) + row * p.hs, *const dy = static_cast<const T*>(p.dy) + row * p.ys;
  const float mean = p.mean[row], rstd = p.rstd[row];
  double2 c = make_double2(0.0, 0.0);
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const float gw = Num<T>::up(dy[k]) * Num<T>::up(static_cast<const T*>(p.weight)[k]);
    c.x += gw;
    c.y += static_cast<double>(gw) * ((Num<T>::up(h[k]) - mean) * rstd);
  }
  c = row_sum<false>(c, s_sum);
  if (threadIdx.x == 0) {
    float* const at = p.partial + 2ll * p.K * p.parts + 2ll * row;
    at[0] = static_cast<float>(c.x / p.K);
    at[1] = static_cast<float>(c.y / p.K);
  }
}
template <typename T> __global__ void __launch_bounds__(256) long_grad_kernel(const __grid_constant__ GradParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long k = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (k >= p.K) return;
  const float w = Num<T>::up(static_cast<const T*>(p.weight)[k]);
  float dw = 0.f, db = 0.f;
  for (int row = blockIdx.y; row < p.M; row += p.parts) {
    const float* const c = p.partial + 2ll * p.K * p.parts + 2ll * row;
    const float rstd = p.rstd[row], d = Num<T>::up((static_cast<const T*>(p.dy) + row * p.ys)[k]);
    const float xh = (Num<T>::up((static_cast<const T*>(p.h) + row * p.hs)[k]) - p.mean[row]) * rstd;
    dw = fmaf(d, xh, dw);
    db += d;
    if (p.dx) {
      float o = rstd * (d * w - c[0] - xh * c[1]);
      if (p.dh) o += Num<T>::up((static_cast<const T*>(p.dh) + row * p.ds)[k]);
      (static_cast<T*>(p.dx) + row * p.xs)[k] = Num<T>::down(o);
    }
  }
  float* const at = p.partial + 2ll * p.K * blockIdx.y + k;
  at[0] = dw;
  at[p.K] = db;
}

constexpr int kGradParts = 296;   // CTAs of the gradients at most, whatever the device: their number fixes the order of the sums

// How the gradients of [M, K] are cut: pieces of VEC, NV of them a thread, ROWS rows at a time; NV = 0: rows that do not fit a CTA.
struct GradPlan {
  int vec, nv, rows, threads, parts;
};
GradPlan grad_plan(int M, int K, int elem, bool pieces) {
  GradPlan g{};
  const int v = 16 / elem, n = pieces ? K / v : K;
  g.vec = pieces ? v : 1;
  if (pieces)
    g.nv = n <= 512 ? 1 : n <= 1024 ? 2 : n <= 2048 ? 4 : 0;
  else
    g.nv = n <= 4096 ? 4 : n <= 16384 ? 16 : 0;
  g.rows = !pieces ? 1 : g.nv == 1 ? 4 : g.nv == 2 ? 2 : 1;
  g.threads = g.nv ? ((n + g.nv - 1) / g.nv + 31) / 32 * 32 : 0;
  g.parts = std::max(1, std::min(kGradParts, (M + g.rows - 1) / g.rows));
  return g;
}

template <typename T> cudaError_t launch_grad_of(GradParams p, bool pieces, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const GradPlan g = grad_plan(p.M, p.K, sizeof(T), pieces);
  p.parts = g.parts;
  float* const room = p.partial;
  if (g.nv == 0) {
    cudaError_t e = launch(long_grad_sums_kernel<T>, p.M, kRowThreads, stream, p);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((p.K + 255) / 256, g.parts);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    e = cudaLaunchKernelEx(&cfg, long_grad_kernel<T>, p);
    if (e != cudaSuccess) return e;
  } else {
    if (p.dweight == nullptr) p.partial = nullptr;
    cudaError_t e;
    if (pieces)
      e = g.nv == 1   ? launch(norm_grad_kernel<T, V, 1, 4, 512>, g.parts, g.threads, stream, p)
          : g.nv == 2 ? launch(norm_grad_kernel<T, V, 2, 2, 512>, g.parts, g.threads, stream, p)
                      : launch(norm_grad_kernel<T, V, 4, 1, 512>, g.parts, g.threads, stream, p);
    else
      e = g.nv == 4 ? launch(norm_grad_kernel<T, 1, 4, 1, kRowThreads>, g.parts, g.threads, stream, p)
                    : launch(norm_grad_kernel<T, 1, 16, 1, kRowThreads>, g.parts, g.threads, stream, p);
    if (e != cudaSuccess) return e;
  }
  if (p.dweight == nullptr) return cudaSuccess;
  p.partial = room;
  return launch(norm_grad_sum_kernel<T>, (2 * p.K + 31) / 32, 256, stream, p);
}

}  // namespace

cudaError_t launch_rows(const glowq_w8a8_rows_t& r, cudaStream_t stream) {
  const RowsParams p{r.x,        r.residual, r.weight,          r.bias,       r.hidden, r.y,          r.codes, r.scales, r.mean, r.rstd,
                     r.eps,      r.x_stride, r.residual_stride, r.hidden_stride, r.y_stride, r.code_stride, r.M,     r.K};
  if (r.dtype == GLOWQ_F16) return launch_rows_typed<__half>(p, r.norm, r.constant, stream);
  if (r.dtype == GLOWQ_BF16) return launch_rows_typed<__nv_bfloat16>(p, r.norm, r.constant, stream);
  return launch_rows_typed<float>(p, r.norm, r.constant, stream);
}

size_t layer_norm_grad_bytes(int M, int K) {
  // every plan's parts (of at most kGradParts CTAs), and the row sums of the plan for long rows
  return (2ull * K * std::min(kGradParts, std::max(M, 1)) + 2ull * std::max(M, 1)) * 4;
}

cudaError_t launch_layer_norm_grad(const glowq_layer_norm_grad_t& g, cudaStream_t stream) {
  const GradParams p{g.h,        g.dy,        g.dh,        g.weight,    g.mean, g.rstd, g.dx, g.dweight, g.dbias, static_cast<float*>(g.workspace),
                     g.h_stride, g.dy_stride, g.dh_stride, g.dx_stride, g.M,    g.K,    1};
  const int v = static_cast<int>(16 / dtype_bytes(g.dtype));
  const auto whole = [v](const void* q, long long stride) { return !q || (on(q, 16) && stride % v == 0); };
  const bool pieces = g.K % v == 0 && whole(g.h, g.h_stride) && whole(g.dy, g.dy_stride) && whole(g.dh, g.dh_stride) &&
                      whole(g.dx, g.dx_stride) && whole(g.weight, 0);
  if (g.dtype == GLOWQ_F16) return launch_grad_of<__half>(p, pieces, stream);
  if (g.dtype == GLOWQ_BF16) return launch_grad_of<__nv_bfloat16>(p, pieces, stream);
  return launch_grad_of<float>(p, pieces, stream);
}

}  // namespace glowq
