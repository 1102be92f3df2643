// Rows in front of a linear: residual add, layer norm or RMSNorm, int8 codes; and the layer norm's gradients.
//
//   h = x + residual;  v = norm(h);  scale = max |v| / 127;  code = nearest integer of v / scale
//
// All of it is bound by memory: a row is read once, stays in registers through the norm, the maximum and the codes, and every output is
// written once.  A row belongs to a CTA of as many threads as it has pieces of 4 x 16 bytes (to one warp up to 1024 16-bit columns,
// several rows to a CTA then).  Values stay in their own type in registers (16 for 32 16-bit values), so that an SM holds 1024 threads'
// rows; above 256 threads a row, CTAs take row after row, and a row's loads go out before the row in front of it is worked on.  64
// registers do not hold all of that beside the arithmetic: behind a norm the compiler spills 10 to 100 bytes a thread (fp32: none to 100),
// with the next row in flight and a residual 140 (RMSNorm) to 240 (layer norm), with eight pieces a thread 160 to 420.
//   Rows that do not begin on 16 bytes are read in 16-byte pieces all the same (see Mode).  (Element by element 4097 x 4999 fp16 took
// 39 us, floor 9.4; so 20.)
//   A code is the nearest integer of the EXACT quotient, ties to even: it does not hang on how a division rounds.  Products with a little
// less and a little more than 1 / s have the same nearest integer but where a border is near (one value in some ten thousand; of 8-bit
// mantissas, many of whose quotients are halves, one in some hundred); there the side of the border that v is on decides, which one FMA
// gives exactly.
//   us (floor), normal values: codes of 4096 x 13824 fp16 29.0 (26.0), bf16 33.1 (29.8 of activations with some loud channels, whose
// quotients are halves less often), fp32 45.0 (43.3); residual + RMSNorm + codes of 4000 x 5120 fp16 25.7 (21.9), with a layer norm 29.3,
// of 4000 x 12288 81 and 101 (52.6); layer norm of 32768 x 2048 fp16 47.5 (41.1).  What is left is bound by issue slots: 11 to 25
// instructions an element, and above 8192 columns by the spills.
//   The statistics of a norm are sums in 64 bits, rounded to fp32 once, so that they - and with them every code - do not depend on the
// order of the sums.  var = S2/K - (S1/K)^2 from one pass over the registers; where the difference costs more than 10 of the 53 bits (rows
// whose mean is 32 times their deviation) a second pass sums the squares around the mean.  (Below that the rounding to 24 bits went another
// way in less than one row of a million; at 64 deviations in one of 400 thousand, at 900 in one of two thousand.  From memory 4000 x 5120 fp16
// with codes 29 -> 50 us of such rows; from the registers 36, but then others' spills take 4 to 10 % more at 12288 columns.)
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "w8a8.h"

namespace glowq {

struct RowsParams {
  const void *x, *residual, *weight, *bias;
  void *hidden, *y;
  int8_t* codes;
  float *scales, *mean, *rstd;
  double eps, inv_k;
  long long xs, rs, hs, ys, cs;
  int M, K;
};
struct GradParams {
  const void *h, *dy, *dh, *weight;
  const float *mean, *rstd;
  void *dx, *dweight, *dbias;
  float* partial;     // [parts][2][K]; long rows: [M][2] sums behind them
  long long hs, ys, ds, xs;
  int M, K, parts, group;   // threads of a group
};

namespace {

constexpr int kNV = 4;             // 16-byte pieces per thread
constexpr int kRowThreads = 1024;  // threads of a row at most
constexpr int kWarpRows = 4;       // rows of a CTA where a warp takes one

__host__ __device__ __forceinline__ bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---------------------------------------------------------------- 16 bytes of a row
struct Vec {
  uint32_t w[4];
};
template <typename T> struct Num;
template <> struct Num<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
  static __device__ __forceinline__ void unpack(const Vec& v, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v.w[i]);
  }
  static __device__ __forceinline__ Vec pack(const float (&f)[4]) {
    return Vec{{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])}};
  }
  static __device__ __forceinline__ Vec add(const Vec& a, const Vec& b) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = __float_as_uint(__uint_as_float(a.w[i]) + __uint_as_float(b.w[i]));
    return v;
  }
  static __device__ __forceinline__ Vec mul(const Vec& a, const Vec& b) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = __float_as_uint(__uint_as_float(a.w[i]) * __uint_as_float(b.w[i]));
    return v;
  }
  // the largest absolute value so far, as bits (a NaN is above all numbers); and as the bits of a float
  static __device__ __forceinline__ uint32_t top(uint32_t m, const Vec& v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, v.w[i] & 0x7FFFFFFFu);
    return m;
  }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return m; }
};
template <> struct Num<__half> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const Vec& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ Vec pack(const float (&f)[8]) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return v;
  }
  // (sums and products of two half values, rounded once: what rounding the fp32 results gives, as 24 >= 2 * 11 + 2)
  static __device__ __forceinline__ Vec add(const Vec& a, const Vec& b) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __hadd2_rn(*reinterpret_cast<const __half2*>(&a.w[i]), *reinterpret_cast<const __half2*>(&b.w[i]));
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return v;
  }
  static __device__ __forceinline__ Vec mul(const Vec& a, const Vec& b) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __hmul2_rn(*reinterpret_cast<const __half2*>(&a.w[i]), *reinterpret_cast<const __half2*>(&b.w[i]));
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return v;
  }
  // (the maximum hands a NaN on)
  static __device__ __forceinline__ uint32_t top(uint32_t m, const Vec& v) {
    __half2 t = *reinterpret_cast<const __half2*>(&m);
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __hmax2_nan(t, __habs2(*reinterpret_cast<const __half2*>(&v.w[i])));
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t m) {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(max(m & 0x7FFFu, (m >> 16) & 0x7FFFu)))));
  }
};
template <> struct Num<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const Vec& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v.w[i] << 16);
      f[2 * i + 1] = __uint_as_float(v.w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ Vec pack(const float (&f)[8]) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return v;
  }
  // (sums and products of two nv_bfloat16 values, rounded once: what rounding the fp32 results gives, as 24 >= 2 * 11 + 2)
  static __device__ __forceinline__ Vec add(const Vec& a, const Vec& b) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a.w[i]), *reinterpret_cast<const __nv_bfloat162*>(&b.w[i]));
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return v;
  }
  static __device__ __forceinline__ Vec mul(const Vec& a, const Vec& b) {
    Vec v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&a.w[i]), *reinterpret_cast<const __nv_bfloat162*>(&b.w[i]));
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return v;
  }
  // (the maximum hands a NaN on)
  static __device__ __forceinline__ uint32_t top(uint32_t m, const Vec& v) {
    __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&m);
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __hmax2_nan(t, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v.w[i])));
    return *reinterpret_cast<const uint32_t*>(&t);
  }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return max(m & 0x7FFFu, (m >> 16) & 0x7FFFu) << 16; }
};
template <typename T> __device__ __forceinline__ float rounded(float v) { return Num<T>::up(Num<T>::down(v)); }

template <typename T> __device__ __forceinline__ Vec zeros_but(const T* row, int k, int K) {   // elements that lie in the row
  constexpr int V = Num<T>::kVec;
  T e[V];
#pragma unroll
  for (int j = 0; j < V; ++j) e[j] = k + j >= 0 && k + j < K ? row[k + j] : Num<T>::down(0.f);
  Vec v;
  memcpy(&v, e, sizeof(v));
  return v;
}
__device__ __forceinline__ Vec ld16(const void* p) {
  const uint4 u = *static_cast<const uint4*>(p);
  return Vec{{u.x, u.y, u.z, u.w}};
}
// How the rows of a call lie.  kWhole: all begin on 16 bytes and consist of whole pieces.  kSame: each row begins at the same place within
// 16 bytes in all of the call's matrices (odd widths, dense): pieces are cut where memory has 16 bytes, the first and the last of a row
// hold less, and only vectors over the columns are read across two pieces.  kAny: pieces are cut by columns.
enum Mode : int { kAny, kSame, kWhole };
template <typename T> __device__ __forceinline__ int row_offset(const T* row) {   // elements by which a row begins behind 16 bytes
  return static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
// Elements [k, k + V) of a row, zeros outside of it.
template <typename T, int MODE> __device__ __forceinline__ Vec load_row(const T* row, int k, int K) {
  constexpr int V = Num<T>::kVec;
  if (k >= K) return Vec{};
  const T* const p = row + k;
  if (MODE == kWhole) return ld16(p);
  if (MODE == kSame) return k >= 0 && k + V <= K ? ld16(p) : zeros_but<T>(row, k, K);
  if (on16(p) && k >= 0 && k + V <= K) return ld16(p);
  // what lies around the piece in whole 16 bytes, as far as it belongs to the row
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), first = at & ~static_cast<uintptr_t>(15);
  if (first < reinterpret_cast<uintptr_t>(row) || first + 32 > reinterpret_cast<uintptr_t>(row + K)) return zeros_but<T>(row, k, K);
  const Vec a = ld16(reinterpret_cast<const void*>(first)), b = ld16(reinterpret_cast<const void*>(first + 16));
  const uint32_t off = static_cast<uint32_t>(at & 15), q = off >> 2, sh = (off & 2) * 8;
  uint32_t w[8] = {a.w[0], a.w[1], a.w[2], a.w[3], b.w[0], b.w[1], b.w[2], b.w[3]};
  if (q & 2) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (q & 1) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  Vec v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.w[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], sh) : w[i];
  return v;
}
// The other way; all lanes of a warp take part, with pieces that follow one another.
template <typename T, int MODE> __device__ __forceinline__ void store_row(T* row, int k, int K, const Vec& v) {
  constexpr int V = Num<T>::kVec;
  if (MODE == kWhole) {
    if (k < K) *reinterpret_cast<uint4*>(row + k) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    return;
  }
  if (MODE == kSame) {
    if (k >= 0 && k + V <= K) {
      *reinterpret_cast<uint4*>(row + k) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    } else if (k < K) {
      T e[V];
      memcpy(e, &v, sizeof(v));
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k + j >= 0 && k + j < K) row[k + j] = e[j];
    }
    return;
  }
  if (on16(row)) {
    if (k + V <= K) {
      *reinterpret_cast<uint4*>(row + k) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    } else if (k < K) {
      T e[V];
      memcpy(e, &v, sizeof(v));
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (k + j < K) row[k + j] = e[j];
    }
    return;
  }
  // the 16 bytes in memory that end in this piece: the last `off` elements of the lane in front, then this lane's first
  const int lane = threadIdx.x & 31;
  const uint32_t bytes = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15), q = bytes >> 2, sh = (bytes & 2) * 8;
  const int off = static_cast<int>(bytes / sizeof(T));
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = __shfl_up_sync(0xffffffffu, v.w[i], 1);
    w[4 + i] = v.w[i];
  }
  // words [4 - q - half, ...) of the eight
  uint32_t u[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) u[i] = w[i + 3];                    // shifted down by 3 words: for q = 0 (and half a word)
  if (q == 1) {
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = w[i + 2];
  } else if (q == 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = w[i + 1];
  } else if (q == 3) {
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = w[i];
  }
  // (without a half the words are u[1..4])
  Vec o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.w[i] = sizeof(T) == 2 && sh ? __funnelshift_r(u[i], u[i + 1], sh) : u[i + 1];
  const int k0 = k - off;
  T mine[V], e[V];
  memcpy(mine, &v, sizeof(v));
  memcpy(e, &o, sizeof(o));
  if (lane > 0 && k0 + V <= K) {
    *reinterpret_cast<uint4*>(row + k0) = make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = lane > 0 || j >= off;   // (the first lane has only its own)
      if (in && k0 + j < K) row[k0 + j] = e[j];
    }
  }
  if (lane == 31) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j >= V - off && k + j < K) row[k + j] = mine[j];
  }
}

// ---------------------------------------------------------------- two fp32 values in one instruction
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair_of(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 parts(F2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <typename T> __device__ __forceinline__ void unpack2(const Vec& v, F2 (&f)[Num<T>::kVec / 2]) {
  float u[Num<T>::kVec];
  Num<T>::unpack(v, u);
#pragma unroll
  for (int i = 0; i < Num<T>::kVec / 2; ++i) f[i] = pair_of(u[2 * i], u[2 * i + 1]);
}

// ---------------------------------------------------------------- codes
struct Scale {
  float s, lo, hi;   // the scale; a little less and a little more than its inverse
  bool plain;        // neither zero, tiny nor NaN
};
// `bits`: the row's largest absolute value, as the bits of a float (a NaN is above all numbers)
__device__ __forceinline__ Scale make_scale(uint32_t bits) {
  Scale r;
  const float a = __uint_as_float(bits);
  r.s = bits >= 0x7F800000u ? CUDART_NAN_F : __fdiv_rn(a, 127.f);
  r.plain = bits < 0x7F800000u && a >= 0x1p-100f;
  const float inv = r.plain ? __fdiv_rn(1.f, r.s) : 0.f;   // (off by half a step at most; lo and hi by two steps and a rounding)
  r.lo = inv * (1.f - 0x1p-22f);
  r.hi = inv * (1.f + 0x1p-22f);
  return r;
}
constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: a sum with it is rounded to an integer
// Which of two neighbouring integers (as sums with kMagic) is nearest to v / s: the side of the border between them that v is on, and the
// even one on the border itself.  (One rounding, of a difference that is zero or more than an ulp: the sign is exact.)
__device__ __forceinline__ float side(float v, float s, float a, float b) {
  const float over = fmaf(-0.5f * s, (a - kMagic) + (b - kMagic), v);
  if (over == 0.f) return __float_as_uint(a) & 1u ? b : a;
  return over > 0.f ? fmaxf(a, b) : fminf(a, b);
}
// Rows of values below 2^-100, where the scale may be a subnormal number: both are scaled up first, which is exact.
__device__ __noinline__ int code_tiny(float v, float s) {
  if (!(s > 0.f)) return 0;   // zero, NaN
  const float sv = v * 0x1p64f, ss = s * 0x1p64f, inv = __fdiv_rn(1.f, ss);
  const float a = fmaf(sv, inv * (1.f - 0x1p-22f), kMagic), b = fmaf(sv, inv * (1.f + 0x1p-22f), kMagic);
  const int n = static_cast<int>((a == b ? a : side(sv, ss, a, b)) - kMagic);
  return max(-127, min(127, n));
}
// The codes of V values, four to a word.
template <int V> __device__ __forceinline__ void codes_of(const float (&v)[V], const Scale& sc, uint32_t (&out)[V / 4]) {
  uint32_t c[V];
  if (sc.plain) {
    // v / s lies between v lo and v hi: where both have the same nearest integer, so has the quotient
    float m[V];
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      float n[4];
      uint32_t differ = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[i + j] = fmaf(v[i + j], sc.lo, kMagic);
        n[j] = fmaf(v[i + j], sc.hi, kMagic);
        differ |= __float_as_uint(m[i + j]) ^ __float_as_uint(n[j]);
      }
      if (differ) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (m[i + j] != n[j]) m[i + j] = side(v[i + j], sc.s, m[i + j], n[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = __float_as_uint(m[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = static_cast<uint32_t>(code_tiny(v[j], sc.s));
  }
#pragma unroll
  for (int i = 0; i < V / 4; ++i)
    out[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
}
// The codes of columns [k, k + V); `al`: the row of codes begins on V bytes.  kSame: k + off is a multiple of V, all lanes of a warp take
// part with pieces that follow one another, and what goes to V bytes of memory comes from two lanes.
template <int V, int MODE> __device__ __forceinline__ void store_codes(int8_t* row, int k, int K, bool al, int off, const uint32_t (&w)[V / 4]) {
  const auto one = [&](uint64_t c, int from, int first, int last) {   // bytes [first, last) of c, the first of which is column `from`'s
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j >= first && j < last && from + j >= 0 && from + j < K) row[from + j] = static_cast<int8_t>(c >> (8 * j));
  };
  const auto all = [&](uint64_t c, int at) {
    if constexpr (V == 8)
      *reinterpret_cast<uint2*>(row + at) = make_uint2(static_cast<uint32_t>(c), static_cast<uint32_t>(c >> 32));
    else
      *reinterpret_cast<uint32_t*>(row + at) = static_cast<uint32_t>(c);
  };
  uint64_t c = w[0];
  if constexpr (V == 8) c |= static_cast<uint64_t>(w[1]) << 32;
  if (MODE != kSame || off == 0) {
    if (k >= K) return;
    if (MODE == kWhole || (al && k + V <= K))
      all(c, k);
    else
      one(c, k, 0, V);
    return;
  }
  const int lane = threadIdx.x & 31, at = k + off - V;   // the V bytes in front of this piece's border
  const uint64_t before = __shfl_up_sync(0xffffffffu, c, 1);
  const uint64_t mix = before >> (8 * off) | c << (8 * (V - off));
  if (lane > 0) {
    if (al && at + V <= K)
      all(mix, at);
    else
      one(mix, at, 0, V);
  } else {
    one(mix, at, V - off, V);   // (the lane in front is another warp's)
  }
  if (lane == 31) one(c >> (8 * off), k + off, 0, V - off);
}

// ---------------------------------------------------------------- sums over a row's threads
// (butterflies: every lane ends with the same bits)
__device__ __forceinline__ double warp_sum(double v, int first = 16) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o <= first) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Both sums of a pair, in 12 shuffles instead of 20: half of the lanes add up one, half the other.
__device__ __forceinline__ double2 warp_sum(double2 v) {
  const bool upper = threadIdx.x & 16;
  const double other = __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
  const double mine = warp_sum((upper ? v.y : v.x) + other, 8), theirs = __shfl_xor_sync(0xffffffffu, mine, 16);
  return upper ? make_double2(theirs, mine) : make_double2(mine, theirs);
}
// Over a row's threads; PAIR: both sums, else y alone.
template <bool WARP, bool PAIR> __device__ __forceinline__ double2 row_sum(double2 v, double2* room) {
  v = PAIR ? warp_sum(v) : make_double2(0.0, warp_sum(v.y));
  if (WARP) return v;
  const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  if (nw <= 4) {   // (as many loads as shuffles would take)
    v = room[0];
    for (int i = 1; i < nw; ++i) {
      const double2 u = room[i];
      if (PAIR) v.x += u.x;
      v.y += u.y;
    }
    return v;
  }
  v = lane < nw ? room[lane] : make_double2(0.0, 0.0);
  return PAIR ? warp_sum(v) : make_double2(0.0, warp_sum(v.y));
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
template <int NORM> __device__ __forceinline__ Stats make_stats(double mean, double var, double eps) {
  if (var < 0.0) var = 0.0;   // (a NaN stays)
  return Stats{NORM == GLOWQ_NORM_LAYER ? static_cast<float>(mean) : 0.f, static_cast<float>(rsqrt(var + eps))};
}
// What h - mean is multiplied by: rstd, but nothing where mean * rstd is above all numbers.  Such a row is constant (values that differ at
// all differ by 2^-24 of their mean, and rstd is no more than the inverse of a 2^16th of that), in rows of a type's lowest value say: its
// h - mean is zero, and the zeros past its end give (0 - mean) * 0 in place of an infinity that no weight of zero takes out of the sums.
__device__ __forceinline__ float times(float mean, float rstd) {
  return fabsf(mean) * rstd > 3.4028235e38f && rstd <= 3.4028235e38f ? 0.f : rstd;
}

// Rows by a CTA of up to THREADS threads, or (THREADS = 32) by a warp; so many CTAs to an SM that a thread has 64 registers.
constexpr int row_ctas(int threads) { return threads == 32 ? 8 : threads == 256 ? 4 : threads == 512 ? 2 : 1; }
template <typename T, int NORM, bool RES, bool CODES, int MODE, int THREADS, int NV = kNV>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kWarpRows : THREADS, row_ctas(THREADS)) rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int V = Num<T>::kVec;
  constexpr bool WARP = THREADS == 32;
  __shared__ double2 s_sum[3][32];
  __shared__ uint32_t s_max[2][32];
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, step = (WARP ? 32 : blockDim.x) * V, K = p.K;
  const int row0 = WARP ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x, rows = WARP ? gridDim.x * kWarpRows : gridDim.x;
  const T *const w = static_cast<const T*>(p.weight), *const b = static_cast<const T*>(p.bias);
  const auto x_row = [&](int row) { return static_cast<const T*>(p.x) + row * p.xs; };
  const auto r_row = [&](int row) { return static_cast<const T*>(p.residual) + row * p.rs; };
  // Columns of the thread's pieces.  Rows of whole pieces: a thread that has none left takes the row's last one again (the same values go
  // to the same place, and sums leave it out); that costs no branches.
  int off = 0;   // kSame: of the present row
  const auto column = [&](int i) { return MODE == kWhole ? min(t * V + i * step, K - V) : t * V + i * step - (MODE == kSame ? off : 0); };
  Vec x[NV], r[RES ? NV : 1];
  const auto fetch = [&](int row) {
    const T *const xr = x_row(row), *const rr = RES ? r_row(row) : nullptr;
    if (MODE == kSame) off = row_offset(xr);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = load_row<T, MODE>(xr, column(i), K);
      if (RES) r[i] = load_row<T, MODE>(rr, column(i), K);
    }
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (only now: the launch behind may take it that all in front of this one is complete)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (row0 < p.M) fetch(row0);
  int buf = 0;
  constexpr bool kAhead = THREADS > 256 && NV == kNV && MODE == kWhole;   // CTAs take row after row; else a row each
  for (int row = row0; row < p.M; row += kAhead ? rows : p.M, buf ^= 1) {
    // (a reduction's room is used again two rows later: everybody is past its barrier by then)
    Vec h[NV];
    if (RES) {
      T* const hid = p.hidden ? static_cast<T*>(p.hidden) + row * p.hs : nullptr;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        h[i] = Num<T>::add(x[i], r[i]);
        if (hid) store_row<T, MODE>(hid, column(i), K, h[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) h[i] = x[i];
    }
    if (kAhead && row + rows < p.M) fetch(row + rows);

    if (NORM != GLOWQ_NORM_NONE) {
      // (elements behind the row's end are zeros)
      double2 sum = make_double2(0.0, 0.0);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float f[V];
        Num<T>::unpack(h[i], f);
        double2 s = make_double2(0.0, 0.0);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double d = f[j];
          if (NORM == GLOWQ_NORM_LAYER) s.x += d;
          s.y = fma(d, d, s.y);
        }
        if (t * V + i * step - (MODE == kSame ? off : 0) < K) {
          sum.x += s.x;
          sum.y += s.y;
        }
      }
      sum = row_sum<WARP, NORM == GLOWQ_NORM_LAYER>(sum, s_sum[buf]);
      const double mean = sum.x * p.inv_k;
      double var = sum.y * p.inv_k - mean * mean;
      if (NORM == GLOWQ_NORM_LAYER && var < 0x1p-10 * mean * mean) {
        // more than 10 bits went in the difference: once more, around the mean (and from memory, which takes no registers from the others;
        // a quotient, which is exact where the mean is: a constant row's deviation is nothing, not 2^-53 of its value)
        const double mu = sum.x / K;
        double2 s = make_double2(0.0, 0.0);
        const T *const xr = x_row(row), *const rr = RES ? r_row(row) : nullptr;
        for (int k = t; k < K; k += step / V) {
          const float f = RES ? rounded<T>(Num<T>::up(xr[k]) + Num<T>::up(rr[k])) : Num<T>::up(xr[k]);
          const double d = static_cast<double>(f) - mu;
          s.y = fma(d, d, s.y);
        }
        var = row_sum<WARP, false>(s, s_sum[2]).y * p.inv_k;
        if (!WARP) __syncthreads();   // (this room has no second half)
      }
      const Stats st = make_stats<NORM>(mean, var, p.eps);
      if (t == 0) {
        if (p.mean) p.mean[row] = st.mean;
        if (p.rstd) p.rstd[row] = st.rstd;
      }
      const float by = CODES ? times(st.mean, st.rstd) : st.rstd;
      T* const y = CODES ? nullptr : static_cast<T*>(p.y) + row * p.ys;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = column(i);
        const Vec wv = load_row<T, MODE == kWhole ? kWhole : kAny>(w, k, K);
        float f[V];
        Num<T>::unpack(h[i], f);
        // (past the end: zeros times zeros)
        if (NORM == GLOWQ_NORM_LAYER) {
          float wf[V], bf[V];
          Num<T>::unpack(wv, wf);
          Num<T>::unpack(b ? load_row<T, MODE == kWhole ? kWhole : kAny>(b, k, K) : Vec{}, bf);
#pragma unroll
          for (int j = 0; j < V; ++j) f[j] = fmaf((f[j] - st.mean) * by, wf[j], bf[j]);
          h[i] = Num<T>::pack(f);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) f[j] *= st.rstd;
          h[i] = Num<T>::mul(Num<T>::pack(f), wv);
        }
        if (!CODES) store_row<T, MODE>(y, k, K, h[i]);
      }
    }

    if (CODES) {
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        top = Num<T>::top(top, h[i]);   // (zeros behind the row's end)
      const Scale sc = make_scale(row_max<WARP>(Num<T>::top_bits(top), s_max[buf]));
      if (t == 0) p.scales[row] = sc.s;
      int8_t* const out = p.codes + row * p.cs;
      const bool al = MODE == kWhole || (reinterpret_cast<uintptr_t>(out) & (V - 1)) == 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = column(i);
        float f[V];
        uint32_t c4[V / 4];
        Num<T>::unpack(h[i], f);
        codes_of<V>(f, sc, c4);
        store_codes<V, MODE>(out, k, K, al, off, c4);
      }
    }
  }
}

// Rows that do not fit a CTA's registers: the same in passes over the row, which stays in L2.
template <typename T, int NORM, bool CODES>
__global__ void __launch_bounds__(kRowThreads) long_rows_kernel(const __grid_constant__ RowsParams p) {
  __shared__ double2 s_sum[32];
  __shared__ uint32_t s_max[32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row = blockIdx.x, K = p.K;
  const T* const x = static_cast<const T*>(p.x) + row * p.xs;
  const T* const res = p.residual ? static_cast<const T*>(p.residual) + row * p.rs : nullptr;
  const auto value = [&](int k) {
    const float v = Num<T>::up(x[k]);
    return res ? rounded<T>(v + Num<T>::up(res[k])) : v;
  };
  Stats st{0.f, 1.f};
  if (NORM != GLOWQ_NORM_NONE) {
    double2 sum = make_double2(0.0, 0.0);
    double mean = 0.0, mu = 0.0;   // (as in rows_kernel: the mean to be held, and that which deviations are taken from)
    if (NORM == GLOWQ_NORM_LAYER) {
      for (int k = threadIdx.x; k < K; k += blockDim.x) sum.x += value(k);
      const double total = row_sum<false, true>(sum, s_sum).x;
      mean = total * p.inv_k;
      mu = total / K;
      __syncthreads();
    }
    for (int k = threadIdx.x; k < K; k += blockDim.x) {
      const double d = static_cast<double>(value(k)) - mu;
      sum.y = fma(d, d, sum.y);
    }
    st = make_stats<NORM>(mean, row_sum<false, true>(sum, s_sum).y * p.inv_k, p.eps);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[row] = st.mean;
      if (p.rstd) p.rstd[row] = st.rstd;
    }
  }
  const T *const w = static_cast<const T*>(p.weight), *const b = static_cast<const T*>(p.bias);
  const auto result = [&](int k) {
    const float h = value(k);
    if (NORM == GLOWQ_NORM_NONE) return h;
    if (NORM == GLOWQ_NORM_LAYER) return rounded<T>(fmaf((h - st.mean) * st.rstd, Num<T>::up(w[k]), b ? Num<T>::up(b[k]) : 0.f));
    return rounded<T>(Num<T>::up(w[k]) * rounded<T>(h * st.rstd));
  };
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
    for (int k = 4 * threadIdx.x; k < K; k += 4 * blockDim.x) {
      float v[4];
      uint32_t c4[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = k + j < K ? result(k + j) : 0.f;
      codes_of<4>(v, sc, c4);
      store_codes<4, kAny>(p.codes + row * p.cs, k, K, false, 0, c4);
    }
  }
}

// ahead: the kernel may begin while the one in front of it still runs (it waits for its end by itself)
template <typename Kernel, typename Params>
cudaError_t launch(Kernel kernel, dim3 grid, int threads, cudaStream_t stream, const Params& p, bool ahead = true) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ahead && use_pdl() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int NORM, bool RES, bool CODES, int MODE>
cudaError_t launch_rows_cut(const RowsParams& p, int sms, cudaStream_t stream) {
  constexpr int V = Num<T>::kVec;
  // (a row that begins within 16 bytes may touch one piece more)
  const int pieces = (p.K + V - 1) / V + (MODE == kSame ? 1 : 0), threads = ((pieces + kNV - 1) / kNV + 31) / 32 * 32;
  if (threads == 32)
    return launch(rows_kernel<T, NORM, RES, CODES, MODE, 32>, dim3((p.M + kWarpRows - 1) / kWarpRows), 32 * kWarpRows, stream, p);
  if (threads <= 256) return launch(rows_kernel<T, NORM, RES, CODES, MODE, 256>, dim3(p.M), threads, stream, p);
  // (where the next row is read ahead, as many CTAs as the registers allow take all rows)
  if constexpr (MODE == kWhole) {
    if (threads <= 512)
      return launch(rows_kernel<T, NORM, RES, CODES, MODE, 512>, dim3(std::min(p.M, sms * (512 * row_ctas(512) / threads))), threads, stream, p);
  }
  if (threads <= kRowThreads)
    return launch(rows_kernel<T, NORM, RES, CODES, MODE, kRowThreads>, dim3(MODE == kWhole ? std::min(p.M, sms) : p.M), threads, stream, p);
  if (pieces <= 2 * kNV * kRowThreads)
    return launch(rows_kernel<T, NORM, RES, CODES, MODE, kRowThreads, 2 * kNV>, dim3(p.M), kRowThreads, stream, p);
  return launch(long_rows_kernel<T, NORM, CODES>, dim3(p.M), kRowThreads, stream, p);
}
template <typename T, int NORM, bool RES, bool CODES> cudaError_t launch_rows_of(const RowsParams& p, int sms, cudaStream_t stream) {
  constexpr int V = Num<T>::kVec;
  const auto whole = [](const void* q, long long stride) { return on16(q) && stride % V == 0; };
  const bool codes = !CODES || ((reinterpret_cast<uintptr_t>(p.codes) & (V - 1)) == 0 && p.cs % V == 0);
  if (p.K % V == 0 && whole(p.x, p.xs) && whole(p.residual, p.rs) && whole(p.hidden, p.hs) && whole(p.y, p.ys) && on16(p.weight) &&
      on16(p.bias) && codes)
    return launch_rows_cut<T, NORM, RES, CODES, kWhole>(p, sms, stream);
  // Codes alone: x is the only matrix whose rows may lie anywhere; shifting what is read takes less than shifting codes (20000 x 2999 fp16
  // 54 us, so 70).  Behind a norm the rows' own places are taken where all matrices share them (6000 x 9001 bf16 with a residual and
  // RMSNorm 148 us, 20000 x 2999 fp16 168); matrices that do not take passes over the row (315 and 413).
  if constexpr (NORM == GLOWQ_NORM_NONE) {
    return launch_rows_cut<T, NORM, RES, CODES, kAny>(p, sms, stream);
  } else {
    const auto same = [&](const void* q, long long stride) {
      return !q || (((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p.x)) & 15u) == 0 && (stride - p.xs) % V == 0);
    };
    if (same(p.residual, p.rs) && same(p.hidden, p.hs) && same(p.y, p.ys) && codes)
      return launch_rows_cut<T, NORM, RES, CODES, kSame>(p, sms, stream);
    return launch(long_rows_kernel<T, NORM, CODES>, dim3(p.M), kRowThreads, stream, p);
  }
}
template <typename T> cudaError_t launch_rows_typed(const RowsParams& p, int norm, int sms, cudaStream_t stream) {
  if (norm == GLOWQ_NORM_NONE) return launch_rows_of<T, GLOWQ_NORM_NONE, false, true>(p, sms, stream);
  if (norm == GLOWQ_NORM_RMS)
    return p.residual ? launch_rows_of<T, GLOWQ_NORM_RMS, true, true>(p, sms, stream) : launch_rows_of<T, GLOWQ_NORM_RMS, false, true>(p, sms, stream);
  if (p.codes)
    return p.residual ? launch_rows_of<T, GLOWQ_NORM_LAYER, true, true>(p, sms, stream)
                      : launch_rows_of<T, GLOWQ_NORM_LAYER, false, true>(p, sms, stream);
  return p.residual ? launch_rows_of<T, GLOWQ_NORM_LAYER, true, false>(p, sms, stream)
                    : launch_rows_of<T, GLOWQ_NORM_LAYER, false, false>(p, sms, stream);
}

// ---------------------------------------------------------------- gradients of the layer norm
// A CTA holds one or several groups of threads that have a row's columns between them (NV pieces of 16 bytes a thread); a group takes ROWS
// rows at a time, and the next ones' loads go out before these are worked on.  A thread keeps to its columns: the sums of dweight and
// dbias stay in its registers until the end.  Reads h, dy (dh) and writes dx once.  32768 x 2048 fp16 90 us (floor 61.6): bound by issue
// slots, 24.5 instructions an element, a third of them moves and addresses, and by a barrier for every round.  Wider rows (16 bits: above 2048
// columns) go one at a time through CTAs of 64 registers a thread: 8192 x 5120 bf16 80 us (38.5) with 35 instructions an element, fp32 130
// (77); with two pieces a thread, which spill 430 bytes a thread of 16-bit rows, 8192 x 9216 bf16 252 (69), 8192 x 12288 297 (92).
// (A warp along each row first and threads down its columns then, the second reads from L1: 2048 columns 26 instructions, 117 us.)
constexpr int kGradParts = 304;    // CTAs of the gradients at most, whatever the device: their number fixes the order of the sums
constexpr int kGradThreads = 1024;

template <typename T, int MODE, int NV, int ROWS, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) norm_grad_kernel(const __grid_constant__ GradParams p) {
  constexpr int V = Num<T>::kVec;
  extern __shared__ float s_all[];                // [2][warps][2 ROWS], at the end [groups][2][K]
  const int g = threadIdx.x / p.group, t = threadIdx.x - g * p.group, groups = blockDim.x / p.group, step = p.group * V, K = p.K;
  const int nw = p.group >> 5, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // A group's rows lie `units` apart, a multiple of eight: all of them begin at the same place within 16 bytes.
  const int units = gridDim.x * groups, unit = blockIdx.x * groups + g, stride = units * ROWS;
  const int off = MODE == kSame ? row_offset(static_cast<const T*>(p.h) + unit * p.hs) : 0;
  // The weights of one piece stay in registers, those of two are read again (from L1) for every row: 8192 x 12288 bf16 298 us, held 358;
  // 8192 x 8192 fp32 172, held 212.
  constexpr bool kHeld = NV == 1;
  F2 w[kHeld ? NV : 1][V / 2], dw[NV][V / 2], db[NV][V / 2];
  const auto weights = [&](int i) {   // of piece i
    if (!kHeld) unpack2<T>(load_row<T, MODE == kWhole ? kWhole : kAny>(static_cast<const T*>(p.weight), t * V + i * step - off, K), w[0]);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kHeld) unpack2<T>(load_row<T, MODE == kWhole ? kWhole : kAny>(static_cast<const T*>(p.weight), t * V + i * step - off, K), w[i]);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) dw[i][j] = db[i][j] = 0ull;
  }
  const float inv_k = 1.f / static_cast<float>(K);
  Vec nh[ROWS][NV], nd[ROWS][NV];
  float nmean[ROWS], nrstd[ROWS];
  const auto fetch = [&](int r0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int row = r0 + r * units;
      const T *const hr = static_cast<const T*>(p.h) + row * p.hs, *const dr = static_cast<const T*>(p.dy) + row * p.ys;
      const int cols = row < p.M ? K : 0;
      nmean[r] = row < p.M ? p.mean[row] : 0.f;
      nrstd[r] = row < p.M ? p.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        nh[r][i] = load_row<T, MODE>(hr, t * V + i * step - off, cols);
        nd[r][i] = load_row<T, MODE>(dr, t * V + i * step - off, cols);
      }
    }
  };
  fetch(unit);
  int buf = 0;
  for (int base = blockIdx.x * groups; base < p.M; base += stride, buf ^= 1) {   // (the same number of rounds for all groups)
    const int r0 = base + g;
    // xh = (h - mean) rstd, as the forward pass has it (h rstd - mean rstd in one FMA rounds mean rstd: a constant row of 999 would give
    // dweight 0.006 dy), and dy; zeros past the end of a row (dy) and past the last row (dy)
    F2 xh[ROWS][NV][V / 2], d[ROWS][NV][V / 2];
    float rstd[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      rstd[r] = nrstd[r];
      const float by = times(nmean[r], rstd[r]);
      const F2 by2 = pair_of(by, by), shift = pair_of(-nmean[r], -nmean[r]);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        unpack2<T>(nh[r][i], xh[r][i]);
        unpack2<T>(nd[r][i], d[r][i]);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) xh[r][i][j] = mul2(add2(xh[r][i][j], shift), by2);
      }
    }
    if (base + stride < p.M) fetch(r0 + stride);
    // sums of dy w and dy w xh over the columns
    constexpr int Q = 2 * ROWS;
    float c[Q];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      F2 s1 = 0ull, s2 = 0ull;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        weights(i);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          const F2 gw = mul2(d[r][i][j], w[kHeld ? i : 0][j]);
          s1 = add2(s1, gw);
          s2 = fma2(gw, xh[r][i][j], s2);
          dw[i][j] = fma2(d[r][i][j], xh[r][i][j], dw[i][j]);
          db[i][j] = add2(db[i][j], d[r][i][j]);
        }
      }
      c[r] = parts(s1).x + parts(s1).y;
      c[ROWS + r] = parts(s2).x + parts(s2).y;
    }
    // Over the lanes: each step halves the sums that a lane keeps, until it has one of the Q, of 32 / Q lanes' values; lane l then has
    // sum l / (32 / Q) of its warp.
    int keep = Q / 2;
#pragma unroll
    for (int o = 16; o >= 32 / Q; o >>= 1, keep >>= 1) {
      const bool upper = lane & o;
#pragma unroll
      for (int q = 0; q < Q / 2; ++q)
        if (q < keep) {
          const float away = upper ? c[q] : c[q + keep], mine = upper ? c[q + keep] : c[q];
          c[q] = mine + __shfl_xor_sync(0xffffffffu, away, o);
        }
    }
#pragma unroll
    for (int o = 16 / Q; o > 0; o >>= 1) c[0] += __shfl_xor_sync(0xffffffffu, c[0], o);
    float sum = c[0];
    int per = 32 / Q;   // lane q * per has the row's sum q
    if (nw > 1) {
      // a group's warps, in an order of their own: lane l adds sum l % Q of every (32 / Q)th of them
      float* const room = s_all + buf * warps * Q;
      if (lane % per == 0) room[warp * Q + lane / per] = sum;
      __syncthreads();   // (two buffers: the next round's sums do not meet this one's readers)
      sum = 0.f;
      for (int i = lane / Q; i < nw; i += 32 / Q) sum += room[(g * nw + i) * Q + lane % Q];
#pragma unroll
      for (int o = 16; o >= Q; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      per = 1;
    }
    if (p.dx == nullptr) continue;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int row = r0 + r * units;
      const float c1 = -__shfl_sync(0xffffffffu, sum, r * per) * inv_k * rstd[r], c2 = -__shfl_sync(0xffffffffu, sum, (ROWS + r) * per) * inv_k * rstd[r];
      if (row >= p.M) continue;   // (whole warps)
      T* const out = static_cast<T*>(p.dx) + row * p.xs;
      const T* const more = p.dh ? static_cast<const T*>(p.dh) + row * p.ds : nullptr;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = t * V + i * step - off;
        weights(i);
        float o[V];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          const float2 u = parts(fma2(xh[r][i][j], pair_of(c2, c2), fma2(mul2(d[r][i][j], w[kHeld ? i : 0][j]), pair_of(rstd[r], rstd[r]), pair_of(c1, c1))));
          o[2 * j] = u.x;
          o[2 * j + 1] = u.y;
        }
        if (more) {
          float a[V];
          Num<T>::unpack(load_row<T, MODE>(more, k, K), a);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += a[j];
        }
        store_row<T, MODE>(out, k, K, Num<T>::pack(o));
      }
    }
  }
  if (p.partial == nullptr) return;
  float* const at = p.partial + static_cast<size_t>(blockIdx.x) * 2 * K;
  if (groups > 1) {   // the groups' sums, added in their order
    __syncthreads();
    float* const mine = s_all + g * 2 * K;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int k = t * V + i * step - off + j;
        if (k >= 0 && k < K) {
          mine[k] = j & 1 ? parts(dw[i][j / 2]).y : parts(dw[i][j / 2]).x;
          mine[K + k] = j & 1 ? parts(db[i][j / 2]).y : parts(db[i][j / 2]).x;
        }
      }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * K; k += blockDim.x) {
      float s = s_all[k];
      for (int i = 1; i < groups; ++i) s += s_all[i * 2 * K + k];
      at[k] = s;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int k = t * V + i * step - off + j;
      if (k >= 0 && k < K) {
        at[k] = j & 1 ? parts(dw[i][j / 2]).y : parts(dw[i][j / 2]).x;
        at[K + k] = j & 1 ? parts(db[i][j / 2]).y : parts(db[i][j / 2]).x;
      }
    }
}

// dweight and dbias: the CTAs' parts, added in their order.
template <typename T> __global__ void __launch_bounds__(256) norm_grad_sum_kernel(const __grid_constant__ GradParams p) {
  __shared__ float s_sum[8][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const long long col = static_cast<long long>(blockIdx.x) * 32 + lane, cols = 2ll * p.K;   // dweight's columns, then dbias's
  float s = 0.f;
  if (col < cols) {
#pragma unroll 8
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
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row = blockIdx.x;
  const T *const h = static_cast<const T*>(p.h) + row * p.hs, *const dy = static_cast<const T*>(p.dy) + row * p.ys;
  const float mean = p.mean[row], rstd = p.rstd[row];
  double2 c = make_double2(0.0, 0.0);
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const float gw = Num<T>::up(dy[k]) * Num<T>::up(static_cast<const T*>(p.weight)[k]);
    c.x += gw;
    c.y += static_cast<double>(gw) * ((Num<T>::up(h[k]) - mean) * rstd);
  }
  c = row_sum<false, true>(c, s_sum);
  if (threadIdx.x == 0) {
    float* const at = p.partial + 2ll * p.K * p.parts + 2ll * row;
    at[0] = static_cast<float>(c.x / p.K);
    at[1] = static_cast<float>(c.y / p.K);
  }
}
template <typename T> __global__ void __launch_bounds__(256) long_grad_kernel(const __grid_constant__ GradParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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

// How the gradients of [M, K] are cut: NV pieces a thread, ROWS rows at a time, groups of a CTA; NV = 0: rows that do not fit a CTA.
struct GradPlan {
  int nv, group, groups, rows, parts;
  size_t smem;
};
GradPlan grad_plan(int M, int K, int vec, bool same) {
  GradPlan g{};
  const int n = (K + vec - 1) / vec + (same ? 1 : 0);
  // (two 16-bit pieces that are shifted need more registers than there are: 6000 x 9001 bf16 278 us, in passes over the rows 264; at 12001
  // and 16001 columns fp16 the passes take 4 to 6 % more)
  g.nv = n <= kGradThreads ? 1 : n <= 2 * kGradThreads && !(same && vec == 8) ? 2 : 0;
  g.group = g.nv ? ((n + g.nv - 1) / g.nv + 31) / 32 * 32 : 256;
  g.groups = g.group >= 256 ? 1 : 256 / g.group;
  // two rows at a time in 128 registers and two CTAs to an SM, or one row in 64 and one or two CTAs
  g.rows = g.nv && g.group * g.groups <= 256 ? 2 : 1;
  const int per = g.rows * g.groups;
  g.parts = std::max(1, std::min(g.nv && g.group <= 512 ? 296 : 148, g.nv ? (M + per - 1) / per : M / 16));
  // (the rows of a group lie a multiple of eight apart, and no CTA is left for a second round)
  if (same && g.nv) g.parts = std::max(8, g.parts / 8 * 8);
  const int warps = g.group * g.groups / 32;
  g.smem = std::max<size_t>(2ull * warps * 2 * g.rows, g.groups > 1 ? 2ull * g.groups * K : 0) * 4;
  return g;
}

template <typename T, int MODE> cudaError_t launch_grad_of(GradParams p, cudaStream_t stream) {
  const GradPlan g = grad_plan(p.M, p.K, Num<T>::kVec, MODE == kSame);
  p.parts = g.parts;
  p.group = g.group;
  float* const room = p.partial;
  cudaError_t e;
  if (g.nv == 0) {
    e = launch(long_grad_sums_kernel<T>, dim3(p.M), kRowThreads, stream, p);
    if (e == cudaSuccess) e = launch(long_grad_kernel<T>, dim3((p.K + 255) / 256, g.parts), 256, stream, p);
  } else {
    if (p.dweight == nullptr) p.partial = nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(g.parts);
    cfg.blockDim = dim3(g.group * g.groups);
    cfg.dynamicSmemBytes = g.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl() ? 1 : 0;
    e = g.nv == 2                    ? cudaLaunchKernelEx(&cfg, norm_grad_kernel<T, MODE, 2, 1, kGradThreads, 1>, p)
        : g.rows == 2                 ? cudaLaunchKernelEx(&cfg, norm_grad_kernel<T, MODE, 1, 2, 256, 2>, p)
                                    : cudaLaunchKernelEx(&cfg, norm_grad_kernel<T, MODE, 1, 1, kGradThreads, 1>, p);
  }
  if (e != cudaSuccess || p.dweight == nullptr) return e;
  p.partial = room;
  return launch(norm_grad_sum_kernel<T>, dim3((2 * p.K + 31) / 32), 256, stream, p);
}

template <typename T> cudaError_t launch_grad_typed(const GradParams& p, cudaStream_t stream) {
  constexpr int V = Num<T>::kVec;
  const auto whole = [](const void* q, long long stride) { return on16(q) && stride % V == 0; };
  if (p.K % V == 0 && whole(p.h, p.hs) && whole(p.dy, p.ys) && whole(p.dh, p.ds) && whole(p.dx, p.xs) && on16(p.weight))
    return launch_grad_of<T, kWhole>(p, stream);
  const auto same = [&](const void* q, long long stride) {
    return !q || (((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p.h)) & 15u) == 0 && (stride - p.hs) % V == 0);
  };
  if (same(p.dy, p.ys) && same(p.dh, p.ds) && same(p.dx, p.xs)) return launch_grad_of<T, kSame>(p, stream);
  return launch_grad_of<T, kAny>(p, stream);
}

}  // namespace
}  // namespace glowq
